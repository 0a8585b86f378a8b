// Attention of a batch whose sequences share a prefix: row s of q head h of
// sequence b attends to the prefix's keys 0 .. n_prefix - 1, stored once for all
// sequences, and to the keys 0 .. n_past[b] + s of its own cache.
//
// One softmax over both parts: each part's rows leave (max, sum, unnormalised O)
// for their share of the keys, and a merge weighs the shares by 2^(m - max m).
//
//   * The prefix: the R = B G S rows of a kv head (G = Hq / Hkv q heads, S new
//     tokens of B sequences) are ONE matrix, so a key is read once for all of
//     them instead of once per sequence.
//   * A sequence's own keys: its G S rows of a kv head.
//
// What bounds it: reading the keys once (decode), the products (many new tokens:
// there the forward kernel's walk, fa2_fwd_bf16.hip, takes over).  A workgroup over
// the prefix holds up to 128 rows, whose K and V tiles come by asynchronous loads two
// tiles ahead (a ring of three in LDS); S^T = K Q^T leaves a row in a lane pair, so
// the running maximum and sum need one exchange each, and P goes into its product
// from registers.  Shares of the prefix fill the CUs where rows are few.  P is rounded
// to bf16 for the matrix cores and the row's sum adds the rounded values, so the
// weights sum to one; maxima, sums and O are fp32, and o is rounded once.
//
// Measured, bf16 Hkv8 G4 D128, us of the attention and the merge (keys' rate): 64
// sequences behind 8191 keys, up to 700 of their own, 33, 6.9 (3.9 TB/s); 4 behind
// 32000 29, 4.2 (4.6 TB/s; a large copy 4.8); 16 behind 2048 10.6, 4.5; 8 x 5 tokens
// behind 3001 16.4, 4.9.  16 heads of 64, 32 sequences behind 1021: 9.7, 4.5.  The
// short ones are chains: two launches and a few tiles of one after another's work.
// Eight wavefronts a workgroup were slower than four.
//
// Reference: no counterpart (no KV cache, examples/llama_generate.rs:373-381);
// each row is the reference's attention (flash_attn2.rs:61-126) over the
// concatenated keys.
#include "attn_rows.h"
#include "f32_mfma.h"

namespace {

// What a launch works on.  Rows of a kv head: r = b GS + rem, rem = g S + s, GS
// = G S; q and o are [B, Hkv, GS, D] = [B, Hq, S, D].
struct Shape {
  int batch, hkv, gs, s;          // sequences, kv heads, rows of a sequence per kv head, new tokens
  int n_prefix, prefix_len;       // prefix keys; rows of a prefix head's slab
  int cache_len;                  // rows of a (b, kv head)'s cache
  const int* past;                // keys in the caches before the call: past[b past_stride]
  int past_stride, past_imm;      // past null: past_imm
  int p_splits, p_keys;           // shares of the prefix, keys per share (a multiple of TK)
  int row_tiles, tile_rows;       // row tiles of a kv head over the prefix, rows of each
  int o_splits;                   // shares of a sequence's own keys
  float scale;
};
// Partials: of prefix share i the rows (hk, r) at [i][hk R + r], of own share i
// the rows (b, hk, rem) at [p_splits R Hkv + i B Hkv GS + ...]: both parts hold N
// = B Hkv GS rows per share.  m in the log2 domain; -inf: no key.
struct Parts {
  float *m, *l, *o;
};

DEVI int past_of(const Shape& a, int b) {
  const int p = a.past ? a.past[(long)b * a.past_stride] : a.past_imm;
  return min(max(p, -a.s), a.cache_len);
}

// ---------------------------------------------------------------------------
// bf16
// ---------------------------------------------------------------------------
constexpr int kRing = 3;  // prefix tiles in LDS: one in use, two loading

template <int D, int NW>
struct __attribute__((aligned(16))) PrefixSmem {
  static constexpr int TILE = TK * D * 2;
  union {
    char ring[kRing][2][TILE];   // the prefix: K and V tiles that all wavefronts use
    char own[NW][2][TILE];       // own keys: a K and a V tile of each wavefront
    char out[NW][32 * D * 4];    // a wavefront's rows on their way out
    struct {
      float o[NW][32 * D];
      float m[NW][32], l[NW][32];
    } c;                         // own keys: the wavefronts' shares
  } u;
};

// grid: p_splits * row_tiles * hkv workgroups over the prefix, then o_splits *
// batch * hkv * ceil(gs / 32) over the sequences' own keys.
template <int D, int NW>
__device__ void prefix_attn(const bf16* __restrict__ q, const bf16* __restrict__ kp,
                            const bf16* __restrict__ vp, const bf16* __restrict__ kc,
                            const bf16* __restrict__ vc, const Shape a, const Parts out) {
  constexpr int TILE = TK * D * 2;
  constexpr int NLD = TILE / 1024;        // 1 KiB loads per K or V tile
  __shared__ PrefixSmem<D, NW> sm;
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const long n_rows = (long)a.batch * a.hkv * a.gs;
  const float sl2 = a.scale * kLog2e;
  const int n_pre = a.p_splits * a.row_tiles * a.hkv;
  Rows<D> st;
  st.init();
  uint32_t pb[8];
  u32x4 va[2][Rows<D>::DT];

  if ((int)blockIdx.x < n_pre) {
    // ---- a share of the prefix, 32 NW of a kv head's rows --------------------
    // row tiles innermost: those of one share run on one XCD and read its keys
    // from that L2
    int id = xcd_remap(blockIdx.x, n_pre);
    const int rt = id % a.row_tiles;
    id /= a.row_tiles;
    const int hk = id % a.hkv, split = id / a.hkv;
    const int rows = a.batch * a.gs;
    const int first = rt * a.tile_rows + wave * 32;  // the wavefront's rows
    const int r_end = min(rows, (rt + 1) * a.tile_rows), r = first + l32;
    {
      const int rc = min(r, rows - 1), b = rc / a.gs;
      st.load_q(q + ((long)(b * a.hkv + hk) * a.gs + (rc - b * a.gs)) * D, r < r_end);
    }
    const int k0 = split * a.p_keys, keys = min(a.p_keys, a.n_prefix - k0);
    const int n_tiles = (keys + TK - 1) / TK;
    // descriptors over this share: rows past it load as zeros
    const long base = ((long)hk * a.prefix_len + k0) * D;
    const auto krs = make_rsrc(kp + base, keys * D * 2);
    const auto vrs = make_rsrc(vp + base, keys * D * 2);
    constexpr int PER = 2 * NLD / NW;  // loads of a wavefront per tile
    static_assert(2 * NLD % NW == 0, "");
    auto load = [&](int it) {
      const int buf = it % kRing;
      const int soff = __builtin_amdgcn_readfirstlane(it * TILE);
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int n = i * NW + wave;  // K loads first
        if (NLD % NW == 0 ? i < NLD / NW : n < NLD)
          dma16(krs, sm.u.ring[buf][0] + n * 1024, swz<SWZ_ROW, D>(n * 64 + lane) * 16, soff);
        else
          dma16(vrs, sm.u.ring[buf][1] + (n - NLD) * 1024,
                swz<SWZ_DUAL, D>((n - NLD) * 64 + lane) * 16, soff);
      }
    };
    load(0);
    if (n_tiles > 1) load(1);
    // q has arrived (it was asked for first); said here, or the loop's first
    // product waits for as many of the tiles' loads as q's would be
#pragma unroll
    for (int c = 0; c < Rows<D>::DC; ++c) pin(st.q[c]);
    for (int it = 0; it < n_tiles; ++it) {
      // tile it has landed (tile it + 1 may still fly); every wavefront is done
      // with tile it - 1, whose buffer tile it + 2 takes
      if (it + 1 < n_tiles) __builtin_amdgcn_s_waitcnt(kVmWait<PER>());
      else __builtin_amdgcn_s_waitcnt(kVmcnt0);
      barrier_only();
      if (it + 2 < n_tiles) load(it + 2);
      if (first >= r_end) continue;  // (uniform: a wavefront without rows only loads)
      const char* kt = sm.u.ring[it % kRing][0];
      const char* vt = sm.u.ring[it % kRing][1];
      f32x16 s = st.scores(kt);
      if ((it + 1) * TK > keys) st.mask(s, keys - it * TK);
      st.softmax(s, sl2, pb);
      st.read_v(vt, va);
      st.product(va, pb);
      __builtin_amdgcn_s_waitcnt(kLgkmcnt0);
    }
    barrier_only();  // the ring becomes the rows' way out
    const float l_tot = st.l + other_half(st.l);
    const long row0 = split * n_rows + (long)hk * rows + first;
    if (g == 0 && r < r_end) {
      out.m[row0 + l32] = st.m;
      out.l[row0 + l32] = l_tot;
    }
    if (first < r_end)
      store_tile_rows<D>(sm.u.out[wave], out.o + row0 * D, r_end - first,
                         [&](int t, int j) {
                           return f32x4{st.acc[t][4 * j], st.acc[t][4 * j + 1],
                                        st.acc[t][4 * j + 2], st.acc[t][4 * j + 3]};
                         });
    return;
  }

  // ---- a share of a sequence's own keys, 32 of its rows: a wavefront takes a part
  // of the share, through a tile of its own ------------------------------------
  const int groups = (a.gs + 31) / 32;
  int id = blockIdx.x - n_pre;
  const int split = id % a.o_splits;
  id /= a.o_splits;
  const int rg = id % groups;
  id /= groups;
  const int hk = id % a.hkv, b = id / a.hkv;
  const int past = __builtin_amdgcn_readfirstlane(past_of(a, b));
  const int rem = rg * 32 + l32;
  const long row0 = (long)(b * a.hkv + hk) * a.gs;
  st.load_q(q + (row0 + min(rem, a.gs - 1)) * D, rem < a.gs);
  const int lim = min(past + rem % a.s + 1, a.cache_len);  // the lane's keys
  const int n_keys = min(past + a.s, a.cache_len);
  const int waves = a.o_splits * NW;
  const int kpw = ((n_keys + waves - 1) / waves + TK - 1) / TK * TK;
  const int k0 = (split * NW + wave) * kpw;
  const int keys = max(0, min(kpw, n_keys - k0));
  const int n_tiles = (keys + TK - 1) / TK;
  const long base = ((long)(b * a.hkv + hk) * a.cache_len + k0) * D;
  const auto krs = make_rsrc(kc + base, keys * D * 2);
  const auto vrs = make_rsrc(vc + base, keys * D * 2);
  auto load_k = [&](int it) {
    const int soff = __builtin_amdgcn_readfirstlane(it * TILE);
#pragma unroll
    for (int i = 0; i < NLD; ++i)
      dma16(krs, sm.u.own[wave][0] + i * 1024, swz<SWZ_ROW, D>(i * 64 + lane) * 16, soff);
  };
  auto load_v = [&](int it) {
    const int soff = __builtin_amdgcn_readfirstlane(it * TILE);
#pragma unroll
    for (int i = 0; i < NLD; ++i)
      dma16(vrs, sm.u.own[wave][1] + i * 1024, swz<SWZ_DUAL, D>(i * 64 + lane) * 16, soff);
  };
  if (n_tiles > 0) {
    load_k(0);
    load_v(0);
  }
  for (int it = 0; it < n_tiles; ++it) {
    // K of a tile before its V, each refilled as soon as it has been read
    __builtin_amdgcn_s_waitcnt(kVmWait<NLD>());
    f32x16 s = st.scores(sm.u.own[wave][0]);
    __builtin_amdgcn_s_waitcnt(kLgkmcnt0);
    if (it + 1 < n_tiles) load_k(it + 1);
    if (k0 + (it + 1) * TK > min(past + 1, n_keys)) st.mask(s, lim - k0 - it * TK);
    st.softmax(s, sl2, pb);
    if (it + 1 < n_tiles) __builtin_amdgcn_s_waitcnt(kVmWait<NLD>());
    else __builtin_amdgcn_s_waitcnt(kVmcnt0);
    st.read_v(sm.u.own[wave][1], va);
    __builtin_amdgcn_s_waitcnt(kLgkmcnt0);
    if (it + 1 < n_tiles) load_v(it + 1);
    st.product(va, pb);
  }
  const float l_tot = st.l + other_half(st.l);
  const int n_here = min(32, a.gs - rg * 32);
  __syncthreads();  // every wavefront is done with its tiles
  if (l32 < n_here) {  // (of 32 rows a group of 4 has 4: all were 5 us of 16 at 64 sequences)
    if (g == 0) {
      sm.u.c.m[wave][l32] = st.m;
      sm.u.c.l[wave][l32] = l_tot;
    }
    float* orow = sm.u.c.o[wave] + l32 * D;
#pragma unroll
    for (int t = 0; t < Rows<D>::DT; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<f32x4*>(orow + 32 * t + 8 * j + 4 * g) = f32x4{
            st.acc[t][4 * j], st.acc[t][4 * j + 1], st.acc[t][4 * j + 2], st.acc[t][4 * j + 3]};
  }
  __syncthreads();
  const long p0 = (a.p_splits + split) * n_rows + row0 + rg * 32;
  for (int i = tid; i < n_here * D; i += NW * 64) {
    const int rr = i / D, d = i - rr * D;
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) mm = fmaxf(mm, sm.u.c.m[w][rr]);
    const float ref = mm == -INFINITY ? 0.0f : mm;
    float num = 0.0f, den = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float e = fast_exp2(sm.u.c.m[w][rr] - ref);
      num += e * sm.u.c.o[w][rr * D + d];
      den += e * sm.u.c.l[w][rr];
    }
    out.o[(p0 + rr) * D + d] = num;
    if (d == 0) {
      out.m[p0 + rr] = mm;
      out.l[p0 + rr] = den;
    }
  }
}

// ---------------------------------------------------------------------------
// fp32: a wavefront per 16 rows, on the fp32 matrix cores, K and V read straight
// from memory in operand order (as the fp32 decode kernel does).
//   shares  grid p_splits * row_tiles * hkv, then o_splits * batch * hkv *
//           ceil(gs / 16): a share of one part's keys, to the merge
//   whole   grid batch * hkv * ceil(gs / 16): all keys of a sequence's rows, both
//           parts one after the other, to the output: few keys, or many rows
// ---------------------------------------------------------------------------
template <int D, bool WHOLE>
__device__ void prefix_attn_f32(const float* __restrict__ q, const float* __restrict__ kp,
                                const float* __restrict__ vp, const float* __restrict__ kc,
                                const float* __restrict__ vc, const Shape a, const Parts out,
                                float* __restrict__ o, int merged) {
  constexpr int NC = Geo<D>::NC, VW = Geo<D>::VW, NH = Geo<D>::NH;
  const int lane = threadIdx.x, j = lane & 15, g = lane >> 4;
  const long n_rows = (long)a.batch * a.hkv * a.gs;
  const int n_share = WHOLE ? 0 : a.p_splits * a.row_tiles * a.hkv;
  const float *kb, *vb, *qrow;
  long prow;           // the lane's row among the partials
  bool valid;
  int k0, k1, lim;     // the keys of the walk; the lane's end
  int hk, b = 0, rem = 0, past = 0;
  if ((int)blockIdx.x < n_share) {
    int id = xcd_remap(blockIdx.x, n_share);
    const int rt = id % a.row_tiles;
    id /= a.row_tiles;
    hk = id % a.hkv;
    const int split = id / a.hkv;
    const int rows = a.batch * a.gs, r = rt * 16 + j;
    const int rc = min(r, rows - 1);
    b = rc / a.gs;
    valid = r < rows;
    qrow = q + ((long)(b * a.hkv + hk) * a.gs + (rc - b * a.gs)) * D;
    kb = kp + (long)hk * a.prefix_len * D;
    vb = vp + (long)hk * a.prefix_len * D;
    k0 = split * a.p_keys;
    k1 = min(k0 + a.p_keys, a.n_prefix);
    lim = k1;
    prow = split * n_rows + (long)hk * rows + rc;
  } else {
    const int groups = (a.gs + 15) / 16, splits = WHOLE ? 1 : a.o_splits;
    int id = blockIdx.x - n_share;
    const int split = id % splits;
    id /= splits;
    const int rg = id % groups;
    id /= groups;
    // (whole: kv head by kv head, for the prefix in an XCD's L2)
    hk = WHOLE ? id / a.batch : id % a.hkv;
    b = WHOLE ? id - hk * a.batch : id / a.hkv;
    past = past_of(a, b);
    rem = min(rg * 16 + j, a.gs - 1);
    valid = rg * 16 + j < a.gs;
    const long row0 = (long)(b * a.hkv + hk) * a.gs;
    qrow = q + (row0 + rem) * D;
    kb = kc + (long)(b * a.hkv + hk) * a.cache_len * D;
    vb = vc + (long)(b * a.hkv + hk) * a.cache_len * D;
    const int n_keys = min(past + a.s, a.cache_len);
    const int per = ((n_keys + splits - 1) / splits + TK - 1) / TK * TK;
    k0 = split * per;
    k1 = min(k0 + per, n_keys);
    lim = min(past + rem % a.s + 1, k1);
    prow = (a.p_splits + split) * n_rows + row0 + rem;
  }
  f32x4 qf[NC];
  row_regs<D>(qrow, g, qf);
  f32x4 acc[NH][VW];
  zero_acc<D>(acc);
  float m = -INFINITY, l = 0.0f;
  // whole: the prefix first, then (kb, vb, k0, k1, lim)
  for (int part = WHOLE && a.n_prefix > 0 ? 0 : 1; part < 2; ++part) {
    const bool pre = WHOLE && part == 0;
    const float* ks = pre ? kp + (long)hk * a.prefix_len * D : kb;
    const float* vs = pre ? vp + (long)hk * a.prefix_len * D : vb;
    const int end = pre ? a.n_prefix : k1, stop = pre ? end : lim;
    for (int t0 = pre ? 0 : k0; t0 < end; t0 += 32) {
      // rows at or past the end re-read the last; their P is zero, and so is their V
      f32x4 kf[2][NC];
      float vf[8][NH][VW];
#pragma unroll
      for (int u = 0; u < 2; ++u)
        row_regs<D>(ks + (long)min(t0 + 16 * u + j, end - 1) * D, g, kf[u]);
#pragma unroll
      for (int s = 0; s < 8; ++s) {
        const float* row = vs + (long)min(t0 + 16 * (s >> 2) + 4 * g + (s & 3), end - 1) * D;
#pragma unroll
        for (int h = 0; h < NH; ++h) {
          if constexpr (VW == 4) {
            const f32x4 x = *reinterpret_cast<const f32x4g*>(row + 64 * h + 4 * j);
#pragma unroll
            for (int e = 0; e < 4; ++e) vf[s][h][e] = x[e];
          } else if constexpr (VW == 2) {
            const f32x2 x = *reinterpret_cast<const f32x2g*>(row + 2 * j);
            vf[s][h][0] = x[0];
            vf[s][h][1] = x[1];
          } else {
            vf[s][h][0] = D == 8 && j >= 8 ? 0.0f : row[j];
          }
        }
      }
      __builtin_amdgcn_sched_barrier(0);  // every load is issued first
      f32x4 s[2] = {};
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int u = 0; u < 2; ++u) s[u] = mfma4(kf[u][c][e], qf[c][e], s[u]);
      float mx = -INFINITY;
      const float m_old = m;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          s[u][r] = t0 + 16 * u + 4 * g + r < stop ? s[u][r] * a.scale : -INFINITY;
          mx = fmaxf(mx, s[u][r]);
        }
      m = fmaxf(m, max_g(mx));
      const float ref = m == -INFINITY ? 0.0f : m;  // no key of the row so far
      const float alpha = expf(m_old - ref);
      l *= alpha;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          s[u][r] = expf(s[u][r] - ref);
          l += s[u][r];
        }
#pragma unroll
      for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int e = 0; e < VW; ++e) acc[h][e] *= alpha;
      if (t0 + 32 > end) {
#pragma unroll
        for (int x = 0; x < 8; ++x)
          if (t0 + 16 * (x >> 2) + 4 * g + (x & 3) >= end)
#pragma unroll
            for (int h = 0; h < NH; ++h)
#pragma unroll
              for (int e = 0; e < VW; ++e) vf[x][h][e] = 0.0f;
      }
      // new tokens' own rows that some row must not see: 0 * Inf of a masked value is
      // NaN in a sum over keys, so a tile that is not finite goes key by key to the
      // rows that see it (tested where S > 1, on a walk's last tiles alone)
      if (!pre && a.s > 1 && min(t0 + 32, end) > past + 1) {
        float bad = 0.0f;
#pragma unroll
        for (int x = 0; x < 8; ++x)
#pragma unroll
          for (int h = 0; h < NH; ++h)
#pragma unroll
            for (int e = 0; e < VW; ++e) bad += 0.0f * vf[x][h][e];
        if (__any(bad != bad)) {
#pragma unroll
          for (int x = 0; x < 8; ++x)
#pragma unroll 1
            for (int kg = 0; kg < 4; ++kg) {
              const int key = t0 + 16 * (x >> 2) + 4 * kg + (x & 3);
              const float p = __shfl(s[x >> 2][x & 3], 16 * kg + j);
              if (key < stop) add_row<D>(vs + (long)key * D, p, g, acc);
            }
          continue;
        }
      }
#pragma unroll
      for (int x = 0; x < 8; ++x)
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
          for (int e = 0; e < VW; ++e)
            acc[h][e] = mfma4(vf[x][h][e], s[x >> 2][x & 3], acc[h][e]);
    }
  }
  l = sum_g(l);
  if (!valid) return;
  if constexpr (WHOLE) {
    long to = ((long)(b * a.hkv + hk) * a.gs + rem) * D;
    if (merged) {
      const int group = a.gs / a.s, h = hk * group + rem / a.s, t = rem % a.s;
      to = (((long)b * a.s + t) * a.hkv * group + h) * D;
    }
    // a row without a key: zeros (l NaN: NaN)
    store_col<D>(o + to, acc, g, [l](float x) { return l == 0.0f ? 0.0f : x / l; });
    return;
  }
  if (g == 0) {
    out.m[prow] = m * kLog2e;
    out.l[prow] = l;
  }
  store_col<D>(out.o + prow * D, acc, g, [](float x) { return x; });
}

// The shares of a row, weighed and summed.  A row takes TPR threads: D / 4 lanes of
// four d each in groups that go over the shares side by side.  A workgroup (256
// threads) a row where rows are few, so that the loads of many shares fly at once; a
// wavefront a row where they are many.
template <typename T, int TPR>
__device__ void prefix_merge(const Parts in, T* __restrict__ o, const Shape a, int head_dim,
                             int merged) {
  constexpr int NT = 256, RPW = NT / TPR;
  // per row a weight per share (padded to 4), then the groups' sums
  extern __shared__ __attribute__((aligned(16))) float lds[];
  __shared__ float red[2][NT / 64];
  const int row_i = threadIdx.x / TPR, tid = threadIdx.x % TPR, shares = a.p_splits + a.o_splits;
  const long n_rows = (long)a.batch * a.hkv * a.gs;
  const long want = (long)blockIdx.x * RPW + row_i, row = min(want, n_rows - 1);
  const int bh = (int)(row / a.gs), rem = (int)(row - (long)bh * a.gs);
  const int b = bh / a.hkv, hk = bh - b * a.hkv;
  const long prow = ((long)hk * a.batch + b) * a.gs + rem;  // among the prefix's rows
  const int padded = (shares + 3) / 4 * 4;
  float* wt = lds + row_i * padded;
  float* sums = lds + RPW * padded + row_i * 4 * TPR;
  auto at = [&](int i) { return i * n_rows + (i < a.p_splits ? prow : row); };
  // the largest of the shares' maxima, and of the sums
  auto across = [&](float v, int slot, bool sum) {
    v = sum ? wave_sum(v) : wave_max(v);
    if (TPR == 64) return v;
    if ((threadIdx.x & 63) == 0) red[slot][threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[slot][0];
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) v = sum ? v + red[slot][w] : fmaxf(v, red[slot][w]);
    return v;
  };
  float mx = -INFINITY;
  for (int i = tid; i < shares; i += TPR) {
    wt[i] = in.m[at(i)];
    mx = fmaxf(mx, wt[i]);
  }
  mx = across(mx, 0, false);
  const float ref = mx == -INFINITY ? 0.0f : mx;  // no key at all: zeros
  float den = 0.0f;
  for (int i = tid; i < shares; i += TPR) {
    const float e = fast_exp2(wt[i] - ref);
    wt[i] = e;
    den += e * in.l[at(i)];
  }
  den = across(den, 1, true);
  __syncthreads();
  const int lanes = head_dim / 4, groups = TPR / lanes;
  const int grp = tid / lanes, d = (tid - grp * lanes) * 4;
  f32x4 acc = {};
  constexpr int U = 4;  // shares of a group in flight
  for (int i0 = grp; i0 < shares; i0 += U * groups) {
    f32x4 v[U];
    float e[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {  // (past the end: the last one, unweighed)
      const int i = min(i0 + u * groups, shares - 1);
      e[u] = i0 + u * groups < shares ? wt[i] : 0.0f;
      v[u] = *reinterpret_cast<const f32x4*>(in.o + at(i) * head_dim + d);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) acc += e[u] * v[u];
  }
  *reinterpret_cast<f32x4*>(sums + grp * head_dim + d) = acc;
  __syncthreads();
  long to = row * head_dim;
  if (merged) {
    const int h = hk * (a.gs / a.s) + rem / a.s, s = rem % a.s;
    to = (((long)b * a.s + s) * a.hkv * (a.gs / a.s) + h) * head_dim;
  }
  for (int dd = tid; dd < head_dim && want < n_rows; dd += TPR) {
    float v = 0.0f;
    for (int i = 0; i < groups; ++i) v += sums[i * head_dim + dd];
    o[to + dd] = (T)(den == 0.0f ? 0.0f : v / den);
  }
}

}  // namespace

#define TEENY_PREFIX_BF16_INST(D, NW)                                                           \
  extern "C" __global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(2)))     \
  void teeny_prefix_attn_bf16_d##D##_w##NW(const bf16* q, const bf16* kp, const bf16* vp,       \
                                           const bf16* kc, const bf16* vc, Shape a, Parts p) {  \
    prefix_attn<D, NW>(q, kp, vp, kc, vc, a, p);                                                \
  }
TEENY_PREFIX_BF16_INST(64, 1)
TEENY_PREFIX_BF16_INST(64, 2)
TEENY_PREFIX_BF16_INST(64, 4)
TEENY_PREFIX_BF16_INST(128, 1)
TEENY_PREFIX_BF16_INST(128, 2)
TEENY_PREFIX_BF16_INST(128, 4)

#define TEENY_PREFIX_F32_INST(D)                                                               \
  extern "C" __global__ __launch_bounds__(64) void teeny_prefix_attn_f32_d##D(                 \
      const float* q, const float* kp, const float* vp, const float* kc, const float* vc,      \
      Shape a, Parts p) {                                                                       \
    prefix_attn_f32<D, false>(q, kp, vp, kc, vc, a, p, nullptr, 0);                            \
  }                                                                                             \
  extern "C" __global__ __launch_bounds__(64) void teeny_prefix_attn_f32_d##D##_whole(         \
      const float* q, const float* kp, const float* vp, const float* kc, const float* vc,      \
      Shape a, float* o, int merged) {                                                          \
    prefix_attn_f32<D, true>(q, kp, vp, kc, vc, a, {}, o, merged);                             \
  }
TEENY_PREFIX_F32_INST(8)
TEENY_PREFIX_F32_INST(16)
TEENY_PREFIX_F32_INST(32)
TEENY_PREFIX_F32_INST(64)
TEENY_PREFIX_F32_INST(128)

#define TEENY_PREFIX_MERGE_INST(TN, T, SFX, TPR)                                               \
  extern "C" __global__ __launch_bounds__(256) void teeny_prefix_merge_##TN##SFX(              \
      Parts p, T* o, Shape a, int head_dim, int merged) {                                       \
    prefix_merge<T, TPR>(p, o, a, head_dim, merged);                                            \
  }
TEENY_PREFIX_MERGE_INST(bf16, bf16, , 256)
TEENY_PREFIX_MERGE_INST(bf16, bf16, _wave, 64)
TEENY_PREFIX_MERGE_INST(f32, float, , 256)
TEENY_PREFIX_MERGE_INST(f32, float, _wave, 64)
