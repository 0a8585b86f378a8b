// A cache in pages: what writes it, attends to it and moves its pages (the layout:
// paged.h).
//
//   split    the QKV projection's rows: q rotated to [T, Hq, D], k (rotated) and v to
//            the rows of their pages
//   attn     attention of a sequence's new tokens over its pages, few rows a kv head
//            (many: the forward kernel, fa2_fwd_bf16.hip), in shares of the keys
//   merge    the shares of a row, weighed and summed
//   copy     pages of all layers copied within the pool
//
// Reference: no counterpart (no KV cache, examples/llama_generate.rs:373-381); a row
// is the reference's attention (flash_attn2.rs:61-126) over the sequence's keys.
#include "attn_rows.h"
#include "f32_mfma.h"
#include "paged.h"

namespace {

// ---------------------------------------------------------------------------
// split: a workgroup a token.  Its row of the projection is one run of memory; a thread's
// first loads are in flight while the first wavefront finds the token's sequence, position
// and page and its (cos, sin), once for all heads.
//
// Angles are formed and reduced in 64 bits: of position p the fp32 product p base^
// (-2k/D) is off by up to p 2^-24 radians (2e-3 at 32768), as much as a bf16 rounds.
//
// Bound by HBM where there are many tokens, else by one chain (starts, length, page table,
// rows).  Hq32 Hkv8 D128, us with rows from HBM: bf16 512 tokens 6.4, 2048 13, 8208 40.5 (5.0
// TB/s), 32768 150; fp32 9.5, 23, 80 (5.0 TB/s), 304; 64 tokens of 64 sequences, in caches,
// 3.5, 4.1.  Workgroups of four tokens: 9.7, 16, 41.7, 158; 15, 26, 85, 318; 6.9, 9.9.
// ---------------------------------------------------------------------------
template <typename T, bool PARTS>
__device__ void paged_split(const T* __restrict__ qkv, const float* __restrict__ parts, int n_parts,
                            long part_stride, T* __restrict__ q_out, T* __restrict__ kp,
                            T* __restrict__ vp, const Paged a, int lg_d, double ln_base) {
  constexpr int NT = 256, VN = Vec16<T>::N, U = PARTS ? 1 : 3;
  __shared__ float2 cs[64];
  __shared__ long at;  // element of the token's row in its page, head 0; -1: none
  __shared__ int live;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int head_dim = 1 << lg_d, lg_v = lg_d - __builtin_ctz(VN);  // vectors of a head
  const int total = (a.hq + 2 * a.hkv) << lg_v;                     // ... of the token
  const int t = blockIdx.x;
  const long src = (long)t * total * VN;
  u32x4 raw[U];
  float sum[VN];
  auto load = [&](int i0) __attribute__((always_inline)) {
    if constexpr (PARTS) {
      if (i0 < total) ld_parts<T, VN>(parts + src + (long)i0 * VN, part_stride, n_parts, sum);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u)
        raw[u] = *reinterpret_cast<const u32x4*>(qkv + src + (long)min(i0 + u * NT, total - 1) * VN);
    }
  };
  load(tid);
  if (wave == 0) {
    const int b = seq_at(a, t);
    long row = -1, pos = 0;
    int in = 0;
    if (b >= 0) {
      const Seq s = seq_of(a, b);
      const int i = t - s.t0;
      in = i >= 0 && i < s.n;
      pos = (long)(a.past ? a.past[b] : a.past_all) + i;  // (behind the table too: q is rotated)
      if (in && pos >= 0 && pos < s.cap) {
        const int page = a.table[(long)b * a.ld + (pos >> a.lg)];
        if ((unsigned)page < (unsigned)a.n_pages)
          row = (((long)page * a.hkv << a.lg) + (pos & ((1 << a.lg) - 1))) << lg_d;
      }
    }
    if (lane == 0) {
      at = row;
      live = in;
    }
    if (lane < head_dim / 2) {
      // turns, less whole ones: in [-1/2, 1/2]
      double turn = (double)pos * (exp(-2.0 * lane * ln_base / head_dim) * 0.15915494309189533577);
      turn -= rint(turn);
      double sn, cn;
      sincospi(2.0 * turn, &sn, &cn);
      cs[lane] = make_float2((float)cn, (float)sn);
    }
  }
  __syncthreads();
  if (!live) return;
  const long head_k = (long)1 << (a.lg + lg_d);  // elements between a page's kv heads
  for (int i0 = tid; i0 < total; i0 += U * NT) {
    if (i0 != tid) load(i0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * NT;
      if (i >= total) break;
      const int head = i >> lg_v, v = i & ((1 << lg_v) - 1);
      T* dst;
      if (head < a.hq) {
        dst = q_out + (((long)t * a.hq + head) << lg_d);
      } else {
        if (at < 0) continue;
        const bool is_k = head < a.hq + a.hkv;
        dst = (is_k ? kp : vp) + at + (head - a.hq - (is_k ? 0 : a.hkv)) * head_k;
      }
      float in[VN], out[VN];
#pragma unroll
      for (int j = 0; j < VN; ++j) {
        const uint32_t w = raw[u][VN == 4 ? j : j / 2];
        if constexpr (PARTS) in[j] = sum[j];
        else if constexpr (VN == 4) in[j] = __builtin_bit_cast(float, w);
        else in[j] = j & 1 ? bf16hi(w) : bf16lo(w);
      }
      if (head < a.hq + a.hkv) {
        const float2* c = cs + v * (VN / 2);
#pragma unroll
        for (int j = 0; j < VN / 2; ++j)
          rope_rotate(in[2 * j], in[2 * j + 1], c[j].x, c[j].y, out[2 * j], out[2 * j + 1]);
      } else {
#pragma unroll
        for (int j = 0; j < VN; ++j) out[j] = in[j];
      }
      Vec16<T>::store(dst + v * VN, out);
    }
  }
}

// ---------------------------------------------------------------------------
// copy: page `to` of a plane becomes page `from` of it, for every pair and plane; no
// page is read by one pair and written by another.  A workgroup moves 16 KiB, four loads
// a thread before its first store.  Bound by HBM: 67 pages of 128 KiB in 64 planes, 1.12 GB
// read and written, 217 us (5.2 TB/s; a copy of 2 GiB reaches 5.0); 16 of 32 KiB 8.4 us.
// ---------------------------------------------------------------------------
constexpr int kMoves = 448;  // pairs in a launch's arguments
struct Moves {
  int n;
  int from[kMoves], to[kMoves];
};
__device__ void copy_pages(char* pages, long plane_bytes, long page_bytes, int chunks, const Moves& m) {
  const int pair = blockIdx.x / chunks, ch = blockIdx.x - pair * chunks;
  char* plane = pages + blockIdx.y * plane_bytes;
  const u32x4* src = reinterpret_cast<const u32x4*>(plane + m.from[pair] * page_bytes);
  u32x4* dst = reinterpret_cast<u32x4*>(plane + m.to[pair] * page_bytes);
  const long n = page_bytes / 16;
  constexpr int U = 4;
  const long i0 = (long)ch * (U * 256) + threadIdx.x;
  u32x4 v[U];
#pragma unroll
  for (int u = 0; u < U; ++u) v[u] = src[min(i0 + u * 256, n - 1)];
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (i0 + u * 256 < n) dst[i0 + u * 256] = v[u];
}

// ---------------------------------------------------------------------------
// attn: softmax(q K^T scale) V with a running maximum and sum, 32 keys at a time.  The
// rows of a kv head (tokens x q heads of its group, up to 32) are the columns of one
// matrix product, so a key is read once for all of them.  A wavefront has K and V tiles
// and a run of the keys of its own: no barrier until the end, its loads (of whole runs of
// 16 rows, which lie in one page whatever the page size) go on while it computes, and
// pages of any order cost a scalar load each.
//
// Bound by HBM with many keys: 64 sequences of up to 8191 keys, Hkv8 D128, 1.09 GB, 204 us
// (5.3 TB/s); 8 of 3001 keys, 5 tokens each, 16 kv heads of 64, 57 MB, 14.5 us (3.9 TB/s: six
// tiles a wavefront, nothing hides the first).  One sequence of 700 keys 10.2 us: a launch, the
// chain from starts to the page's rows, three tiles a wavefront, the wavefronts' join.
// ---------------------------------------------------------------------------
template <int D, int NW>
struct __attribute__((aligned(16))) AttnSmem {
  static constexpr int TILE = TK * D * 2;
  union {
    char tile[NW][2][TILE];  // a K and a V tile of each wavefront
    struct {
      float o[NW][32 * D];
      float m[NW][32], l[NW][32];
    } c;                     // the wavefronts' shares
  } u;
};

template <int DT>
DEVI bool any_bad(const u32x4 (*va)[DT]) {
  uint32_t bad = 0;
#pragma unroll
  for (int hh = 0; hh < 2; ++hh)
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) bad |= bf16_bad(va[hh][t][i]);
  return __any(bad != 0);
}

// grid: splits * groups * batch * hkv; a workgroup: a share of the keys of 32 rows,
// of which each wavefront takes a run through tiles of its own.
template <int D, int NW>
__device__ void paged_attn(const bf16* __restrict__ q, const bf16* __restrict__ kp,
                           const bf16* __restrict__ vp, bf16* __restrict__ o, const Paged a,
                           const PagedPlan pl, const PagedParts out) {
  constexpr int TILE = TK * D * 2, NLD = TILE / 1024;
  __shared__ AttnSmem<D, NW> sm;
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int id = blockIdx.x;
  const int rg = id % pl.groups;
  id /= pl.groups;
  const int hk = id % a.hkv;
  id /= a.hkv;
  const int split = id % pl.splits, b = id / pl.splits;
  PageWalk walk(a, b);
  const Seq s = seq_of(a, b);
  const int G = a.hq / a.hkv;
  const long all = (long)s.n * G;
  if (all > pl.few || rg * 32 >= all) return;
  const int rows = (int)all, n_sh = paged_shares(s, pl.keys, pl.splits);
  if (split >= n_sh) return;
  const int r = rg * 32 + l32, rc = min(r, rows - 1), tok = rc / G;
  const long row = (long)(s.t0 + tok) * a.hq + hk * G + (rc - tok * G);
  const float sl2 = pl.scale * kLog2e;
  Rows<D> st;
  st.init();
  st.load_q(q + row * D, r < rows);
  // keys: of the lane's row; of the rows' first and last token
  const int lim = s.keys(tok), lim0 = s.keys(rg * 32 / G);
  const int last = s.keys((min(rows, rg * 32 + 32) - 1) / G);
  const int s0 = split * pl.keys, s1 = split + 1 < pl.splits ? min(s0 + pl.keys, last) : last;
  const int kpw = ((max(0, s1 - s0) + NW - 1) / NW + TK - 1) / TK * TK;
  const int k0 = s0 + wave * kpw, end = min(k0 + kpw, s1);
  const int n_tiles = max(0, end - k0 + TK - 1) / TK;
  // loads of a tile: 16 rows lie in one page (its rows at or past `end`, and absent
  // pages, lie outside the descriptor and load as zeros); returns the absent halves
  auto load = [&](const bf16* pool, char* to, int it, auto sw) __attribute__((always_inline)) {
    int absent = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int key = k0 + it * TK + 16 * h, page = walk.at(key >> a.lg);
      const int n = page < 0 ? 0 : min(max(end - key, 0), 16);
      const long at = (((long)max(page, 0) * a.hkv + hk) << a.lg) + (key & ((1 << a.lg) - 1));
      const auto rs = make_rsrc_uniform(pool + at * D, n * D * 2);
      absent |= (page < 0) << h;
#pragma unroll
      for (int i = h * NLD / 2; i < (h + 1) * NLD / 2; ++i)
        dma16(rs, to + i * 1024, swz<decltype(sw)::value, D>(i * 64 + lane) * 16 - h * 16 * D * 2, 0);
    }
    return absent;
  };
  using RowSwz = std::integral_constant<Swz, SWZ_ROW>;
  using DualSwz = std::integral_constant<Swz, SWZ_DUAL>;
  char *kt = sm.u.tile[wave][0], *vt = sm.u.tile[wave][1];
  uint32_t pb[8];
  u32x4 va[2][Rows<D>::DT];
  int absent = 0;
  if (n_tiles > 0) {
    absent = load(kp, kt, 0, RowSwz{});
    load(vp, vt, 0, DualSwz{});
  }
  for (int it = 0; it < n_tiles; ++it) {
    // K of a tile before its V, each refilled as soon as it has been read
    __builtin_amdgcn_s_waitcnt(kVmWait<NLD>());
    f32x16 sc = st.scores(kt);
    __builtin_amdgcn_s_waitcnt(kLgkmcnt0);
    int next = 0;
    if (it + 1 < n_tiles) next = load(kp, kt, it + 1, RowSwz{});
    const int t0 = k0 + it * TK;
    const bool edge = t0 + TK > min(lim0, end);
    if (edge) st.mask(sc, min(lim, end) - t0);
    if (absent) {
#pragma unroll
      for (int x = 0; x < 16; ++x)
        if (absent >> (x >> 3) & 1) sc[x] = -INFINITY;
    }
    st.softmax(sc, sl2, pb);
    if (it + 1 < n_tiles) __builtin_amdgcn_s_waitcnt(kVmWait<NLD>());
    else __builtin_amdgcn_s_waitcnt(kVmcnt0);
    st.read_v(vt, va);
    __builtin_amdgcn_s_waitcnt(kLgkmcnt0);
    const bool bad = edge && lim0 < last && any_bad<Rows<D>::DT>(va);
    if (bad) {
      add_keys<D>(st.acc, vt, pb, min(lim, end) - t0);
      __builtin_amdgcn_s_waitcnt(kLgkmcnt0);
    }
    if (it + 1 < n_tiles) load(vp, vt, it + 1, DualSwz{});
    if (!bad) st.product(va, pb);
    absent = next;
  }
  const float l_tot = st.l + other_half(st.l);
  const int n_here = min(32, rows - rg * 32);
  __syncthreads();  // every wavefront is done with its tiles
  if (l32 < n_here) {
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
  for (int i = tid; i < n_here * (D / 4); i += NW * 64) {
    const int rr = i / (D / 4), d = (i - rr * (D / 4)) * 4;
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) mm = fmaxf(mm, sm.u.c.m[w][rr]);
    const float ref = mm == -INFINITY ? 0.0f : mm;
    f32x4 num = {};
    float den = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float e = fast_exp2(sm.u.c.m[w][rr] - ref);
      num += e * *reinterpret_cast<const f32x4*>(sm.u.c.o[w] + rr * D + d);
      den += e * sm.u.c.l[w][rr];
    }
    const int ri = rg * 32 + rr, ti = ri / G;
    const long to = (long)(s.t0 + ti) * a.hq + hk * G + (ri - ti * G);
    if (n_sh == 1) {
      const float inv = den == 0.0f ? 0.0f : 1.0f / den;  // a row without a key: zeros
      *reinterpret_cast<u32x2*>(o + to * D + d) =
          u32x2{pack_bf16x2(num[0] * inv, num[1] * inv), pack_bf16x2(num[2] * inv, num[3] * inv)};
      continue;
    }
    const long at = few_row(a, pl, split, b, hk, ri, to);
    *reinterpret_cast<f32x4*>(out.o + at * D + d) = num;
    if (d == 0) {
      out.m[at] = mm;
      out.l[at] = den;
    }
  }
}

// ---------------------------------------------------------------------------
// fp32: a wavefront per 16 rows and share, on the fp32 matrix cores, K and V read
// straight from the pages in operand order.  The same grid, groups of 16 rows.  Bound by
// the latency of each 32 keys' loads (a wavefront's registers hold one such step; shares
// and groups bring the others): 4 sequences of 3 tokens behind 61, 4 heads of 64, 7.2 us.
// ---------------------------------------------------------------------------
template <int D>
__device__ void paged_attn_f32(const float* __restrict__ q, const float* __restrict__ kp,
                               const float* __restrict__ vp, float* __restrict__ o, const Paged a,
                               const PagedPlan pl, const PagedParts out) {
  constexpr int NC = Geo<D>::NC, VW = Geo<D>::VW, NH = Geo<D>::NH;
  const int lane = threadIdx.x, j = lane & 15, g = lane >> 4;
  int hk, id;
  if (!paged_place(a.hkv, pl.splits * pl.groups * a.batch, &hk, &id)) return;
  const int rg = pl.groups - 1 - id % pl.groups;  // the last rows, with the most keys, first
  id /= pl.groups;
  const int split = id % pl.splits, b = id / pl.splits;
  PageWalk walk(a, b);
  const Seq s = seq_of(a, b);
  const int G = a.hq / a.hkv;
  const long rows = (long)s.n * G;
  if (rows > pl.few || (long)rg * 16 >= rows) return;
  const int n_sh = paged_shares(s, pl.keys, pl.splits);
  if (split >= n_sh) return;
  const long rc = min((long)rg * 16 + j, rows - 1);
  const int tok = (int)(rc / G);
  const bool valid = (long)rg * 16 + j < rows;
  const long row = (long)(s.t0 + tok) * a.hq + hk * G + (int)(rc - (long)tok * G);
  const int last = s.keys((int)((min(rows, (long)rg * 16 + 16) - 1) / G));
  const int lim0 = s.keys((int)((long)rg * 16 / G));
  const int k0 = split * pl.keys, end = split + 1 < pl.splits ? min(k0 + pl.keys, last) : last;
  const int stop = min(s.keys(tok), end);
  f32x4 qf[NC];
  row_regs<D>(q + row * D, g, qf);
  f32x4 acc[NH][VW];
  zero_acc<D>(acc);
  float m = -INFINITY, l = 0.0f;
  for (int t0 = k0; t0 < end; t0 += 32) {
    f32x4 kf[2][NC];
    float vf[8][NH][VW];
    // 16 rows lie in one page; rows at or past the end re-read the last one before it
    // (where there is none, the pool's first): their P is zero, and so is their V
    long base[2];
    int n[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int key = t0 + 16 * u, page = walk.at(key >> a.lg);
      n[u] = page < 0 ? 0 : min(max(end - key, 0), 16);
      base[u] = n[u] == 0 ? 0 : (((long)page * a.hkv + hk) << a.lg) + (key & ((1 << a.lg) - 1));
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
      row_regs<D>(kp + (base[u] + max(0, min(j, n[u] - 1))) * D, g, kf[u]);
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const int u = x >> 2;
      const float* vr = vp + (base[u] + max(0, min(4 * g + (x & 3), n[u] - 1))) * D;
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        if constexpr (VW == 4) {
          const f32x4 y = *reinterpret_cast<const f32x4g*>(vr + 64 * h + 4 * j);
#pragma unroll
          for (int e = 0; e < 4; ++e) vf[x][h][e] = y[e];
        } else if constexpr (VW == 2) {
          const f32x2 y = *reinterpret_cast<const f32x2g*>(vr + 2 * j);
          vf[x][h][0] = y[0];
          vf[x][h][1] = y[1];
        } else {
          vf[x][h][0] = D == 8 && j >= 8 ? 0.0f : vr[j];
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);  // every load is issued first
    f32x4 sc[2] = {};
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int u = 0; u < 2; ++u) sc[u] = mfma4(kf[u][c][e], qf[c][e], sc[u]);
    float mx = -INFINITY;
    const float m_old = m;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const bool seen = t0 + 16 * u + 4 * g + r < stop && 4 * g + r < n[u];
        sc[u][r] = seen ? sc[u][r] * pl.scale : -INFINITY;
        mx = fmaxf(mx, sc[u][r]);
      }
    m = fmaxf(m, max_g(mx));
    const float ref = m == -INFINITY ? 0.0f : m;  // no key of the row so far
    const float alpha = expf(m_old - ref);
    l *= alpha;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        sc[u][r] = expf(sc[u][r] - ref);
        l += sc[u][r];
      }
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
      for (int e = 0; e < VW; ++e) acc[h][e] *= alpha;
    if (n[0] < 16 || n[1] < 16) {
#pragma unroll
      for (int x = 0; x < 8; ++x)
        if (4 * g + (x & 3) >= n[x >> 2])
#pragma unroll
          for (int h = 0; h < NH; ++h)
#pragma unroll
            for (int e = 0; e < VW; ++e) vf[x][h][e] = 0.0f;
    }
    // rows that some query of the 16 must not see: as add_keys
    if (lim0 < last && min(t0 + 32, end) > lim0) {
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
            const int in = 4 * kg + (x & 3);
            const float p = __shfl(sc[x >> 2][x & 3], 16 * kg + j);
            if (t0 + 16 * (x >> 2) + in < stop && in < n[x >> 2])
              add_row<D>(vp + (base[x >> 2] + in) * D, p, g, acc);
          }
        continue;
      }
    }
#pragma unroll
    for (int x = 0; x < 8; ++x)
#pragma unroll
      for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int e = 0; e < VW; ++e) acc[h][e] = mfma4(vf[x][h][e], sc[x >> 2][x & 3], acc[h][e]);
  }
  l = sum_g(l);
  if (!valid) return;
  if (n_sh == 1) {
    store_col<D>(o + row * D, acc, g, [l](float x) { return l == 0.0f ? 0.0f : x / l; });
    return;
  }
  const long to = few_row(a, pl, split, b, hk, (int)rc, row);
  if (g == 0) {
    out.m[to] = m * kLog2e;
    out.l[to] = l;
  }
  store_col<D>(out.o + to * D, acc, g, [](float x) { return x; });
}

// The shares of a row, weighed by 2^(m - max m) and summed: a wavefront a row, whose
// lanes hold four d each in groups that go over the shares side by side.  With a stride the
// rows are those kept for each (sequence, kv head), then (the sequences of many rows, where
// they have shares) those of all heads of all tokens; else the latter alone.
// Bound by the chain of its loads: 640 rows of 64 with 4 shares 4.0 us.
template <typename T>
__device__ void paged_merge(const PagedParts parts, T* __restrict__ o, const Paged a,
                            const PagedPlan pl, int lg_d) {
  const int lane = threadIdx.x & 63, G = a.hq / a.hkv;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long item = (long)blockIdx.x * 4 + wave, n_few = (long)a.batch * a.hkv * pl.stride;
  PagedParts in = parts;
  long row, first, step;  // the output row; the first share's partials, those to the next
  int n;
  if (item < n_few) {
    const int bh = (int)(item / pl.stride), r = (int)(item - (long)bh * pl.stride);
    const int b = bh / a.hkv, hk = bh - b * a.hkv;
    const Seq s = seq_of(a, b);
    const long rows = (long)s.n * G;
    if (r >= rows || rows > pl.few) return;
    n = paged_shares(s, pl.keys, pl.splits);
    row = (long)(s.t0 + r / G) * a.hq + hk * G + r % G;
    first = item;
    step = n_few;
  } else {
    row = item - n_few;
    step = (long)a.tokens * a.hq;
    if (row >= step) return;
    const int t = (int)(row / a.hq), b = seq_at(a, t);
    if (b < 0) return;
    const Seq s = seq_of(a, b);
    if (t < s.t0 || t >= s.t0 + s.n) return;
    const bool many = (long)s.n * G > pl.few;
    if (pl.stride > 0 && !many) return;
    n = many ? paged_shares(s, pl.keys_many, pl.splits_many) : paged_shares(s, pl.keys, pl.splits);
    first = row;
    if (many) in = PagedParts{in.m_many, in.l_many, in.o_many, nullptr, nullptr, nullptr};
  }
  if (n <= 1) return;
  float mx = -INFINITY;
  for (int i = lane; i < n; i += 64) mx = fmaxf(mx, in.m[first + i * step]);
  mx = wave_max(mx);
  const float ref = mx == -INFINITY ? 0.0f : mx;  // no key at all: zeros
  const int lanes = 1 << (lg_d - 2), grp = lane >> (lg_d - 2), groups = 64 >> (lg_d - 2);
  const int d = (lane & (lanes - 1)) * 4;
  f32x4 acc = {};
  float den = 0.0f;
  constexpr int U = 4;  // shares of a group in flight
  for (int i0 = grp; i0 - grp < n; i0 += U * groups) {
    f32x4 v[U];
    float mi[U], li[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {  // (past the end: the last one, unweighed)
      const long at = first + min(i0 + u * groups, n - 1) * step;
      v[u] = *reinterpret_cast<const f32x4*>(in.o + (at << lg_d) + d);
      mi[u] = in.m[at];
      li[u] = in.l[at];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i0 + u * groups >= n) continue;
      // (a share without a key has sums of zero; one whose scores are all NaN has no maximum
      // either, but NaN in its sums, which the row's are then)
      const float e = fast_exp2(mi[u] - ref);
      acc += e * v[u];
      den += e * li[u];
    }
  }
  for (int off = lanes; off < 64; off <<= 1) {
    den += __shfl_xor(den, off);
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] += __shfl_xor(acc[i], off);
  }
  if (grp > 0) return;
  const float inv = den == 0.0f ? 0.0f : 1.0f / den;
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i] *= inv;
  T* to = o + (row << lg_d) + d;
  if constexpr (sizeof(T) == 2)
    *reinterpret_cast<u32x2*>(to) = u32x2{pack_bf16x2(acc[0], acc[1]), pack_bf16x2(acc[2], acc[3])};
  else
    *reinterpret_cast<f32x4g*>(to) = acc;
}

}  // namespace

#define TEENY_PAGED_SPLIT_INST(TN, T)                                                            \
  extern "C" __global__ __launch_bounds__(256) void teeny_paged_split_##TN(                       \
      const T* qkv, T* q_out, T* kp, T* vp, Paged a, int lg_d, double ln_base) {                  \
    paged_split<T, false>(qkv, nullptr, 0, 0, q_out, kp, vp, a, lg_d, ln_base);                   \
  }
TEENY_PAGED_SPLIT_INST(bf16, bf16)
TEENY_PAGED_SPLIT_INST(f32, float)
#define TEENY_PAGED_SPLIT_PARTS_INST(TN, T)                                                      \
  extern "C" __global__ __launch_bounds__(256) void teeny_paged_split_parts_##TN(                 \
      const float* parts, int n_parts, long part_stride, T* q_out, T* kp, T* vp, Paged a,         \
      int lg_d, double ln_base) {                                                                 \
    paged_split<T, true>(nullptr, parts, n_parts, part_stride, q_out, kp, vp, a, lg_d, ln_base);  \
  }
TEENY_PAGED_SPLIT_PARTS_INST(bf16, bf16)
TEENY_PAGED_SPLIT_PARTS_INST(f32, float)

extern "C" __global__ __launch_bounds__(256) void teeny_copy_pages(char* pages, long plane_bytes,
                                                                    long page_bytes, int chunks,
                                                                    Moves m) {
  copy_pages(pages, plane_bytes, page_bytes, chunks, m);
}

#define TEENY_PAGED_ATTN_BF16_INST(D, NW)                                                        \
  extern "C" __global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(2)))       \
  void teeny_paged_attn_bf16_d##D##_w##NW(const bf16* q, const bf16* kp, const bf16* vp, bf16* o, \
                                          Paged a, PagedPlan pl, PagedParts p) {                           \
    paged_attn<D, NW>(q, kp, vp, o, a, pl, p);                                                   \
  }
TEENY_PAGED_ATTN_BF16_INST(64, 4)
TEENY_PAGED_ATTN_BF16_INST(64, 8)
TEENY_PAGED_ATTN_BF16_INST(128, 4)
TEENY_PAGED_ATTN_BF16_INST(128, 8)

#define TEENY_PAGED_ATTN_F32_INST(D)                                                             \
  extern "C" __global__ __launch_bounds__(64) void teeny_paged_attn_f32_d##D(                    \
      const float* q, const float* kp, const float* vp, float* o, Paged a, PagedPlan pl, PagedParts p) {    \
    paged_attn_f32<D>(q, kp, vp, o, a, pl, p);                                                   \
  }
TEENY_PAGED_ATTN_F32_INST(8)
TEENY_PAGED_ATTN_F32_INST(16)
TEENY_PAGED_ATTN_F32_INST(32)
TEENY_PAGED_ATTN_F32_INST(64)
TEENY_PAGED_ATTN_F32_INST(128)

#define TEENY_PAGED_MERGE_INST(TN, T)                                                            \
  extern "C" __global__ __launch_bounds__(256) void teeny_paged_merge_##TN(PagedParts p, T* o,         \
                                                           Paged a, PagedPlan pl, int lg_d) {   \
    paged_merge<T>(p, o, a, pl, lg_d);                                                           \
  }
TEENY_PAGED_MERGE_INST(bf16, bf16)
TEENY_PAGED_MERGE_INST(f32, float)
