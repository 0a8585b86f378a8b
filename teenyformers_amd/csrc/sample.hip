// Sampling a token per row of logits from given random numbers, with
// temperature, top-k, top-p and min-p.
//
// Reference: temperature sampling on the host (examples/llama_generate.rs:254-275):
// the softmax of logits / T, and the first index whose running sum exceeds the
// random number.  The filters have no counterpart there.
//
// A row's tokens in the order "higher logit first, lower index first among
// equal ones"; with w_i = 2^-d_i, d_i = (max x - x_i) log2(e) / T, each filter
// leaves a leading part of that order:
//   top-k   the first k;
//   top-p   of those, every token before which less than p of their weight lies;
//   min-p   tokens with w_i >= min_p.
// The draw walks the kept tokens in index order (as the reference does) to the
// first whose running weight exceeds u times the kept weight.
//
// Numbers: the border between two tokens among 1e5 is narrower than fp32 sums
// resolve, and sums of floats depend on their order.  So L = x log2(e) / T and
// 2^-d are evaluated in fp64 and a weight is held as a whole number of 2^-44
// (64 bits; at most 2^19 columns, so no sum overflows): sums are exact, in any
// order, with atomics too.  A weight that rounds to zero cannot be drawn.
// Weights are relative to the largest logit of the token's CHUNK (8192 columns)
// where chunks are summed alone, and a chunk's sum is brought to the row's
// scale by one fp64 factor, so one pass over the logits serves.
//
// Two launches:
//   scan   (chunk, row): one 16-byte load a thread (8 bf16; two for fp32), the
//          chunk's maximum, and its weight; with filters its weights and
//          counts by bins of d a quarter octave wide (192 LDS bins).
//   draw   (row): merges the chunks; without filters picks the chunk, and the
//          token in it.  With filters: finds the bin that a filter's border
//          lies in, collects that bin's tokens (in LDS, or by passing over the
//          row again where they are too many), narrows the border to one key
//          by a radix select of 1024 sub-bins, and to an index among equal
//          keys; then the kept weight of every chunk, the chunk, the token.
#include "common.h"

namespace {

typedef unsigned long long u64;

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kTok = 8;                   // tokens per thread and chunk
constexpr int kChunk = kThreads * kTok;   // columns per chunk
constexpr int kMaxChunks = 65;            // 2^19 columns and a misaligned start
constexpr int kBins = 180;                // quarter octaves below the row's maximum: 45 octaves
constexpr double kLog2e = 1.4426950408889634074;
constexpr int kFrac = 44;                 // fraction bits of a weight
constexpr int kList = 8192;               // tokens that a border's bin may hold in LDS

struct Chunk {
  double lref;  // L of the chunk's maximum
  u64 mass;     // sum of the chunk's weights (without filters)
  float xmax;   // the chunk's maximum; -inf: no token
  int pad[3];
};
static_assert(sizeof(Chunk) == 32, "the host sizes the workspace by it");

struct Settings {
  double c;       // log2(e) / T
  double p, lmin; // top-p; log2(min_p), -inf without
  int k;
  bool fk, fp, filters;
};

// One row's settings: a value for all rows, or a device array of one per row.
struct Args {
  double t, p, m;
  const float *ts, *ps, *ms;
  const int* ks;
  int k;
};

DEVI Settings settings(const Args& a, int row, int cols) {
  Settings s;
  const double t = a.ts ? (double)a.ts[row] : a.t;
  const double p = a.ps ? (double)a.ps[row] : a.p;
  const double m = a.ms ? (double)a.ms[row] : a.m;
  int k = a.ks ? a.ks[row] : a.k;
  const bool greedy = !(t > 0.0);  // the first of the order (NaN too)
  if (greedy) k = 1;
  s.c = greedy ? kLog2e : kLog2e / t;
  s.k = k;
  s.fk = k > 0 && k < cols;
  s.fp = p < 1.0 && !greedy;
  s.p = p > 0.0 ? p : 0.0;
  s.lmin = m > 0.0 && !greedy ? (m < 1.0 ? log2(m) : 0.0) : -INFINITY;
  s.filters = s.fk || s.fp || s.lmin > -INFINITY;
  return s;
}

// 2^-d for d in [0, 46): 2^-d = 2^i 2^f, f in [0, 1), and 2^f from the series
// of exp around f = 1/2 (eleven terms leave 2^-47 relative).
DEVI double exp2_neg(double d) {
  const double y = -d, i = floor(y);
  const double r = (y - i - 0.5) * 0.69314718055994530942;
  double s = 1.0 / 39916800.0;
  s = fma(s, r, 1.0 / 3628800.0);
  s = fma(s, r, 1.0 / 362880.0);
  s = fma(s, r, 1.0 / 40320.0);
  s = fma(s, r, 1.0 / 5040.0);
  s = fma(s, r, 1.0 / 720.0);
  s = fma(s, r, 1.0 / 120.0);
  s = fma(s, r, 1.0 / 24.0);
  s = fma(s, r, 1.0 / 6.0);
  s = fma(s, r, 0.5);
  s = fma(s, r, 1.0);
  s = fma(s, r, 1.0);
  return ldexp(s * 1.41421356237309504880, (int)i);
}
// The weight of a token d octaves below the reference; 0 for d >= 46 and NaN.
DEVI u64 weight(double d) {
  if (!(d < 46.0)) return 0;
  if (d == 0.0) return 1ull << kFrac;
  // adding 2^52 rounds to a whole number, which is then in the low bits
  const double w = exp2_neg(d) * (double)(1ull << kFrac) + 4503599627370496.0;
  return __builtin_bit_cast(u64, w) & ((1ull << 52) - 1);
}

// Order-preserving unsigned key of a logit (no NaN, no -0) and back.
DEVI uint32_t key_of(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
DEVI float of_key(uint32_t k) {
  return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// The logits of thread slot `slot` of chunk ch: columns col .. col + 7, those
// outside the row as -inf.  A chunk starts at a 16-byte aligned address, which
// may lie before the row (mis elements), so whole vectors load at once and only
// a row's two ends go one by one.  NaN becomes -inf (never drawn), -0 becomes 0
// (the two are equal logits).
template <typename T>
DEVI int load8(const T* row, int cols, int mis, int ch, int slot, float* x) {
  constexpr int VN = Vec16<T>::N;
  const int col = ch * kChunk + slot * kTok - mis;
  if (col >= 0 && col + kTok <= cols) {
#pragma unroll
    for (int j = 0; j < kTok; j += VN) Vec16<T>::load(row + col + j, x + j);
  } else {
#pragma unroll
    for (int j = 0; j < kTok; ++j)
      x[j] = col + j >= 0 && col + j < cols ? (float)row[col + j] : -INFINITY;
  }
#pragma unroll
  for (int j = 0; j < kTok; ++j) x[j] = x[j] == x[j] ? x[j] + 0.0f : -INFINITY;
  return col;
}
template <typename T> DEVI int misaligned(const T* row) {
  return (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
}

DEVI u64 shfl_up64(u64 v, int d) {
  const uint32_t lo = __shfl_up((uint32_t)v, d, 64), hi = __shfl_up((uint32_t)(v >> 32), d, 64);
  return (u64)hi << 32 | lo;
}
DEVI u64 wave_scan(u64 v) {  // inclusive
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const u64 o = shfl_up64(v, d);
    if (lane >= d) v += o;
  }
  return v;
}
// Exclusive prefix sum over the workgroup; total in *total.  tmp: kWaves words
// of LDS that no earlier phase still reads.
DEVI u64 block_scan(u64 v, u64* tmp, u64* total) {
  const int wave = threadIdx.x >> 6;
  const u64 inc = wave_scan(v);
  if ((threadIdx.x & 63) == 63) tmp[wave] = inc;
  __syncthreads();
  u64 base = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const u64 t = tmp[w];
    base += w < wave ? t : 0;
    all += t;
  }
  __syncthreads();
  *total = all;
  return base + inc - v;
}

// ---------------------------------------------------------------------------
// scan: grid (chunks, rows)
// ---------------------------------------------------------------------------
template <typename T>
__device__ void sample_scan(const T* __restrict__ logits, long ld, int cols, const Args a,
                            Chunk* __restrict__ rec, uint32_t* __restrict__ cnt,
                            u64* __restrict__ mass) {
  __shared__ uint32_t h_cnt[kBins];
  __shared__ u64 h_mass[kBins];
  __shared__ float red[kWaves];
  __shared__ u64 sums[kWaves];
  const int tid = threadIdx.x, ch = blockIdx.x, row_i = blockIdx.y;
  const long slot = (long)row_i * gridDim.x + ch;
  const T* row = logits + row_i * ld;
  float x[kTok];
  load8(row, cols, misaligned(row), ch, tid, x);
  const Settings s = settings(a, row_i, cols);
  if (s.filters && tid < kBins) {
    h_cnt[tid] = 0;
    h_mass[tid] = 0;
  }
  float mx = x[0];
#pragma unroll
  for (int j = 1; j < kTok; ++j) mx = fmaxf(mx, x[j]);
  mx = wave_max(mx);
  if ((tid & 63) == 0) red[tid >> 6] = mx;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) mx = fmaxf(mx, red[w]);
  const double lref = (double)mx * s.c;
  if (!s.filters) {
    u64 sum = 0;
#pragma unroll
    for (int j = 0; j < kTok; ++j)
      if (x[j] > -INFINITY) sum += weight(x[j] == mx ? 0.0 : lref - (double)x[j] * s.c);
    const u64 inc = wave_scan(sum);
    if ((tid & 63) == 63) sums[tid >> 6] = inc;
    __syncthreads();
    if (tid == 0) {
      u64 all = 0;
      for (int w = 0; w < kWaves; ++w) all += sums[w];
      rec[slot] = Chunk{lref, all, mx, {}};
    }
    return;
  }
  const double bmax = floor(4.0 * lref);
#pragma unroll
  for (int j = 0; j < kTok; ++j) {
    if (!(x[j] > -INFINITY)) continue;
    const double l = (double)x[j] * s.c;
    const bool top = x[j] == mx;
    const double r = top ? 0.0 : bmax - floor(4.0 * l);
    if (r < (double)kBins) {  // false for NaN
      atomicAdd(&h_cnt[(int)r], 1u);
      atomicAdd(&h_mass[(int)r], weight(top ? 0.0 : lref - l));
    }
  }
  __syncthreads();
  if (tid < kBins) {
    cnt[slot * kBins + tid] = h_cnt[tid];
    mass[slot * kBins + tid] = h_mass[tid];
  }
  if (tid == 0) rec[slot] = Chunk{lref, 0, mx, {}};
}

// ---------------------------------------------------------------------------
// draw: grid (rows)
// ---------------------------------------------------------------------------
struct DrawSmem {
  u64 list[kList];              // key << 32 | column of the collected tokens
  u64 sub_mass[kThreads];       // radix select: weight and count by sub-bin
  uint32_t sub_cnt[kThreads];
  u64 mass[kBins];              // the row's bins
  uint32_t cnt[kBins];
  double f[kMaxChunks];         // chunk scale -> row scale; 0: the chunk does not count
  double lref[kMaxChunks];
  float xmax[kMaxChunks];
  int off[kMaxChunks];          // bins that the chunk's maximum lies below the row's
  u64 kept[kMaxChunks];         // kept weight of a chunk, in its own scale
  uint32_t tie[kMaxChunks];
  u64 tmp[kWaves];
  uint32_t n_list, kmin, kmax;
  u64 a, b;                     // a value that one thread hands to all
  int i, j;
};

template <typename T>
__device__ void sample_draw(const T* __restrict__ logits, long ld, int cols, const Args a,
                            const float* __restrict__ us, const Chunk* __restrict__ rec,
                            const uint32_t* __restrict__ cnt, const u64* __restrict__ mass,
                            int n_ch, long long* __restrict__ out, int* __restrict__ advance) {
  __shared__ DrawSmem sm;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row_i = blockIdx.x;
  if (advance && row_i == 0 && tid == 0) *advance += 1;
  const T* row = logits + row_i * ld;
  const int mis = misaligned(row);
  const Settings s = settings(a, row_i, cols);
  const double c = s.c;
  rec += (long)row_i * n_ch;
  cnt += (long)row_i * n_ch * kBins;
  mass += (long)row_i * n_ch * kBins;

  // ---- the row's maximum, and each chunk's place below it -------------------
  float xr = -INFINITY;
  for (int i = 0; i < n_ch; ++i) xr = fmaxf(xr, rec[i].xmax);
  if (xr == -INFINITY) {  // no token left to draw
    if (tid == 0) out[row_i] = -1;
    return;
  }
  const double lrow = (double)xr * c, brow = floor(4.0 * lrow);
  if (tid < n_ch) {
    const Chunk r = rec[tid];
    const double d = r.xmax == xr ? 0.0 : lrow - r.lref;
    const bool in = r.xmax > -INFINITY && d < 46.0;
    sm.f[tid] = in ? (d == 0.0 ? 1.0 : exp2_neg(d)) : 0.0;
    sm.off[tid] = in && d != 0.0 ? (int)(brow - floor(4.0 * r.lref)) : 0;
    sm.lref[tid] = r.lref;
    sm.xmax[tid] = r.xmax;
    sm.kept[tid] = r.mass;
  }
  __syncthreads();

  // A token's bin below the row's maximum; kBins or more: it does not count.
  auto bin_of = [&](float x) {
    if (x == xr) return 0;
    const double r = brow - floor(4.0 * ((double)x * c));
    return r < (double)kBins ? (int)r : kBins;
  };
  auto row_weight = [&](float x) { return weight(x == xr ? 0.0 : lrow - (double)x * c); };
  auto chunk_weight = [&](int ch, float x) {
    return weight(x == sm.xmax[ch] ? 0.0 : sm.lref[ch] - (double)x * c);
  };

  // the border that top-k and top-p leave: tokens with a higher key, or the same
  // key and a column up to cut_col; jc: its bin (kBins: no border)
  uint32_t cut_key = 0;
  int cut_col = 0x7fffffff, jc = kBins;
  const double lmin = lrow + s.lmin;  // min-p in terms of L
  auto keeps = [&](float x, int col) {
    const uint32_t key = key_of(x);
    return (key > cut_key || (key == cut_key && col <= cut_col)) &&
           (x == xr || (double)x * c >= lmin || s.lmin == -INFINITY);
  };

  if (s.filters) {
    // ---- the row's bins ------------------------------------------------------
    if (tid < kBins) {
      uint32_t n = 0;
      u64 m = 0;
      for (int ch = 0; ch < n_ch; ++ch) {
        const int r = tid - sm.off[ch];
        const double f = sm.f[ch];
        if (f > 0.0 && r >= 0) {
          n += cnt[ch * kBins + r];
          const u64 v = mass[ch * kBins + r];
          m += f == 1.0 ? v : (u64)((double)v * f + 0.5);
        }
      }
      sm.cnt[tid] = n;
      sm.mass[tid] = m;
    }
    __syncthreads();
    // exclusive prefix sums over the bins, in registers of threads 0 .. kBins-1
    u64 total_n, total_m;
    const u64 n_here = tid < kBins ? sm.cnt[tid] : 0, m_here = tid < kBins ? sm.mass[tid] : 0;
    const u64 n_before = block_scan(n_here, sm.tmp, &total_n);
    const u64 m_before = block_scan(m_here, sm.tmp, &total_m);

    int list_lo = 1, list_hi = 0;  // the bins whose tokens the list holds
    // f(x, column) for every token of bins lo .. hi, from the list or the row
    auto each = [&](int lo, int hi, auto&& f) {
      if (lo >= list_lo && hi <= list_hi) {
        const int n = sm.n_list;
        for (int i = tid; i < n; i += kThreads) {
          const u64 e = sm.list[i];
          const float x = of_key((uint32_t)(e >> 32));
          const int b = bin_of(x);
          if (b >= lo && b <= hi) f(x, (int)(uint32_t)e);
        }
        return;
      }
      for (int ch = wave; ch < n_ch; ch += kWaves) {  // a wavefront takes whole chunks
        if (!(sm.f[ch] > 0.0) || sm.off[ch] > hi) continue;
        for (int it = 0; it < kThreads / 64; ++it) {
          float x[kTok];
          const int col = load8(row, cols, mis, ch, it * 64 + lane, x);
#pragma unroll
          for (int j = 0; j < kTok; ++j)
            if (x[j] > -INFINITY) {
              const int b = bin_of(x[j]);
              if (b >= lo && b <= hi) f(x[j], col + j);
            }
        }
      }
    };
    // collects the tokens of bins lo .. hi, n of them, in LDS if they fit
    auto collect = [&](int lo, int hi, u64 n) {
      if ((lo >= list_lo && hi <= list_hi) || n > (u64)kList) return;
      __syncthreads();
      if (tid == 0) sm.n_list = 0;
      __syncthreads();
      list_lo = 1;
      list_hi = 0;  // read from the row
      each(lo, hi, [&](float x, int col) {
        const uint32_t at = atomicAdd(&sm.n_list, 1u);
        sm.list[at & (kList - 1)] = (u64)key_of(x) << 32 | (uint32_t)col;
      });
      __syncthreads();
      list_lo = lo;
      list_hi = hi;
    };
    // The border in bin j: the token at which the running count (BY_COUNT) or
    // weight of the bin's tokens, in the order, reaches need.  Sets the cut.
    auto border = [&](int j, u64 need, bool by_count) {
      __syncthreads();
      if (tid == 0) {
        sm.kmin = 0xffffffffu;
        sm.kmax = 0;
      }
      __syncthreads();
      each(j, j, [&](float x, int) {
        atomicMin(&sm.kmin, key_of(x));
        atomicMax(&sm.kmax, key_of(x));
      });
      __syncthreads();
      uint32_t k0 = sm.kmin, k1 = sm.kmax;
      u64 ties = 0;
      do {
        const uint32_t span = k1 - k0;
        const int sh = span < (uint32_t)kThreads ? 0 : 22 - __builtin_clz(span);
        sm.sub_mass[tid] = 0;
        sm.sub_cnt[tid] = 0;
        __syncthreads();
        each(j, j, [&](float x, int) {
          const uint32_t k = key_of(x);
          if (k >= k0 && k <= k1) {
            atomicAdd(&sm.sub_cnt[(k1 - k) >> sh], 1u);
            if (!by_count) atomicAdd(&sm.sub_mass[(k1 - k) >> sh], row_weight(x));
          }
        });
        __syncthreads();
        const u64 n = sm.sub_cnt[tid], v = by_count ? n : sm.sub_mass[tid];
        u64 all;
        const u64 before = block_scan(v, sm.tmp, &all);
        if (need > all) need = all;  // the merged bin's sum was rounded up
        if (need == 0) break;        // every weight here rounds to zero: all are kept
        if (v > 0 && before < need && need <= before + v) {
          sm.i = tid;
          sm.a = need - before;
          sm.b = n;
        }
        __syncthreads();
        const uint32_t sub = sm.i;
        need = sm.a;
        ties = sm.b;
        __syncthreads();
        const uint32_t top = k1 - (sub << sh);
        k0 = top - k0 < (1u << sh) ? k0 : top - (1u << sh) + 1;
        k1 = top;
      } while (k0 < k1);
      cut_key = k0;
      cut_col = 0x7fffffff;
      jc = j;
      if (need == 0) return;
      const float x = of_key(k0);
      if (!by_count) {  // as many of the equal tokens as their weight needs
        const u64 w = row_weight(x);
        need = (need + w - 1) / w;
      }
      if (need >= ties) return;
      // the column of the need-th of the equal tokens: its chunk, then in it
      if (tid < kMaxChunks) sm.tie[tid] = 0;
      __syncthreads();
      each(j, j, [&](float y, int col) {
        if (key_of(y) == k0) atomicAdd(&sm.tie[(col + mis) / kChunk], 1u);
      });
      __syncthreads();
      if (tid == 0) {
        u64 left = need;
        int ch = 0;
        while (ch < n_ch - 1 && left > sm.tie[ch]) left -= sm.tie[ch++];
        sm.i = ch;
        sm.a = left;
      }
      __syncthreads();
      float y[kTok];
      const int col = load8(row, cols, mis, sm.i, tid, y);
      const u64 left = sm.a;
      u64 here = 0, all;
#pragma unroll
      for (int t = 0; t < kTok; ++t) here += y[t] == x;
      const u64 before = block_scan(here, sm.tmp, &all);
      if (before < left && left <= before + here) {
        u64 n = before;
#pragma unroll
        for (int t = 0; t < kTok; ++t)
          if (y[t] == x && ++n == left) sm.j = col + t;
      }
      __syncthreads();
      cut_col = sm.j;
    };
    // the bin at which a running sum over the bins reaches need (thread j holds
    // bin j's sum and what lies before it); what is needed within the bin, and
    // what it holds, in sm.a and sm.b
    auto find_bin = [&](u64 before, u64 here, u64 need) {
      __syncthreads();
      if (here > 0 && before < need && need <= before + here) {
        sm.i = tid;
        sm.a = need - before;
      }
      __syncthreads();
      return sm.i;
    };

    u64 m_left = total_m;  // the weight that top-k leaves
    if (s.fk && (u64)s.k < total_n) {
      const int jk = find_bin(n_before, n_here, (u64)s.k);
      const u64 need = sm.a;
      __syncthreads();
      if (tid == jk) {
        sm.b = n_before + n_here;
        sm.a = m_before;
      }
      __syncthreads();
      const u64 up_to = sm.b, above = sm.a;
      // every token up to the border's bin where that is few, else the bin's
      collect(up_to <= (u64)kList ? 0 : jk, jk, up_to <= (u64)kList ? up_to : sm.cnt[jk]);
      border(jk, need, true);
      if (s.fp) {
        u64 mine = 0, part;
        each(jk, jk, [&](float x, int col) {
          const uint32_t key = key_of(x);
          if (key > cut_key || (key == cut_key && col <= cut_col)) mine += row_weight(x);
        });
        block_scan(mine, sm.tmp, &part);
        m_left = above + part;
      }
    }
    if (s.fp) {
      u64 need = (u64)ceil(s.p * (double)m_left);
      need = max(1ull, min(need, min(m_left, total_m)));
      // (bins past top-k's border hold weight too, but the need is met before)
      const int jp = find_bin(m_before, m_here, need);
      const u64 in_bin = sm.a;
      const uint32_t old_key = cut_key;
      const int old_col = cut_col, old_bin = jc;
      collect(jp, jp, sm.cnt[jp]);
      border(jp, in_bin, false);
      // never past top-k's border (the sums around it are rounded)
      if (old_bin < kBins && (cut_key < old_key || (cut_key == old_key && cut_col > old_col))) {
        cut_key = old_key;
        cut_col = old_col;
        jc = old_bin;
      }
    }
    if (s.lmin > -INFINITY) {
      const double r = brow - floor(4.0 * lmin);
      jc = min(jc, r < (double)kBins ? (int)r : kBins);
    }
    // ---- each chunk's kept weight: whole bins, and the border's bin ----------
    __syncthreads();
    const int whole = jc;  // bins 0 .. whole - 1 are kept
    for (int ch = wave; ch < n_ch; ch += kWaves) {
      u64 v = 0;
      if (sm.f[ch] > 0.0)
        for (int r = lane; r < whole - sm.off[ch]; r += 64) v += mass[ch * kBins + r];
      v = wave_scan(v);
      if (lane == 63) sm.kept[ch] = v;
    }
    __syncthreads();
    if (jc < kBins)
      each(jc, jc, [&](float x, int col) {
        if (keeps(x, col)) {
          const int ch = (col + mis) / kChunk;
          atomicAdd(&sm.kept[ch], chunk_weight(ch, x));
        }
      });
    __syncthreads();
  }

  // ---- the chunk that u falls into -------------------------------------------
  if (tid == 0) {
    u64 total = 0;
    for (int ch = 0; ch < n_ch; ++ch)
      total += (u64)((double)sm.kept[ch] * sm.f[ch] + 0.5);
    const double u = (double)us[row_i];
    const double at = (u > 0.0 ? u : 0.0) * (double)total;
    u64 t = at < (double)total ? (u64)at : total;
    if (t >= total) t = total - 1;
    int pick = -1;
    u64 rest = 0;
    for (int ch = 0; ch < n_ch; ++ch) {
      const u64 w = (u64)((double)sm.kept[ch] * sm.f[ch] + 0.5);
      if (w == 0) continue;
      pick = ch;
      if (t < w) {
        rest = (u64)((double)t / sm.f[ch]);  // in the chunk's scale
        break;
      }
      t -= w;
    }
    if (rest >= sm.kept[pick]) rest = sm.kept[pick] - 1;
    sm.i = pick;
    sm.a = rest;
  }
  __syncthreads();
  // ---- the token in it ---------------------------------------------------------
  const int ch = sm.i;
  const u64 target = sm.a;
  float x[kTok];
  const int col = load8(row, cols, mis, ch, tid, x);
  u64 w[kTok], mine = 0, all;
#pragma unroll
  for (int j = 0; j < kTok; ++j) {
    const bool in = x[j] > -INFINITY && (!s.filters || (bin_of(x[j]) < kBins && keeps(x[j], col + j)));
    w[j] = in ? chunk_weight(ch, x[j]) : 0;
    mine += w[j];
  }
  u64 before = block_scan(mine, sm.tmp, &all);
  if (before <= target && target < before + mine) {
    int at = 0;
#pragma unroll
    for (int j = kTok - 1; j >= 0; --j) {  // the first whose running weight exceeds target
      u64 run = before;
#pragma unroll
      for (int t = 0; t <= j; ++t) run += w[t];
      if (run > target) at = col + j;
    }
    out[row_i] = at;
  }
}

}  // namespace

#define TEENY_SAMPLE_INST(TN, T)                                                                  \
  extern "C" __global__ __launch_bounds__(1024) void teeny_sample_scan_##TN(                     \
      const T* logits, long ld, int cols, Args a, Chunk* rec, uint32_t* cnt, u64* mass) {         \
    sample_scan<T>(logits, ld, cols, a, rec, cnt, mass);                                          \
  }                                                                                               \
  extern "C" __global__ __launch_bounds__(1024) void teeny_sample_draw_##TN(                     \
      const T* logits, long ld, int cols, Args a, const float* u, const Chunk* rec,               \
      const uint32_t* cnt, const u64* mass, int n_ch, long long* out, int* advance) {             \
    sample_draw<T>(logits, ld, cols, a, u, rec, cnt, mass, n_ch, out, advance);                   \
  }
TEENY_SAMPLE_INST(f32, float)
TEENY_SAMPLE_INST(bf16, bf16)
