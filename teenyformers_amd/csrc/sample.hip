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
// resolve, and sums of floats depend on their order.  So q = 4 x log2(e) / T (a
// token's place in quarter octaves) and 2^(q/4) are evaluated in fp64, and a
// weight is held as a whole number of 2^-44 of a reference (64 bits; at most
// 524280 columns, so no sum overflows): sums are exact, in any order, with
// atomics too.  A weight that rounds to zero cannot be drawn.
//   With filters, floor(q) is a token's bin and 2^(frac(q)/4), of one scale in
// every bin of the row, its weight there: bins are summed over chunks as they
// are and scaled once, to 2^-44 of the row's largest.  Without, the reference is the
// largest logit of the token's CHUNK (8192 columns), and a chunk's sum is brought to
// the row's scale by one fp64 factor.  Either way one pass over the logits serves.
//
// Two launches, because a border needs the whole row's bins and one workgroup a row
// would leave the device to a few rows:
//   scan   (chunk, row): 16-byte loads of 8 tokens (fp32: two), one or two a thread.
//          The chunk's maximum, and its weight by 512 columns.  With filters: its
//          tokens weighed and counted by bins below the chunk's maximum, in LDS,
//          and the tokens of its first bins, up to 1024, written out bin by bin,
//          so that the draw reads those alone.  A small top-k needs no more
//          than the chunk's own first k and no weight: the largest token of each
//          vector of 8 says from which bin on none of them lies, and a wavefront
//          goes over the others only (16 rows 7.1 -> 5.5 us).
//   draw   (row): 512 threads.  Without filters picks the chunk, the 512 columns
//          and the token.  With a small top-k: everything that the chunks wrote
//          out, in LDS.  Else: merges the chunks' bins, finds the bin that a
//          filter's border lies in, and collects that bin's tokens.  The border
//          is narrowed to one key by a radix select of 1024 sub-bins, and to an
//          index among equal keys; then the kept weight of every chunk, the
//          chunk, 64 columns of it, the token.  What does not fit (a bin with
//          thousands of tokens) is counted by chunk and key where the bin has few
//          keys (bf16: 512 mixed rows 184 -> 78 us), else read from the row again.
//
// Measured, bf16 x 128256, us of scan and draw: 1 row without filters 6.0, 4.2; 16
// with top-k 50 and top-p 5.6, 11; 64 with top-p 17, 14; 512 of mixed settings 82,
// 75; fp32, 24 x 32001 with min-p 5.5, 9.5.  Few rows are bound by their chains
// (load, maximum, weights, borders), a workgroup each.  Rows by the hundred are bound
// in the scan by vector instructions (57 a token and wavefront with top-p) and by
// workgroups that wait for their loads: 512 rows are read at 1.6 TB/s (temperature
// alone: a call 106 us, an fp64 exponential of 12 steps a token).  Their draws
// (a workgroup a CU: 200 registers; in 128 the compiler spills, and 64 rows took 25
// us) take the time of the rows with the fullest border bins.  A call with top-p 0.9
// whose border bin holds 4300 tokens takes 69 us for one row (fp32 182, passes alone),
// with 8400 of more keys than are counted 203 (fp32 248); with top-p 0.95 and a bin
// that fits 19.5.
#include "common.h"

#include <type_traits>

namespace {

typedef unsigned long long u64;

constexpr int kTok = 8;                   // tokens of a thread's vector
constexpr int kChunk = 8192;              // columns per chunk
constexpr int kSlots = kChunk / kTok;     // vectors of a chunk
constexpr int kParts = kSlots / 64;       // parts of 512 columns: a wavefront's vectors
constexpr int kMaxChunks = 64;            // a lane each
constexpr int kBins = 180;                // quarter octaves below the row's maximum: 45 octaves
constexpr int kFirstBins = 48;            // of them those that are counted first: 12 octaves
constexpr int kCand = 1024;               // tokens that a chunk writes out
constexpr int kSmallK = 512;              // a top-k that the chunk's own first k settle ...
constexpr int kFewTokens = 3200;          // ... k times the chunks
constexpr double kLog2e = 1.4426950408889634074;
constexpr int kFrac = 44;                 // fraction bits of a weight
constexpr u64 kLow52 = (1ull << 52) - 1;

struct Chunk {
  double lref;   // without filters: log2 weight of the chunk's maximum
  u64 mass;      // ... and the sum of the chunk's weights below it
  float xmax;    // the chunk's maximum; -inf: no token
  int last;      // with filters: the last bin whose tokens are written out
  int n_out;     // ... how many they are
  int complete;  // ... and whether a small top-k needs no other
};
static_assert(sizeof(Chunk) == 32, "the host sizes the workspace by it");
struct Bins {
  u64 mass[kBins];           // weights by bin; without filters by 512 columns
  u64 list[kCand];           // key << 32 | column, bin by bin
  uint32_t first[kBins + 4]; // tokens before each bin (of those counted)
};
static_assert(sizeof(Bins) == 8 * kBins + 8 * kCand + 4 * (kBins + 4), "as the host has it");

struct Settings {
  double c;        // log2(e) / T
  double p, lmin;  // top-p; log2(min_p), -inf without
  int k;
  bool fk, fp, filters;
  bool few;        // a small top-k: the chunks' first tokens alone
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
  // Small: up to kSmallK, and the draw's list takes the first k of all chunks and the
  // rest of the bin that completes each chunk's.  us by this way and by bins, bf16 (fp32)
  // x 128256, 16 chunks: 16 rows with k = 50 14.7, 21.9 (16.6, 22.8), 165 19.7, 22.1, 200
  // 20.5, 22.4 (22.6, 24.3); 64 rows with 200 26.7, 32.9; 16 x 32001 with 512 22.9, 19.9.
  // Where they do not fit this way passes over the row: with 225 and more of 16 chunks
  // 172, by bins 22.6.
  s.few = s.fk && k <= kSmallK && k * ((cols + 7 + kChunk - 1) / kChunk) <= kFewTokens;
  return s;
}

// 2^-d for d in [0, 46): 2^-d = 2^i 2^f, f in [0, 1), and 2^f from the series
// of exp around f = 1/2 (terms to the eleventh leave 2^-47 relative).
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
  return __builtin_bit_cast(u64, w) & kLow52;
}
// The weight of a token within its bin, 2^((f - 1) / 4) for f = frac(q), from the
// series around f = 1/2: |t ln 2 / 4| < 0.087, terms to the eighth leave 2^-50.
// (The last sum is at 2^52, which rounds it to a whole number.)
constexpr double kLn2Q = 0.69314718055994530942 / 4;
constexpr double kC0 = 17592186044416.0 * 0.91700404320467123175;  // 2^(44 - 1/8)
constexpr double kC1 = kC0 * kLn2Q, kC2 = kC1 * kLn2Q / 2, kC3 = kC2 * kLn2Q / 3,
                 kC4 = kC3 * kLn2Q / 4, kC5 = kC4 * kLn2Q / 5, kC6 = kC5 * kLn2Q / 6,
                 kC7 = kC6 * kLn2Q / 7, kC8 = kC7 * kLn2Q / 8;
struct Series {
  double c0 = kC0 + 4503599627370496.0, c1 = kC1, c2 = kC2, c3 = kC3, c4 = kC4, c5 = kC5,
         c6 = kC6, c7 = kC7;
  // As literals the compiler writes each into a vector register pair before its
  // step, two more instructions a step; the scan, which its vector instructions
  // bound (at 64 rows of 128256 77% of the issue slots), holds them in scalar
  // registers: 19.3 -> 18.5 us there, with 16 wavefronts a workgroup.
  DEVI void hold() {
    asm("" : "+s"(c0), "+s"(c1), "+s"(c2), "+s"(c3), "+s"(c4), "+s"(c5), "+s"(c6), "+s"(c7));
  }
};
DEVI u64 bin_weight(double f, const Series& c) {
  const double t = f - 0.5;
  double s = fma(kC8, t, c.c7);
  s = fma(s, t, c.c6);
  s = fma(s, t, c.c5);
  s = fma(s, t, c.c4);
  s = fma(s, t, c.c3);
  s = fma(s, t, c.c2);
  s = fma(s, t, c.c1);
  return __builtin_bit_cast(u64, fma(s, t, c.c0)) & kLow52;
}
// A token's bin below that of xmax (kBins: it does not count) and its weight in
// it.  q4 = 4 c.  (Compiled without contraction: x q4 - floor(x q4) with the
// product unrounded has no place in [0, 1) where logits are masked with -1e38,
// and gave equal logits other weights in one place than in another.)
// The largest token is in bin 0 also where its q is not finite (+inf; 0 * inf), and
// then alone with its equals.
DEVI int bin_of(float x, float xmax, double q4, u64* w, const Series& c = Series()) {
  const double top = floor((double)xmax * q4), q = (double)x * q4, fl = floor(q);
  const double r = top - fl;
  const bool fin = fabs(top) < INFINITY;
  *w = bin_weight(fin ? q - fl : 0.5, c);
  const int b = x == xmax ? 0 : fin && r < (double)kBins ? (int)r : kBins;
  return x > -INFINITY ? b : kBins;
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
  for (int j = 0; j < kTok; ++j) x[j] = fmaxf(x[j] + 0.0f, -INFINITY);
  return col;
}
// x[j] of a vector in registers
DEVI float nth_of(const float* x, int j) {
  const float a0 = j & 1 ? x[1] : x[0], a1 = j & 1 ? x[3] : x[2];
  const float a2 = j & 1 ? x[5] : x[4], a3 = j & 1 ? x[7] : x[6];
  const float b0 = j & 2 ? a1 : a0, b1 = j & 2 ? a3 : a2;
  return j & 4 ? b1 : b0;
}
template <typename T> DEVI int misaligned(const T* row) {
  return (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
}

// Wavefront sums through DPP (every lane active): within rows of 16 lanes, then
// lane 15 of a row into the next, then lane 31 into the upper half.
template <int CTRL, int ROWS> DEVI uint32_t dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS> DEVI u64 dpp(u64 v) {
  return (u64)dpp<CTRL, ROWS>((uint32_t)(v >> 32)) << 32 | dpp<CTRL, ROWS>((uint32_t)v);
}
template <typename V> DEVI V wave_scan(V v) {  // inclusive
  v += dpp<0x111, 0xf>(v);  // row_shr:1
  v += dpp<0x112, 0xf>(v);
  v += dpp<0x114, 0xf>(v);
  v += dpp<0x118, 0xf>(v);
  v += dpp<0x142, 0xa>(v);  // row_bcast:15
  v += dpp<0x143, 0xc>(v);  // row_bcast:31
  return v;
}
DEVI uint32_t lane_value(uint32_t v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
DEVI u64 lane_value(u64 v, int lane) {
  return (u64)lane_value((uint32_t)(v >> 32), lane) << 32 | lane_value((uint32_t)v, lane);
}
DEVI uint32_t wave_max_u32(uint32_t v) {
  v = max(v, dpp<0x111, 0xf>(v));
  v = max(v, dpp<0x112, 0xf>(v));
  v = max(v, dpp<0x114, 0xf>(v));
  v = max(v, dpp<0x118, 0xf>(v));
  v = max(v, dpp<0x142, 0xa>(v));
  v = max(v, dpp<0x143, 0xc>(v));
  return lane_value(v, 63);
}
template <typename V> DEVI V wave_total(V v) { return lane_value(wave_scan(v), 63); }

// ---------------------------------------------------------------------------
// scan: grid (chunks, rows)
// ---------------------------------------------------------------------------
template <int VEC> struct ScanSmem {
  u64 mass[kBins];
  uint32_t cnt[192];
  uint32_t tops[192];   // threads whose largest token is in each bin
  uint32_t first[192];  // tokens before each bin
  float red[kParts / VEC];
  u64 sums[kParts];
  int last;
};

// VEC: vectors of 8 tokens a thread.
template <typename T, int VEC>
__device__ void sample_scan(const T* __restrict__ logits, long ld, int cols, const Args a,
                            Chunk* __restrict__ rec, Bins* __restrict__ bins) {
  constexpr int kScan = kSlots / VEC, kScanWaves = kScan / 64;
  __shared__ ScanSmem<VEC> sm;
  const int tid = threadIdx.x, lane = tid & 63, ch = blockIdx.x, row_i = blockIdx.y;
  const long slot = (long)row_i * gridDim.x + ch;
  const T* row = logits + row_i * ld;
  float x[VEC][kTok];
  int col[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v)
    col[v] = load8(row, cols, misaligned(row), ch, v * kScan + tid, x[v]);
  const Settings s = settings(a, row_i, cols);
  if (tid < 192) {
    sm.cnt[tid] = sm.tops[tid] = 0;
    if (tid < kBins) sm.mass[tid] = 0;
  }
  float mine[VEC], mx = -INFINITY;  // the largest of each vector
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    mine[v] = x[v][0];
#pragma unroll
    for (int j = 1; j < kTok; ++j) mine[v] = fmaxf(mine[v], x[v][j]);
    mx = fmaxf(mx, mine[v]);
  }
  mx = wave_max(mx);
  if (lane == 0) sm.red[tid >> 6] = mx;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kScanWaves; ++w) mx = fmaxf(mx, sm.red[w]);
  mx = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, mx)));
  Bins& to = bins[slot];
  if (!s.filters) {
    const double lref = (double)mx * s.c;
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      u64 sum = 0;
#pragma unroll
      for (int j = 0; j < kTok; ++j) {
        const float y = x[v][j];
        if (y > -INFINITY) sum += weight(y == mx ? 0.0 : lref - (double)y * s.c);
      }
      sum = wave_total(sum);
      if (lane == 0) sm.sums[v * kScanWaves + (tid >> 6)] = sum;
    }
    __syncthreads();
    if (tid < 64) {
      const u64 w = lane < kParts ? sm.sums[lane] : 0, all = wave_total(w);
      if (lane < kParts) to.mass[lane] = w;
      if (lane == 0) rec[slot] = Chunk{lref, all, mx, 0, 0, 0};
    }
    return;
  }
  // Without top-p, tokens that min-p drops even by the chunk's own maximum do not
  // count.
  const double q4 = 4.0 * s.c, least = s.fp ? -INFINITY : (double)mx * s.c + s.lmin;
  Series series;
  series.hold();
  auto place = [&](float y, auto limited, u64* w) __attribute__((always_inline)) {
    const int b = bin_of(y, mx, q4, w, series);
    return decltype(limited)::value && (double)y * s.c < least && y != mx ? kBins : b;
  };
  int counted = s.fk ? kBins : kFirstBins;
  if (s.few) {
    // the first bins in which k vectors have their largest token hold the chunk's
    // first k (no such: all bins)
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      u64 unused;
      const int b = place(mine[v], std::true_type{}, &unused);
      if (b < kBins) atomicAdd(&sm.tops[b], 1u);
    }
    __syncthreads();
    uint32_t sum = 0;
#pragma unroll
    for (int i = 0; i < 3; ++i) sum += sm.tops[3 * lane + i];
    const uint32_t inc = wave_scan(sum);
    const u64 enough = __ballot(inc >= (uint32_t)s.k);
    counted = enough ? min(3 * (int)__builtin_ctzll(enough) + 3, kBins) : kBins;
  }
  int bin[VEC][kTok];
  uint32_t rank[VEC][kTok];
  uint32_t nth[VEC];  // a digit each: the token that x[v][i], bin[v][i], rank[v][i] is of
  if (s.few || least > -INFINITY) {
    // Few tokens count: those under `floor_x` are left by one fp32 comparison (a
    // margin of 1e-6 below the border that fp64 decides), and a wavefront goes over
    // the others, not over its columns.
    const double top = floor((double)mx * q4);
    const float edge = (float)(s.few ? (top - (counted - 1)) / q4 : least / s.c);
    const float floor_x = fabsf(edge) < 1e37f ? edge - 1e-6f * fabsf(edge) - 1e-37f : -INFINITY;
    auto few = [&](auto vector) __attribute__((always_inline)) {
      constexpr int v = decltype(vector)::value;
      uint32_t left = 0;
      nth[v] = 0;
#pragma unroll
      for (int j = 0; j < kTok; ++j) {
        left |= (uint32_t)(x[v][j] >= floor_x) << j;
        bin[v][j] = kBins;
      }
#pragma unroll
      for (int i = 0; i < kTok; ++i) {
        if (!__any(left != 0)) break;
        if (left != 0) {
          const int j = __builtin_ctz(left);
          left &= left - 1;
          const float y = nth_of(x[v], j);
          u64 w;
          const int b = bin[v][i] = place(y, std::true_type{}, &w);
          if (!s.few && b < kBins) atomicAdd(&sm.mass[b], w);
          if (b < counted) rank[v][i] = atomicAdd(&sm.cnt[b], 1u);
          x[v][i] = y;  // (j >= i, and no later token of this vector is x[v][i])
          nth[v] |= (uint32_t)j << 4 * i;
        }
      }
    };
    // (as a loop its body's arrays are not held in registers)
    static_assert(VEC <= 2, "");
    few(std::integral_constant<int, 0>{});
    if constexpr (VEC == 2) few(std::integral_constant<int, 1>{});
  } else {
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      nth[v] = 0x76543210;
#pragma unroll
      for (int j = 0; j < kTok; ++j) {
        u64 w;
        const int b = bin[v][j] = place(x[v][j], std::false_type{}, &w);
        if (b < kBins) atomicAdd(&sm.mass[b], w);
        if (b < counted) rank[v][j] = atomicAdd(&sm.cnt[b], 1u);
      }
    }
  }
  __syncthreads();
  if (tid < 64) {  // three bins a lane
    uint32_t n[3], sum = 0;
#pragma unroll
    for (int i = 0; i < 3; ++i) sum += n[i] = sm.cnt[3 * lane + i];
    const uint32_t inc = wave_scan(sum);
    uint32_t before = inc - sum;
    // written out: whole bins while they fit, up to the one that completes a
    // small top-k
    int last = 0;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const int b = 3 * lane + i;
      sm.first[b] = before;
      last += b < counted && before + n[i] <= (uint32_t)kCand &&
              !(s.few && before >= (uint32_t)s.k);
      before += n[i];
    }
    // (the bins for which that holds are the first ones)
    last = (int)wave_total((uint32_t)last) - 1;
    const uint32_t all = lane_value(inc, 63);
    if (lane == 0) sm.last = last;
    // written above by this wavefront: LDS keeps its order
    const uint32_t n_out = last + 1 < 192 ? sm.first[last + 1] : all;
    if (lane == 0)
      rec[slot] = Chunk{0.0, 0, mx, last, (int)n_out,
                        s.few && (n_out >= (uint32_t)s.k || n_out == all)};
  }
  __syncthreads();
  const int last = sm.last;
#pragma unroll
  for (int v = 0; v < VEC; ++v)
#pragma unroll
    for (int j = 0; j < kTok; ++j)
      if (bin[v][j] <= last)
        to.list[sm.first[bin[v][j]] + rank[v][j]] =
            (u64)key_of(x[v][j]) << 32 | (uint32_t)(col[v] + (int)(nth[v] >> 4 * j & 15));
  if (s.few) return;
  if (tid <= kBins) to.first[tid] = sm.first[tid];
  if (tid < kBins) to.mass[tid] = sm.mass[tid];
}

// ---------------------------------------------------------------------------
// draw: grid (rows)
// ---------------------------------------------------------------------------
constexpr int kDraw = 512, kDrawWaves = kDraw / 64;
constexpr int kSub = 1024;      // sub-bins of the radix select
constexpr int kList = 4096;     // tokens collected in LDS
constexpr int kMost = kList - kSmallK;  // ... for a small top-k, what it leaves behind them
static_assert(kFewTokens < kMost, "");
constexpr int kCell = 64, kCells = kChunk / kCell;  // columns of a chunk's cells

// A pass over (a part of) the row, by the workgroup, for its tokens between two
// keys: what bins with too many tokens for the list are worked on with.
enum PassMode { kCollect, kSubs, kKeys, kKeep, kBinsOf, kCellsOf };
struct DrawSmem {
  u64 list[kList];              // key << 32 | column of the collected tokens
  u64 few_w[kSmallK];           // weights of what a small top-k leaves
  u64 sub_mass[kSub];           // radix select: weight and count by sub-bin
  uint32_t sub_cnt[kSub];
  u64 mass[kBins];              // the row's bins, weights in the row's scale
  uint32_t cnt[kBins];
  double scale[kBins];          // a bin's scale: 2^(-bin / 4)
  int off[kMaxChunks];          // bins that the chunk's maximum lies below the row's; kBins: out
  int last[kMaxChunks];
  uint32_t from[kMaxChunks], base[kMaxChunks + 1];  // collecting: where in a chunk's list, and ours
  u64 kept[kMaxChunks];         // kept weight of a chunk
  u64 cell[kCells];             // ... of a chunk's 64 columns
  u64 tmp[kDrawWaves];
  uint32_t ends[2];             // keys of the first and last logit of some bins
  uint32_t kmin, kmax, n_few;
  int ties[64];                 // columns of a border's equal tokens
  uint32_t n_ties;
  u64 a, b;                     // a value that one thread hands to all
  float xr;
  double c, lmin;               // log2(e) / T; min-p in terms of L = x c, -inf without
  int i, j;
};

// A bin with too many tokens for the list, of up to kKeysMax keys (bf16 logits):
// their counts by chunk and key take the list's place.
constexpr int kKeysMax = kList * 2 / kMaxChunks;
// (of the module, not the kernel: the calls below reach it as LDS, not through
// generic pointers, whose accesses made a pass over a row 15 times as long)
static __shared__ DrawSmem sm;
DEVI uint32_t& key_count(int ch, uint32_t below_top) {
  return reinterpret_cast<uint32_t*>(sm.list)[ch * kKeysMax + below_top];
}

// Exclusive prefix sum over the workgroup; total in *total.
DEVI u64 block_scan(u64 v, u64* total) {
  const int wave = threadIdx.x >> 6;
  const u64 inc = wave_scan(v);
  if ((threadIdx.x & 63) == 63) sm.tmp[wave] = inc;
  __syncthreads();
  u64 base = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kDrawWaves; ++w) {
    const u64 t = sm.tmp[w];
    base += w < wave ? t : 0;
    all += t;
  }
  __syncthreads();
  *total = all;
  return base + inc - v;
}

// Which sub-bin a token falls in.  By key (cs < 0): keys top - sub << sh downwards.
// By column, whose bits from prev on are those of col0: its bits from cs on.
struct Digit {
  uint32_t top;
  int sh, cs, prev, col0;
  DEVI bool skips(int col) const { return cs >= 0 && (col ^ col0) >> prev; }
  DEVI uint32_t sub(uint32_t key, int col, int subs) const {
    return cs < 0 ? (top - key) >> sh : (uint32_t)(col >> cs) & (subs - 1);
  }
};
constexpr int kColBits = 19;
struct Pass {
  uint32_t k0, k1;               // the keys
  Digit digit;                   // kSubs
  int by_count, min_p;           // kSubs; kKeep, kCellsOf: and those that min-p keeps
  uint32_t cut_key;              // kSubs, kKeep, kCellsOf: tokens above this cut
  int cut_col;
};
// One round of a radix select by N threads (a wavefront, or the workgroup): clear
// the sub-bins, add the tokens to sm.sub_cnt and sm.sub_mass at at(sub-bin),
// and pick the sub-bin at which the running sum of counts, or weights, reaches
// *need, which becomes what is needed in it (0: no sum at all); *n: its count.
// at: a thread's PER consecutive sub-bins, N apart (no bank conflicts).
// A round is by a part of the key, or by LOG2 bits of the column: see Digit.
template <int N, int LOG2>
struct Select {
  static constexpr int SUBS = 1 << LOG2, PER = SUBS / N;
  DEVI static uint32_t at(uint32_t sub) { return sub % PER * N + sub / PER; }
  DEVI static void sync() {
    if (N > 64) __syncthreads();
    else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  DEVI static void clear() {
    const int r = threadIdx.x % N;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      sm.sub_mass[i * N + r] = 0;
      sm.sub_cnt[i * N + r] = 0;
    }
    sync();
  }
  DEVI static uint32_t pick(bool by_count, u64* need, u64* n) {
    const int r = threadIdx.x % N;
    sync();
    u64 v[PER], sum = 0, all, before;
    uint32_t cnt[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      cnt[i] = sm.sub_cnt[i * N + r];
      if (!by_count) v[i] = sm.sub_mass[i * N + r];
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) sum += by_count ? v[i] = cnt[i] : v[i];
    if constexpr (N > 64) {
      before = block_scan(sum, &all);
    } else {
      const u64 inc = wave_scan(sum);
      before = inc - sum;
      all = lane_value(inc, 63);
    }
    const u64 want = min(*need, all);  // (a merged bin's sum may have been rounded up)
    if (before < want && want <= before + sum) {  // one thread: find it among its own
      int at = 0;
      u64 left = want - before;
      uint32_t n_at = cnt[0];
#pragma unroll
      for (int i = 0; i + 1 < PER; ++i) {  // (once left is within v[at], no more)
        const bool next = at == i && left > v[i];
        left -= next ? v[i] : 0;
        at += next;
        n_at = next ? cnt[i + 1] : n_at;
      }
      sm.i = r * PER + at;
      sm.a = left;
      sm.b = n_at;
    }
    sync();
    const uint32_t sub = sm.i;
    *need = want > 0 ? sm.a : 0;
    *n = sm.b;
    sync();
    return sub;
  }
};

using BlockSelect = Select<kDraw, 10>;
using WaveSelect = Select<64, 8>;

// floor(x total) for x in [0, 1), in whole numbers: fp64 would round totals past
// 2^53, and a border of equal weights would move.
DEVI u64 share(double x, u64 total) {
  return __umul64hi((u64)(x * 18446744073709551616.0), total);
}
// The weight that top-p's part holds at least: p total, less the rounding of p
// itself (0.9 of 40 equal tokens are 36 of them, though the nearest fp64 to 0.9
// is above it).
DEVI u64 part_of(double p, u64 total) {
  const u64 n = share(p, total), slack = total >> 50;
  return n > slack ? n - slack : 1;
}
// u times a total, as the running weight that the drawn token exceeds.
DEVI u64 target_of(float u, u64 total) {
  return u < 1.0f ? (u > 0.0f ? share(u, total) : 0) : u >= 1.0f ? total - 1 : 0;
}

// Without filters, by one wavefront: the chunk, its 512 columns, the token.
template <typename T>
DEVI void draw_plain(const T* row, int cols, int mis, const Settings& s, float u,
                     const Chunk* rec, const Bins* bins, int n_ch, long long* out) {
  const int lane = threadIdx.x & 63;
  Chunk r{};
  r.xmax = -INFINITY;
  if (lane < n_ch) r = rec[lane];
  const float xr = wave_max(r.xmax);
  if (xr == -INFINITY) {  // no token to draw
    if (lane == 0) *out = -1;
    return;
  }
  const double d = r.xmax == xr ? 0.0 : (double)xr * s.c - r.lref;
  const bool in = r.xmax > -INFINITY && d < 46.0;
  const double f = in ? (d == 0.0 ? 1.0 : exp2_neg(d)) : 0.0;  // chunk scale -> row scale
  const u64 w = !in ? 0 : f == 1.0 ? r.mass : (u64)((double)r.mass * f + 0.5);
  const u64 inc = wave_scan(w);
  u64 t = target_of(u, lane_value(inc, 63));
  // one lane: the running sums are increasing
  const int ch = __builtin_ctzll(__ballot(inc - w <= t && t < inc));
  t -= lane_value(inc - w, ch);
  const double fc = __builtin_bit_cast(double, lane_value(__builtin_bit_cast(u64, f), ch));
  if (fc != 1.0) t = (u64)((double)t / fc);  // in the chunk's scale
  t = min(t, lane_value(r.mass, ch) - 1);
  const double lref = __builtin_bit_cast(double, lane_value(__builtin_bit_cast(u64, r.lref), ch));
  const float xmax = __builtin_bit_cast(float, lane_value(__builtin_bit_cast(uint32_t, r.xmax), ch));
  const u64 part = lane < kParts ? bins[ch].mass[lane] : 0, pinc = wave_scan(part);
  const int sub = __builtin_ctzll(__ballot(pinc - part <= t && t < pinc));
  t -= lane_value(pinc - part, sub);
  float x[kTok];
  const int col = load8(row, cols, mis, ch, sub * 64 + lane, x);
  u64 v[kTok], mine = 0;
#pragma unroll
  for (int j = 0; j < kTok; ++j) {
    v[j] = x[j] > -INFINITY ? weight(x[j] == xmax ? 0.0 : lref - (double)x[j] * s.c) : 0;
    mine += v[j];
  }
  u64 run = wave_scan(mine) - mine;
  if (run <= t && t < run + mine) {
    int at = col;
#pragma unroll
    for (int j = 0; j < kTok; ++j) {  // tokens whose running weight does not exceed t
      run += v[j];
      at += run <= t;
    }
    *out = at;
  }
}

// A token's bin below the row's maximum and its weight in the row's scale (0
// past the bins).
DEVI u64 row_weight(float x, int* b) {
  u64 w;
  *b = bin_of(x, sm.xr, 4.0 * sm.c, &w);
  const u64 scaled = (u64)((double)w * sm.scale[min(*b, kBins - 1)] + 0.5);
  return *b == 0 ? w : *b < kBins ? scaled : 0;
}
DEVI bool above(uint32_t key, int col, uint32_t cut_key, int cut_col) {
  return key > cut_key || (key == cut_key && col <= cut_col);
}
DEVI bool min_p_keeps(float x) {
  return x == sm.xr || (double)x * sm.c >= sm.lmin || sm.lmin == -INFINITY;
}

// The least and one past the greatest key of the logits of bins lo .. hi, into
// sm.ends: a bin falls with the logit, so each end is the least key of a bin up to
// a bound (wavefront 0: up to hi; 1: below lo).  It lies next to bound / q4; where
// it does not (q4 = 0, ends of the range), a search over the keys, 64 at a time.
DEVI void find_ends(int lo, int hi) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  __syncthreads();
  if (wave < 2) {
    const int bound = wave == 0 ? hi : lo - 1;
    const double q4 = 4.0 * sm.c;
    uint32_t first = key_of(-INFINITY) + 1, end = key_of(sm.xr) + 1;  // it lies in [first, end]
    auto up_to = [&](uint32_t k) __attribute__((always_inline)) {
      u64 w;
      return bin_of(of_key(k), sm.xr, q4, &w) <= bound;
    };
    if (bound < 0) {
      first = end;
    } else {
      const float guess = (float)((floor((double)sm.xr * q4) - bound) / q4) + 0.0f;
      const uint32_t k = key_of(guess == guess ? guess : 0.0f) - 32 + lane;
      const u64 yes = __ballot(k >= first && k < end && up_to(k));
      const u64 no = __ballot(k >= first && k < end && !up_to(k));
      if (yes && no) {  // (the noes come first)
        const int n = __builtin_ctzll(yes);
        first = end = lane_value(k, n);
      }
    }
    while (first < end) {
      const uint32_t step = (end - first) / 64 + 1;
      const uint32_t k = first + (uint32_t)min((u64)step * lane, (u64)(end - first - 1));
      const u64 yes = __ballot(up_to(k));
      // lanes from the first yes on; the answer is that lane's key or before it
      const int n = yes ? __builtin_ctzll(yes) : 64;
      if (n < 64) end = lane_value(k, n);
      if (n == 0) break;
      first = lane_value(k, n - 1) + 1;
    }
    if (lane == 0) sm.ends[wave] = end;
  }
  __syncthreads();
}

// The pass over columns of parts [part, end) (half chunks).  kCollect: into the
// list, sm.base[64] counting them, past what fits too.  Calls of their own, because
// few rows need them and each place that may is code.
template <typename T, int MODE>
__device__ __attribute__((noinline)) void pass(const T* row, int cols, int mis, int part, int end,
                                               Pass p) {
  const int lane = threadIdx.x & 63;
  __syncthreads();
  if (MODE == kCollect) {
    if (threadIdx.x == 0) sm.base[64] = 0;
    __syncthreads();
  }
  constexpr int U = 2;                        // vectors of 8 logits: one in use, one loading
  constexpr int VW = kTok / Vec16<T>::N;      // loads a vector
  constexpr int KS = sizeof(T) == 2 ? 16 : 0;
  const float x0 = of_key(p.k0), x1 = of_key(p.k1);
  // a thread's vector of 8 logits in columns c ..: of the weights, all are formed
  // before the first is used
  auto vec8 = [&](const float* y, int c) __attribute__((always_inline)) {
    if (MODE == kCollect) {  // one place in the list for all of a wavefront's tokens
      uint32_t left = 0;
#pragma unroll
      for (int j = 0; j < kTok; ++j) left |= (uint32_t)(y[j] >= x0 && y[j] <= x1) << j;
      const uint32_t n = __builtin_popcount(left), inc = wave_scan(n), all = lane_value(inc, 63);
      if (all == 0) return;
      uint32_t at = 0;
      if (lane == 0) at = atomicAdd(&sm.base[64], all);
      at = lane_value(at, 0) + inc - n;
      while (left != 0) {
        const int j = __builtin_ctz(left);
        left &= left - 1;
        if (at < (uint32_t)kList)
          sm.list[at] = (u64)key_of(nth_of(y, j)) << 32 | (uint32_t)(c + j);
        ++at;
      }
      return;
    }
    bool in[kTok];
    uint32_t key[kTok];
    int b[kTok];
    u64 w[kTok];
#pragma unroll
    for (int j = 0; j < kTok; ++j) {
      in[j] = y[j] >= x0 && y[j] <= x1;
      key[j] = key_of(y[j]);
      if (MODE != kBinsOf && MODE != kKeys)
        in[j] = in[j] && above(key[j], c + j, p.cut_key, p.cut_col);
      if (MODE == kSubs) in[j] = in[j] && !p.digit.skips(c + j);
      if (MODE == kKeep || MODE == kCellsOf) in[j] = in[j] && (!p.min_p || min_p_keeps(y[j]));
    }
    if (MODE != kKeys && (MODE != kSubs || !p.by_count)) {
#pragma unroll
      for (int j = 0; j < kTok; ++j) w[j] = row_weight(in[j] ? y[j] : sm.xr, &b[j]);
    }
    u64 sum = 0;
#pragma unroll
    for (int j = 0; j < kTok; ++j) {
      if (MODE == kSubs && in[j]) {
        const uint32_t at =
            BlockSelect::at(p.digit.sub(key[j] >> KS, c + j, BlockSelect::SUBS));
        atomicAdd(&sm.sub_cnt[at], 1u);
        if (!p.by_count) atomicAdd(&sm.sub_mass[at], w[j]);
      }
      if (MODE == kKeys && in[j])
        atomicAdd(&key_count((c + mis) / kChunk, p.digit.top - (key[j] >> KS)), 1u);
      if (MODE == kBinsOf && in[j]) {
        atomicAdd(&sm.cnt[b[j]], 1u);
        atomicAdd(&sm.mass[b[j]], w[j]);
      }
      if (MODE == kKeep || MODE == kCellsOf) sum += in[j] ? w[j] : 0;
      if (MODE == kCellsOf && in[j] && w[j] == 0)
        atomicMin(&sm.kmin, (uint32_t)((c + j + mis) % kChunk));
    }
    if (MODE == kKeep) {  // (a wavefront's 512 columns lie in one chunk)
      sum = wave_total(sum);
      if (lane == 0 && sum > 0) atomicAdd(&sm.kept[(c + mis) / kChunk], sum);
    }
    // (a thread's 8 columns lie in one cell)
    if (MODE == kCellsOf && sum > 0) atomicAdd(&sm.cell[(c + mis) % kChunk / kCell], sum);
  };
  // A vector of 8 logits at a time, the next one in flight (four or eight at a time
  // are no faster: one CU issues the instructions of a row of 128256 in about 26 us).
  // (One body, looped: code that a row runs through once is fetched from memory as
  // it goes, and a body for each of 32 logits took longer to arrive than its data.)
  const int s0 = part * (kSlots / 2), s1 = end * (kSlots / 2);
  // (a call's pointer argument may be to LDS for all that the compiler knows: loads
  // through it would be waited for with every LDS operation)
  typedef __attribute__((address_space(1))) u32x4 GlobalVec;
  u32x4 raw[U][VW];
  auto load = [&](int slot, u32x4* to) __attribute__((always_inline)) {
    // whole vectors inside the row; elsewhere one of the row's, not used
    const int col = slot * kTok - mis;
    const int at = slot < s1 && col >= 0 && col + kTok <= cols ? col : mis ? kTok - mis : 0;
    if (at + kTok <= cols) {
#pragma unroll
      for (int v = 0; v < VW; ++v)
        to[v] = *(const GlobalVec*)(uintptr_t)(row + at + v * (kTok / VW));
    }
  };
  int slot = s0 + threadIdx.x;
#pragma unroll
  for (int i = 0; i < U; ++i) load(slot + i * kDraw, raw[i]);
  for (; slot - (int)threadIdx.x < s1; slot += kDraw) {  // (uniform)
    float x[kTok];
    const int col = slot * kTok - mis;
    if (slot < s1 && col >= 0 && col + kTok <= cols) {
#pragma unroll
      for (int j = 0; j < kTok; ++j) {
        const uint32_t w = raw[0][j / (kTok / VW)][KS ? j / 2 : j % 4];
        const float y = !KS ? __builtin_bit_cast(float, w) : j & 1 ? bf16hi(w) : bf16lo(w);
        x[j] = y + 0.0f;  // (NaN: outside every interval)
      }
    } else {
      load8(row, slot < s1 ? cols : 0, mis, 0, slot, x);
    }
#pragma unroll
    for (int i = 0; i + 1 < U; ++i)
#pragma unroll
      for (int v = 0; v < VW; ++v) raw[i][v] = raw[i + 1][v];
    load(slot + U * kDraw, raw[U - 1]);
    if (MODE == kCollect && sm.base[64] > (uint32_t)kList) break;  // they do not fit
    vec8(x, col);
  }
  __syncthreads();
}

template <typename T>
__device__ void sample_draw(const T* __restrict__ logits, long ld, int cols, const Args a,
                            const float* __restrict__ us, const Chunk* __restrict__ rec,
                            const Bins* __restrict__ bins, int n_ch, long long* __restrict__ out,
                            int* __restrict__ advance) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row_i = blockIdx.x;
  if (advance && row_i == 0 && tid == 0) *advance += 1;
  const T* row = logits + row_i * ld;
  const int mis = misaligned(row);
  rec += (long)row_i * n_ch;
  bins += (long)row_i * n_ch;
  out += row_i;
  const float u = us[row_i];
  const Settings s = settings(a, row_i, cols);
  if (!s.filters) {
    if (wave == 0) draw_plain(row, cols, mis, s, u, rec, bins, n_ch, out);
    return;
  }
  const double c = s.c, q4 = 4.0 * c;

  // ---- the row's maximum, and each chunk's place below it -------------------
  if (wave == 0) {
    Chunk r{};
    r.xmax = -INFINITY;
    if (lane < n_ch) r = rec[lane];
    const float m = wave_max(r.xmax);
    u64 w;
    const int off = r.xmax > -INFINITY ? bin_of(r.xmax, m, q4, &w) : kBins;
    sm.off[lane] = off;
    sm.last[lane] = r.last;
    sm.from[lane] = 0;
    sm.kept[lane] = 0;
    // what a small top-k collects: all that the chunks wrote out
    const uint32_t n = off < kBins ? r.n_out : 0, inc = wave_scan(n);
    sm.base[lane] = inc - n;
    if (lane == 63) sm.base[64] = inc;
    const bool all = __all(off >= kBins || r.complete);
    if (lane == 0) {
      sm.xr = m;
      sm.c = c;
      sm.lmin = s.lmin > -INFINITY ? (double)m * c + s.lmin : -INFINITY;
      sm.i = all;
      sm.kmin = sm.kmax = sm.n_few = sm.n_ties = 0;
    }
  }
  for (int i = tid; i < kBins; i += kDraw) {
    sm.cnt[i] = 0;
    sm.mass[i] = 0;
    sm.scale[i] = exp2_neg(0.25 * i);
  }
  if (tid < kCells) sm.cell[tid] = 0;
  __syncthreads();
  const float xr = sm.xr;
  if (xr == -INFINITY) {  // no token to draw
    if (tid == 0) *out = -1;
    return;
  }
  // a small top-k whose chunks wrote out all that it needs, and that fits
  const bool fast = s.few && sm.i && sm.base[64] <= (uint32_t)kMost;

  // the border that top-k and top-p leave: tokens with a higher key, or the same
  // key and a column up to cut_col; jc: its bin (kBins: no border)
  uint32_t cut_key = 0;
  int cut_col = 0x7fffffff, jc = kBins;
  auto above_cut = [&](uint32_t key, int col) __attribute__((always_inline)) {
    return above(key, col, cut_key, cut_col);
  };

  // Copies the chunks' list entries [from, from + base[ch + 1] - base[ch]) into
  // ours: 16 lanes a chunk.
  auto gather = [&]() __attribute__((always_inline)) {
    const int l16 = tid & 15;
    for (int ch = tid >> 4; ch < n_ch; ch += kDraw / 16) {
      const uint32_t b0 = sm.base[ch], n = sm.base[ch + 1] - b0;
      const u64* src = bins[ch].list + sm.from[ch];
      for (uint32_t i = l16; i < n; i += 64) {
        u64 e[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) e[t] = src[min(i + 16 * t, n - 1)];
#pragma unroll
        for (int t = 0; t < 4; ++t)
          if (i + 16 * t < n) sm.list[b0 + i + 16 * t] = e[t];
      }
    }
    __syncthreads();
  };

  // The border among the tokens between keys k0 and k1 that are above the present
  // cut: the one at which their running count (by_count) or weight, in the order,
  // reaches need.  Sets the cut.  A round finds a sub-bin: by key, until one is
  // left, then by column among its equals.
  // subs(k0, k1, digit, by_count): adds the tokens between k0 and k1 (without the
  // low bits that every key shares); narrowed(k0, k1, n): n of them are left;
  // equals(k, f): f(column) of those with key k, if they are at hand.
  constexpr int KS = sizeof(T) == 2 ? 16 : 0;
  // (bf16: the low half of a key is all zeros, of a negative logit's all ones)
  auto key_back = [](uint32_t k) __attribute__((always_inline)) {
    return KS ? k << 16 | (k & 0x8000u ? 0u : 0xffffu) : k;
  };
  auto border = [&](auto select, auto weighs, uint32_t k0, uint32_t k1, u64 need, bool by_count,
                    auto&& subs, auto&& narrowed, auto&& equals) __attribute__((always_inline)) {
    constexpr bool WEIGH = decltype(weighs)::value;
    constexpr int SUBS = decltype(select)::SUBS, BITS = __builtin_ctz(SUBS);
    k0 >>= KS;
    k1 >>= KS;
    Digit dg{0, 0, -1, kColBits, 0};
    bool all_equals = true;
    for (;;) {
      const uint32_t span = k1 - k0;
      dg.sh = span < (uint32_t)SUBS ? 0 : 32 - BITS - __builtin_clz(span);
      dg.top = k1;
      select.clear();
      // a key per sub-bin: counted, and weighed once for all its tokens
      const bool weigh = WEIGH && !by_count && dg.sh == 0;
      subs(k0, k1, dg, by_count || weigh);
      if (weigh) {
        __syncthreads();
        for (uint32_t i = tid; i <= k1 - k0; i += kDraw) {
          int b;
          const uint32_t cnt = sm.sub_cnt[select.at(i)];
          if (cnt > 0) sm.sub_mass[select.at(i)] = cnt * row_weight(of_key(key_back(k1 - i)), &b);
        }
      }
      u64 n = 0;
      const uint32_t sub = select.pick(by_count, &need, &n);
      if (need == 0) break;  // every weight here rounds to zero: all are kept
      if (dg.cs < 0) {
        const uint32_t top = k1 - (sub << dg.sh);
        k0 = top - k0 < (1u << dg.sh) ? k0 : top - (1u << dg.sh) + 1;
        k1 = top;
        narrowed(KS ? k0 << 16 : k0, KS ? k1 << 16 | 0xffffu : k1, n);
        if (k0 < k1) continue;
        if (!by_count) {  // as many of the equal tokens as their weight needs
          int b;
          const u64 w = row_weight(of_key(key_back(k0)), &b);
          need = (need + w - 1) / w;
          by_count = true;
        }
        if (need >= n) break;  // all of them
        all_equals = false;
        // up to 64: a lane each, which counts the columns before its own (64 rows
        // with top-p 13.9 us, by two more rounds 15.9)
        if (n <= 64 && equals(k0, [&](int col) __attribute__((always_inline)) {
              const uint32_t i = atomicAdd(&sm.n_ties, 1u);
              if (i < 64) sm.ties[i] = col;
            })) {
          select.sync();
          const int ties = __builtin_amdgcn_readfirstlane((int)n);
          const int col = lane < ties ? sm.ties[lane] : 0x7fffffff;
          u64 before = 0;
          for (int i = 0; i < ties; ++i) before += (int)lane_value((uint32_t)col, i) < col;
          const u64 at = __ballot(lane < ties && before == need - 1);
          dg.col0 = (int)lane_value((uint32_t)col, __builtin_ctzll(at));
          select.sync();
          if (tid == 0) sm.n_ties = 0;
          break;
        }
        dg.cs = kColBits - BITS;
      } else {
        dg.col0 = dg.col0 >> (dg.cs + BITS) << (dg.cs + BITS) | (int)(sub << dg.cs);
        if (dg.cs == 0) break;
        dg.prev = dg.cs;
        dg.cs = max(dg.cs - BITS, 0);
      }
    }
    k0 = key_back(k0);
    if (!all_equals) {
      cut_key = k0;
      cut_col = dg.col0;
    } else if (k0 > cut_key) {  // (of equals of the cut those up to its column stay)
      cut_key = k0;
      cut_col = 0x7fffffff;
    }
  };

  if (fast) {
    // ---- a small top-k: all that the chunks wrote out, then the k of them --------
    gather();
    const uint32_t n_all = sm.base[64];
    uint32_t lo = 0, hi = 0;  // of ~key and key
    for (uint32_t i = tid; i < n_all; i += kDraw) {
      const uint32_t key = (uint32_t)(sm.list[i] >> 32);
      lo = max(lo, ~key);
      hi = max(hi, key);
    }
    lo = wave_max_u32(lo);
    hi = wave_max_u32(hi);
    if (lane == 0) {
      atomicMax(&sm.kmin, lo);
      atomicMax(&sm.kmax, hi);
    }
    __syncthreads();
    const uint32_t key0 = ~sm.kmin, key1 = sm.kmax;
    if (n_all > (uint32_t)s.k)
      border(
          BlockSelect{}, std::false_type{}, key0, key1, s.k, true,
          [&](uint32_t k0, uint32_t k1, Digit dg, bool) __attribute__((always_inline)) {
            for (uint32_t i = tid; i < n_all; i += kDraw) {
              const u64 e = sm.list[i];
              const uint32_t k = (uint32_t)(e >> 32) >> KS;
              const int col = (int)(uint32_t)e;
              if (k >= k0 && k <= k1 && !dg.skips(col))
                atomicAdd(&sm.sub_cnt[BlockSelect::at(dg.sub(k, col, BlockSelect::SUBS))], 1u);
            }
          },
          [](uint32_t, uint32_t, u64) {},
          [&](uint32_t k, auto&& f) __attribute__((always_inline)) {
            for (uint32_t i = tid; i < n_all; i += kDraw) {
              const u64 e = sm.list[i];
              if ((uint32_t)(e >> 32) >> KS == k) f((int)(uint32_t)e);
            }
            return true;
          });
    __syncthreads();
    for (uint32_t i = tid; i < n_all; i += kDraw) {
      const u64 e = sm.list[i];
      if (!above_cut((uint32_t)(e >> 32), (int)(uint32_t)e)) continue;
      const uint32_t at = atomicAdd(&sm.n_few, 1u);
      int b;
      sm.list[kMost + at] = e;
      sm.few_w[at] = row_weight(of_key((uint32_t)(e >> 32)), &b);
    }
    __syncthreads();
    // the rest by one wavefront, without barriers
    if (wave > 0) return;
    // (up to 64 tokens a lane each, which sums the weights of those before it, instead
    // of rounds of a radix select: 16 rows with 50 tokens 11.5 -> 14.9 us)
    constexpr int E = kSmallK / 64;  // tokens a lane
    const uint32_t n = sm.n_few;
    uint32_t key[E];
    int col[E];
    u64 w[E], mine = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const uint32_t at = lane + 64 * i;
      const u64 e = at < n ? sm.list[kMost + at] : 0;
      key[i] = (uint32_t)(e >> 32);
      col[i] = (int)(uint32_t)e;
      w[i] = at < n ? sm.few_w[at] : 0;
      mine += w[i];
    }
    if (s.fp) {
      const u64 total = wave_total(mine);
      border(
          WaveSelect{}, std::false_type{}, max(key0, cut_key), key1,
          max(1ull, min(part_of(s.p, total), total)), false,
          [&](uint32_t k0, uint32_t k1, Digit dg, bool by_count) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < E; ++i) {
              if (64 * i >= n) break;
              const uint32_t k = key[i] >> KS;
              if (lane + 64 * i >= n || k < k0 || k > k1 || dg.skips(col[i])) continue;
              const uint32_t at = WaveSelect::at(dg.sub(k, col[i], WaveSelect::SUBS));
              atomicAdd(&sm.sub_cnt[at], 1u);
              if (!by_count) atomicAdd(&sm.sub_mass[at], w[i]);
            }
          },
          [](uint32_t, uint32_t, u64) {},
          [&](uint32_t k, auto&& f) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < E; ++i) {
              if (64 * i >= n) break;
              if (lane + 64 * i < n && key[i] >> KS == k) f(col[i]);
            }
            return true;
          });
    }
    mine = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      if (lane + 64 * i < n && !(above_cut(key[i], col[i]) && min_p_keeps(of_key(key[i]))))
        w[i] = 0;
      mine += w[i];
    }
    // the token, in index order
    u64 t = target_of(u, wave_total(mine)) + 1, unused;
    constexpr int SUBS = WaveSelect::SUBS, BITS = __builtin_ctz(SUBS);
    Digit dg{0, 0, kColBits - BITS, kColBits, 0};
    for (;;) {
      WaveSelect::clear();
#pragma unroll
      for (int i = 0; i < E; ++i) {
        if (64 * i >= n) break;
        if (w[i] > 0 && !dg.skips(col[i]))
          atomicAdd(&sm.sub_mass[WaveSelect::at(dg.sub(0, col[i], SUBS))], w[i]);
      }
      const int sub = WaveSelect::pick(false, &t, &unused);
      dg.col0 = dg.col0 >> (dg.cs + BITS) << (dg.cs + BITS) | sub << dg.cs;
      if (dg.cs == 0) break;
      dg.prev = dg.cs;
      dg.cs = max(dg.cs - BITS, 0);
    }
    if (lane == 0) *out = dg.col0;
    return;
  }

  // ---- the row's bins ----------------------------------------------------------
  u64 m_before, m_here = 0;      // thread b: the weight before bin b, and in it
  u64 n_before = 0, n_here = 0;  // ... and tokens
  u64 total_n = 0, total_m;
  Pass p{};
  if (s.few) {  // too many for what the chunks wrote out: by passing over the row
    if (tid < kMaxChunks) sm.last[tid] = -1;
    find_ends(0, kBins - 1);
    p.k0 = sm.ends[0];
    p.k1 = sm.ends[1] - 1;
    pass<T, kBinsOf>(row, cols, mis, 0, 2 * n_ch, p);
  } else {
    const int counted = s.fk ? kBins : 0, all = n_ch * kBins;
    for (int i0 = tid; i0 < all; i0 += 4 * kDraw) {
      u64 m[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {  // (past the end: the last one again)
        const int i = min(i0 + t * kDraw, all - 1), ch = i / kBins;
        m[t] = bins[ch].mass[i - ch * kBins];
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int i = i0 + t * kDraw, ch = i / kBins, b = i - ch * kBins;
        const int r = i < all ? b + sm.off[ch] : kBins;
        if (r >= kBins) continue;
        if (m[t] > 0) atomicAdd(&sm.mass[r], m[t]);
        if (b < counted) atomicAdd(&sm.cnt[r], bins[ch].first[b + 1] - bins[ch].first[b]);
      }
    }
    __syncthreads();
    if (tid > 0 && tid < kBins)
      sm.mass[tid] = (u64)((double)sm.mass[tid] * sm.scale[tid] + 0.5);
  }
  __syncthreads();
  if (tid < kBins) {
    m_here = sm.mass[tid];
    n_here = sm.cnt[tid];
  }
  m_before = block_scan(m_here, &total_m);
  if (s.fk) n_before = block_scan(n_here, &total_n);

  // The list holds the tokens between keys list0 and list1 (none: list0 > list1).
  uint32_t list0 = 1, list1 = 0;
  // collects the tokens of bin j in the list, from what the chunks wrote out or
  // else from the row, if they fit; k0, k1: the bin's keys
  uint32_t bin0 = 0, bin1 = 0;
  int dense = -1;  // the bin whose tokens are held as counts by chunk and key
  auto collect = [&](int j) __attribute__((always_inline)) {
    find_ends(j, j);
    bin0 = sm.ends[0];
    bin1 = sm.ends[1] - 1;
    if ((bin0 >= list0 && bin1 <= list1) || dense == j) return;
    dense = -1;
    __syncthreads();
    if (wave == 0) {
      uint32_t f0 = 0, n = 0;
      const int b = lane < n_ch && sm.off[lane] < kBins ? j - sm.off[lane] : -1;
      if (b >= 0 && b <= sm.last[lane]) {
        f0 = bins[lane].first[b];
        n = bins[lane].first[b + 1] - f0;
      }
      const uint32_t inc = wave_scan(n);
      sm.from[lane] = f0;
      sm.base[lane] = inc - n;
      const bool ok = __all(b < 0 || b <= sm.last[lane]);
      if (lane == 63) sm.base[64] = inc;
      if (lane == 0) sm.i = ok && lane_value(inc, 63) <= (uint32_t)kList;
    }
    __syncthreads();
    list0 = 1;
    list1 = 0;
    if (sm.i) {
      gather();
    } else {
      p.k0 = bin0;
      p.k1 = bin1;
      pass<T, kCollect>(row, cols, mis, 0, 2 * n_ch, p);
      if (sm.base[64] > (uint32_t)kList) {
        p.digit.top = bin1 >> KS;
        if (p.digit.top - (bin0 >> KS) < (uint32_t)kKeysMax) {
          __syncthreads();
          for (int i = tid; i < kMaxChunks * kKeysMax; i += kDraw)
            reinterpret_cast<uint32_t*>(sm.list)[i] = 0;
          pass<T, kKeys>(row, cols, mis, 0, 2 * n_ch, p);
          dense = j;
        }
        return;
      }
    }
    list0 = bin0;
    list1 = bin1;
  };
  // f(key, column) for the list's tokens between two keys
  auto listed = [&](uint32_t k0, uint32_t k1, auto&& f) __attribute__((always_inline)) {
    const uint32_t n = sm.base[64];
    for (uint32_t i = tid; i < n; i += kDraw) {
      const u64 e = sm.list[i];
      const uint32_t key = (uint32_t)(e >> 32);
      if (key >= k0 && key <= k1) f(key, (int)(uint32_t)e);
    }
  };
  // The border in the dense bin; what is past it leaves the counts.
  auto dense_border = [&](u64 need, bool by_count) __attribute__((always_inline)) {
    const uint32_t top = bin1 >> KS;
    u64 cnt = 0, w = 0, all;
    int b;
    if (tid < kKeysMax) {
      for (int ch = 0; ch < n_ch; ++ch) cnt += key_count(ch, tid);
      if (cnt > 0) w = row_weight(of_key(key_back(top - tid)), &b);
    }
    const u64 v = by_count ? cnt : cnt * w, before = block_scan(v, &all);
    need = min(need, all);
    if (v > 0 && before < need && need <= before + v) {
      sm.i = tid;
      sm.a = by_count ? need - before : (need - before + w - 1) / w;  // of the equal tokens
    }
    __syncthreads();
    if (need == 0) return;  // every weight here rounds to zero: all are kept
    const int below = sm.i;
    const u64 ties = sm.a;
    __syncthreads();
    // the chunk of the last of them, and how many it has before
    if (wave == 0) {
      const u64 n = lane < n_ch ? key_count(lane, below) : 0, sum = wave_scan(n) - n;
      if (sum < ties && ties <= sum + n) {
        sm.i = lane;
        sm.a = ties - sum;
      }
    }
    __syncthreads();
    const int last_ch = sm.i;
    const u64 left = sm.a;
    // its column: 16 a thread
    const float x = of_key(key_back(top - below));
    float y[2][kTok];
    const int col = load8(row, cols, mis, last_ch, 2 * tid, y[0]);
    load8(row, cols, mis, last_ch, 2 * tid + 1, y[1]);
    u64 here = 0;
#pragma unroll
    for (int t = 0; t < 2 * kTok; ++t) here += y[t / kTok][t % kTok] == x;
    u64 n = block_scan(here, &all);
    if (n < left && left <= n + here) {
#pragma unroll
      for (int t = 0; t < 2 * kTok; ++t)
        if (y[t / kTok][t % kTok] == x && ++n == left) sm.j = col + t;
    }
    for (int i = tid; i < n_ch * kKeysMax; i += kDraw) {
      const int ch = i / kKeysMax, k = i - ch * kKeysMax;
      if (k > below || (k == below && ch > last_ch)) key_count(ch, k) = 0;
      else if (k == below && ch == last_ch) key_count(ch, k) = (uint32_t)left;
    }
    __syncthreads();
    cut_key = key_back(top - below);
    cut_col = sm.j;
  };
  static_assert(kKeysMax <= kDraw && 2 * kDraw * kTok == kChunk, "a key, 16 columns a thread");
  // sm.kept[chunk] += the kept weight of bin jc's tokens (min_p: and that it keeps)
  auto keep_bin = [&](bool min_p) __attribute__((always_inline)) {
    __syncthreads();
    if (bin0 >= list0 && bin1 <= list1) {
      listed(bin0, bin1, [&](uint32_t key, int col) __attribute__((always_inline)) {
        int b;
        const float x = of_key(key);
        if (above_cut(key, col) && (!min_p || min_p_keeps(x)))
          atomicAdd(&sm.kept[(col + mis) / kChunk], row_weight(x, &b));
      });
    } else if (dense == jc) {
      for (int i = tid; i < n_ch * kKeysMax; i += kDraw) {
        const int ch = i / kKeysMax, k = i - ch * kKeysMax;
        const uint32_t n = key_count(ch, k);
        if (n == 0) continue;
        int b;
        const float x = of_key(key_back((bin1 >> KS) - k));
        if (!min_p || min_p_keeps(x)) atomicAdd(&sm.kept[ch], n * row_weight(x, &b));
      }
    } else {
      p.k0 = max(bin0, cut_key);
      p.k1 = bin1;
      p.cut_key = cut_key;
      p.cut_col = cut_col;
      p.min_p = min_p;
      pass<T, kKeep>(row, cols, mis, 0, 2 * n_ch, p);
    }
    __syncthreads();
  };
  // ---- the borders: top-k's by count, then top-p's by weight --------------------
  for (int stage = s.fk ? 0 : 1; stage < (s.fp ? 2 : 1); ++stage) {
    u64 need;
    if (stage == 0) {
      need = min((u64)s.k, total_n);  // (fewer tokens than k: all of them)
    } else {
      u64 left = total_m;  // the weight that top-k leaves
      if (s.fk) {
        keep_bin(false);
        u64 mine = tid < kMaxChunks ? sm.kept[tid] : 0;
        if (tid == jc) mine += m_before;  // and the bins above
        block_scan(mine, &left);
        if (tid < kMaxChunks) sm.kept[tid] = 0;
      }
      need = max(1ull, min(part_of(s.p, left), min(left, total_m)));
    }
    // the bin at which the running sum over the bins reaches need
    const u64 before = stage == 0 ? n_before : m_before, here = stage == 0 ? n_here : m_here;
    __syncthreads();
    if (here > 0 && before < need && need <= before + here) {
      sm.i = tid;
      sm.a = need - before;
    }
    __syncthreads();
    const int j = sm.i;
    need = sm.a;
    if (j > jc) break;  // (by rounding) past top-k's border: that one holds
    collect(j);
    jc = j;
    if (dense == j) {
      dense_border(need, stage == 0);
      continue;
    }
    border(
        BlockSelect{}, std::true_type{}, bin0, bin1, need, stage == 0,
        [&](uint32_t k0, uint32_t k1, Digit dg, bool by_count) __attribute__((always_inline)) {
          const uint32_t a0 = k0 << KS, a1 = KS ? k1 << 16 | 0xffffu : k1;
          // (a bin's first key may lie above the first of its low half)
          if (max(a0, bin0) >= list0 && min(a1, bin1) <= list1) {
            listed(a0, a1, [&](uint32_t key, int col) __attribute__((always_inline)) {
              if (!above_cut(key, col) || dg.skips(col)) return;
              const uint32_t at = BlockSelect::at(dg.sub(key >> KS, col, BlockSelect::SUBS));
              int b;
              atomicAdd(&sm.sub_cnt[at], 1u);
              if (!by_count) atomicAdd(&sm.sub_mass[at], row_weight(of_key(key), &b));
            });
          } else {
            p.by_count = by_count;
            p.k0 = max(a0, bin0);
            p.k1 = min(a1, bin1);
            p.digit = dg;
            p.cut_key = cut_key;
            p.cut_col = cut_col;
            pass<T, kSubs>(row, cols, mis, 0, 2 * n_ch, p);
          }
        },
        [&](uint32_t k0, uint32_t k1, u64 n) __attribute__((always_inline)) {
          k0 = max(k0, bin0);
          k1 = min(k1, bin1);
          // (those below a top-k's cut are collected too, and may not fit)
          if ((k0 >= list0 && k1 <= list1) || n > (u64)kList) return;
          p.k0 = k0;
          p.k1 = k1;
          pass<T, kCollect>(row, cols, mis, 0, 2 * n_ch, p);
          const bool fits = sm.base[64] <= (uint32_t)kList;
          list0 = fits ? k0 : 1;
          list1 = fits ? k1 : 0;
        },
        [&](uint32_t k, auto&& f) __attribute__((always_inline)) {
          const uint32_t a0 = max(k << KS, bin0), a1 = min(KS ? k << 16 | 0xffffu : k, bin1);
          if (a0 < list0 || a1 > list1) return false;
          listed(a0, a1, [&](uint32_t key, int col) __attribute__((always_inline)) {
            if (above_cut(key, col)) f(col);
          });
          return true;
        });
  }
  if (s.lmin > -INFINITY) {
    const double r = floor((double)xr * q4) - floor(4.0 * sm.lmin);
    const int jm = r < (double)kBins ? (int)r : kBins;
    if (jm < jc) collect(jc = jm);
  }
  // ---- each chunk's kept weight: whole bins, and the border's bin --------------
  {
    const int l16 = tid & 15;
    for (int ch = tid >> 4; ch < n_ch && !s.few; ch += kDraw / 16) {
      const int off = sm.off[ch];
      u64 v = 0;
#pragma unroll 4
      for (int r = l16; r < jc - off; r += 16)
        v += r + off == 0 ? bins[ch].mass[r]
                          : (u64)((double)bins[ch].mass[r] * sm.scale[r + off] + 0.5);
      if (v > 0) atomicAdd(&sm.kept[ch], v);
    }
  }
  if (s.few) {  // (its chunks left no weights: every token up to the border)
    find_ends(0, min(jc, kBins - 1));
    bin0 = sm.ends[0];
    bin1 = sm.ends[1] - 1;
    list0 = 1;
    list1 = 0;
    dense = -1;
  }
  if (s.few || jc < kBins) keep_bin(true);
  __syncthreads();

  // ---- the chunk that u falls into, and where in it ---------------------------
  if (wave == 0) {
    const u64 w = lane < n_ch ? sm.kept[lane] : 0, inc = wave_scan(w);
    const u64 t = target_of(u, lane_value(inc, 63));
    if (inc - w <= t && t < inc) {
      sm.i = lane;
      sm.a = t - (inc - w);
    }
    if (lane == 0) sm.kmin = kChunk - 1;
  }
  __syncthreads();
  const int ch = sm.i, off = sm.off[ch];
  u64 t = sm.a;
  // ---- its kept weight by 64 columns ---------------------------------------------
  if (jc - off <= sm.last[ch]) {  // the chunk wrote out what can be kept
    const uint32_t end = bins[ch].first[jc - off + 1];
    for (uint32_t i = tid; i < end; i += kDraw) {
      const u64 e = bins[ch].list[i];
      const uint32_t key = (uint32_t)(e >> 32);
      const int col = (int)(uint32_t)e, at = col + mis - ch * kChunk;
      const float x = of_key(key);
      int b;
      const u64 w = row_weight(x, &b);
      if (b >= kBins || !above_cut(key, col) || !min_p_keeps(x)) continue;
      if (w > 0) atomicAdd(&sm.cell[at / kCell], w);
      else atomicMin(&sm.kmin, (uint32_t)at);
    }
  } else {
    find_ends(0, min(jc, kBins - 1));
    p.k0 = sm.ends[0];
    p.k1 = sm.ends[1] - 1;
    p.cut_key = cut_key;
    p.cut_col = cut_col;
    p.min_p = 1;
    pass<T, kCellsOf>(row, cols, mis, 2 * ch, 2 * ch + 2, p);
  }
  __syncthreads();
  // ---- the columns and the token, by one wavefront -------------------------------
  if (wave > 0) return;
  const u64 w0 = sm.cell[2 * lane], w1 = sm.cell[2 * lane + 1];
  const u64 inc = wave_scan(w0 + w1), all = lane_value(inc, 63);
  if (all == 0) {  // (a bin's weight was rounded as such, no token's own is above zero)
    if (lane == 0) *out = (long long)ch * kChunk + (int)sm.kmin - mis;
    return;
  }
  t = min(t, all - 1);
  const u64 b0 = inc - w0 - w1;
  const int at = __builtin_ctzll(__ballot(b0 <= t && t < inc));
  const u64 first = lane_value(b0, at), half = lane_value(w0, at);
  const bool second = t >= first + half;
  t -= first + (second ? half : 0);
  const int col = ch * kChunk + (2 * at + second) * kCell + lane - mis;
  float x = col >= 0 && col < cols ? (float)row[col] : -INFINITY;
  x = x == x ? x + 0.0f : -INFINITY;
  int b;
  u64 w = row_weight(x, &b);
  if (b >= kBins || !above_cut(key_of(x), col) || !min_p_keeps(x)) w = 0;
  const u64 run = wave_scan(w);
  if (run - w <= t && t < run) *out = col;
}

}  // namespace

#define TEENY_SAMPLE_INST(TN, T)                                                                  \
  extern "C" __global__ __launch_bounds__(512) void teeny_sample_scan_##TN(                       \
      const T* logits, long ld, int cols, Args a, Chunk* rec, Bins* bins) {                       \
    sample_scan<T, 2>(logits, ld, cols, a, rec, bins);                                            \
  }                                                                                               \
  extern "C" __global__ __launch_bounds__(1024) void teeny_sample_scan_##TN##_w16(                \
      const T* logits, long ld, int cols, Args a, Chunk* rec, Bins* bins) {                       \
    sample_scan<T, 1>(logits, ld, cols, a, rec, bins);                                            \
  }                                                                                               \
  extern "C" __global__ __launch_bounds__(512) void teeny_sample_draw_##TN(                      \
      const T* logits, long ld, int cols, Args a, const float* u, const Chunk* rec,               \
      const Bins* bins, int n_ch, long long* out, int* advance) {                                 \
    sample_draw<T>(logits, ld, cols, a, u, rec, bins, n_ch, out, advance);                        \
  }
TEENY_SAMPLE_INST(f32, float)
TEENY_SAMPLE_INST(bf16, bf16)
