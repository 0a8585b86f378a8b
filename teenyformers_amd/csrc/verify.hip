// Verification of drafted tokens against the target's probabilities from given
// random numbers.
//
// For a sequence with drafts d_0 .. d_{K-1}, target logits of K + 1 rows and the
// draft model's of K: p_i = softmax(target_i / T), q_i = softmax(draft_i / T), or
// without draft logits q_i all on d_i.  Draft i is accepted while u_i q_i(d_i) <
// p_i(d_i); the token after the accepted ones is drawn, in index order, from
// max(p_n - q_n, 0) where draft n was refused and from p_n where there was none:
// whatever the drafts, the tokens are distributed as the target's own.  Temperature
// 0: one-hot at the lowest index of the row's maximum.
//
// Numbers: a weight is 2^(x c - K) in fp32, c = log2(e) / T rounded to fp32 and K = c
// max x rounded (the exponent is one fused product: whatever rounds K is common to all
// weights, c's rounding moves a weight d octaves down by d 2^-24); sums of eight in fp32
// and from there in fp64; what decides (acceptance, the place of u among running sums) is
// fp64.  A draw from one row sums unscaled weights, exact for equal logits.  One order
// of sums: no atomics on them.
//
//   scan   workgroups take chunks of 8192 columns of the rows in turn: their maximum and
//          the weights' sum below it, each wavefront's below its own first (one barrier a
//          chunk), the next chunk's loads in flight meanwhile.  Reading the rows bounds it:
//          48 sequences of 8 drafts, 816 rows of 128256 bf16, 209 MB, 45 us (4.6 TB/s); 144
//          rows, 37 MB, 11 us; 5 rows 4.2 us.
//   rest   (chunk, sequence): each workgroup finds the sequence's accepted drafts from the
//          scan's sums (a wavefront a draft, a lane a chunk) and sums its chunk of what the
//          next token is drawn from; the one that ends last finds the chunk and the token.
//          Bound by a chain: records and drafts' logits, the chunk's rows, the count, the
//          sums, the drawn chunk once more: 16 sequences 11.6 us, 1 without draft logits (no
//          differences, no count) 6.6; 48, with 25 MB of rows and two exponentials a column,
//          18.
#include "sample.h"

namespace {

constexpr int kThreads = 512, kWaves = kThreads / 64;
constexpr int kMaxDrafts = 64;  // a lane each
constexpr double kLog2e = 1.4426950408889634074;
static_assert(kThreads * 2 * kTok == kChunk, "two vectors a thread");

struct Rec {
  double sum;  // weights of the chunk, relative to its maximum
  float xmax;  // -inf: no token
  int first;   // column of the first maximum
};
static_assert(sizeof(Rec) == 16, "the host sizes the workspace by it");

struct Args {
  const void *target, *draft;       // [B, K + 1, V], [B, K, V] or null
  long t_seq, t_row, d_seq, d_row;  // strides, elements
  const long long* drafts;          // [B, K]
  const float *u, *ts;              // [B, K + 1]; temperatures, or null: t
  double t;
  int batch, k, cols, n_ch;
};

// log2(e) / T (0: greedy)
struct Factor {
  float c;
  bool greedy;
  DEVI float ref(float xmax) const { return xmax * c; }  // K
};
DEVI Factor factor_of(const Args& a, float ts) {
  const double t = a.ts ? (double)ts : a.t;
  Factor f;
  f.greedy = !(t > 0.0);  // (NaN too)
  // (a factor past 1e30 leaves the same tokens)
  f.c = f.greedy ? (float)kLog2e : (float)fmin(kLog2e / t, 1e30);
  return f;
}
DEVI Factor factor_of(const Args& a, int b) { return factor_of(a, a.ts ? a.ts[b] : 0.0f); }
// The weight of x, K = ref; -inf and NaN have none.  (fmaxf takes the number where the
// exponent is NaN, and 2^-200 is zero.)
DEVI float weight(float x, float ref, const Factor& f) {
  return __builtin_amdgcn_exp2f(fmaxf(__builtin_fmaf(x, f.c, -ref), -200.0f));
}
// Whether K is small enough for that: its rounding, a factor of all weights, is 2^-9
// octaves at most.  Else (tiny temperatures, huge logits) the exponent is (x - max x) c;
// an infinite maximum and its equals have weight alone.  (A part without a token: any sum,
// which `below` leaves out.)
DEVI bool fused(float ref) { return fabsf(ref) < 65536.0f; }
DEVI float weight_apart(float x, float xmax, const Factor& f) {
  return __builtin_amdgcn_exp2f(x == xmax ? 0.0f : fmaxf((x - xmax) * f.c, -200.0f));
}
DEVI float weight(float x, float xmax, float ref, const Factor& f) {
  if (fused(ref)) return weight(x, ref, f);
  return xmax > -INFINITY ? weight_apart(x, xmax, f) : 0.0f;
}
// The reference of a row's, or a part's, weights as it was used
DEVI double ref_of(float xmax, const Factor& f) {
  const float k = f.ref(xmax);
  return fused(k) ? (double)k : (double)xmax * (double)f.c;
}
// 2^(a - b) of the references of maxima xa <= xb
DEVI float below(float xa, float xb, const Factor& f) {
  if (!(xa > -INFINITY)) return 0.0f;
  if (xa == xb) return 1.0f;
  return __builtin_amdgcn_exp2f(fmaxf((float)(ref_of(xa, f) - ref_of(xb, f)), -200.0f));
}

template <typename T> DEVI const T* target_row(const Args& a, int b, int i) {
  return (const T*)a.target + b * a.t_seq + i * a.t_row;
}
template <typename T> DEVI const T* draft_row(const Args& a, int b, int i) {
  return (const T*)a.draft + b * a.d_seq + i * a.d_row;
}
// Records: target rows (b, i) at b (K + 1) + i, then draft rows at b K + i.
DEVI const Rec* target_rec(const Args& a, const Rec* rec, int b, int i) {
  return rec + ((long)b * (a.k + 1) + i) * a.n_ch;
}
DEVI const Rec* draft_rec(const Args& a, const Rec* rec, int b, int i) {
  return rec + ((long)a.batch * (a.k + 1) + (long)b * a.k + i) * a.n_ch;
}

// Over the wavefront, through DPP: lane 63 has the whole (as wave_scan in sample.h).
template <int CTRL, int ROWS> DEVI float dpp_f(float v, float none) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(
      __builtin_bit_cast(int, none), __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false));
}
DEVI float wave_top(float v) {
  v = fmaxf(v, dpp_f<0x111, 0xf>(v, -INFINITY));
  v = fmaxf(v, dpp_f<0x112, 0xf>(v, -INFINITY));
  v = fmaxf(v, dpp_f<0x114, 0xf>(v, -INFINITY));
  v = fmaxf(v, dpp_f<0x118, 0xf>(v, -INFINITY));
  v = fmaxf(v, dpp_f<0x142, 0xa>(v, -INFINITY));
  v = fmaxf(v, dpp_f<0x143, 0xc>(v, -INFINITY));
  return __builtin_bit_cast(float, lane_value(__builtin_bit_cast(uint32_t, v), 63));
}
template <int CTRL, int ROWS> DEVI double dpp_d(double v) {
  return __builtin_bit_cast(double, dpp<CTRL, ROWS>(__builtin_bit_cast(u64, v)));
}
DEVI double wave_run(double v) {  // inclusive
  v += dpp_d<0x111, 0xf>(v);
  v += dpp_d<0x112, 0xf>(v);
  v += dpp_d<0x114, 0xf>(v);
  v += dpp_d<0x118, 0xf>(v);
  v += dpp_d<0x142, 0xa>(v);
  v += dpp_d<0x143, 0xc>(v);
  return v;
}
DEVI double lane_double(double v, int lane) {
  return __builtin_bit_cast(double, lane_value(__builtin_bit_cast(u64, v), lane));
}
DEVI double wave_add(double v) { return lane_double(wave_run(v), 63); }

// ---------------------------------------------------------------------------
// scan: workgroups of 4 wavefronts take (row, chunk) in turn
// ---------------------------------------------------------------------------
constexpr int kScan = 256, kScanWaves = kScan / 64, kVec = kChunk / (kScan * kTok);

template <typename T>
__device__ void verify_scan(const Args& a, Rec* __restrict__ rec, int* __restrict__ arrived) {
  constexpr int VW = kTok / Vec16<T>::N;  // loads a vector
  __shared__ double sums[2][kScanWaves];
  __shared__ float tops[2][kScanWaves];
  __shared__ int firsts[2][kScanWaves];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // (the next launch counts its workgroups here)
  for (int i = blockIdx.x * kScan + tid; i < a.batch; i += gridDim.x * kScan) arrived[i] = 0;
  const int n_target = a.batch * (a.k + 1);
  const int items = (n_target + (a.draft ? a.batch * a.k : 0)) * a.n_ch;
  struct Place {
    const T* row;
    int c0;   // the chunk's first column
    float t;  // the sequence's temperature, if each has its own
  };
  auto place = [&](int i) __attribute__((always_inline)) {
    const int row_i = i / a.n_ch, ch = i - row_i * a.n_ch;
    const bool is_target = row_i < n_target;
    const int per = is_target ? a.k + 1 : a.k, at = is_target ? row_i : row_i - n_target;
    const int b = at / per;
    Place p;
    p.row = is_target ? target_row<T>(a, b, at - b * per) : draft_row<T>(a, b, at - b * per);
    p.c0 = ch * kChunk - misaligned(p.row);
    p.t = a.ts ? a.ts[b] : 0.0f;
    return p;
  };
  u32x4 raw[kVec][VW];
  auto load = [&](const Place& p) __attribute__((always_inline)) {
    if (a.cols < 2 * kTok) return;
#pragma unroll
    for (int v = 0; v < kVec; ++v) {
      const T* src = p.row + vector_col(p.c0 + (v * kScan + tid) * kTok, a.cols);
#pragma unroll
      for (int w = 0; w < VW; ++w)
        raw[v][w] = *reinterpret_cast<const u32x4*>(src + w * Vec16<T>::N);
    }
  };
  int item = blockIdx.x;
  if (item >= items) return;
  Place p = place(item);
  load(p);
  for (int buf = 0; item < items; item += gridDim.x, buf ^= 1) {
    float x[kVec][kTok];
#pragma unroll
    for (int v = 0; v < kVec; ++v)
#pragma unroll
      for (int j = 0; j < kTok; ++j) {
        const uint32_t w = raw[v][j / (kTok / VW)][VW == 1 ? j / 2 : j % 4];
        x[v][j] = VW == 2 ? __builtin_bit_cast(float, w) : j & 1 ? bf16hi(w) : bf16lo(w);
      }
    if (p.c0 < 0 || p.c0 + kChunk > a.cols) {  // a row's ends one by one
#pragma unroll
      for (int v = 0; v < kVec; ++v) {
        const int c = p.c0 + (v * kScan + tid) * kTok;
        if (c < 0 || c + kTok > a.cols || a.cols < 2 * kTok)
#pragma unroll
          for (int j = 0; j < kTok; ++j)
            x[v][j] = c + j >= 0 && c + j < a.cols ? (float)p.row[c + j] : -INFINITY;
      }
    }
    const Place q = p;
    if (item + (int)gridDim.x < items) {
      p = place(item + gridDim.x);
      load(p);
    }
    const Factor f = factor_of(a, q.t);
    float mx = -INFINITY;  // (NaN: not the larger one)
#pragma unroll
    for (int v = 0; v < kVec; ++v)
#pragma unroll
      for (int j = 0; j < kTok; ++j) mx = fmaxf(mx, x[v][j]);
    mx = wave_top(mx);
    double sum = 0.0;
    uint32_t first = 0x7fffffff;
    if (f.greedy) {
#pragma unroll
      for (int v = 0; v < kVec; ++v)
#pragma unroll
        for (int j = 0; j < kTok; ++j)
          if (x[v][j] == mx) first = min(first, (uint32_t)(q.c0 + (v * kScan + tid) * kTok + j));
#pragma unroll
      for (int off = 32; off >= 1; off >>= 1) first = min(first, __shfl_xor(first, off, 64));
    } else {
      const float ref = f.ref(mx);
      float s[kVec];
      if (!fused(ref)) {
#pragma unroll
        for (int v = 0; v < kVec; ++v) {
          s[v] = 0.0f;
#pragma unroll
          for (int j = 0; j < kTok; ++j) s[v] += weight_apart(x[v][j], mx, f);
        }
      } else {
#pragma unroll
        for (int v = 0; v < kVec; ++v) {
          s[v] = 0.0f;
#pragma unroll
          for (int j = 0; j < kTok; ++j) s[v] += weight(x[v][j], ref, f);
        }
      }
#pragma unroll
      for (int v = 0; v < kVec; ++v) sum += (double)s[v];
      sum = wave_add(sum);
    }
    if (lane == 0) {
      sums[buf][wave] = sum;
      tops[buf][wave] = mx;
      firsts[buf][wave] = (int)first;
    }
    // (the loads in flight are not waited for: the barrier alone, after the LDS writes)
    __builtin_amdgcn_s_waitcnt(15 | (3 << 14) | (7 << 4));
    asm volatile("s_barrier" ::: "memory");
    // (the buffers alternate: the next barrier comes before this one's next write)
    if (tid == 0) {
      float top = tops[buf][0];
#pragma unroll
      for (int w = 1; w < kScanWaves; ++w) top = fmaxf(top, tops[buf][w]);
      Rec r{0.0, top, 0x7fffffff};
#pragma unroll
      for (int w = kScanWaves - 1; w >= 0; --w) {
        r.sum += f.greedy ? 0.0 : sums[buf][w] * (double)below(tops[buf][w], top, f);
        if (tops[buf][w] == top) r.first = min(r.first, firsts[buf][w]);
      }
      rec[item] = r;
    }
  }
}

// A row's maximum and sum of weights from its chunks' (by a wavefront, a lane a chunk).
struct Row {
  double sum;
  float xmax;
  int first;  // greedy: the token
};
DEVI Row row_of(const Rec& r, const Factor& f) {
  Row o;
  o.xmax = wave_top(r.xmax);
  o.first = 0x7fffffff;
  o.sum = 0.0;
  if (f.greedy) {
    const u64 has = __ballot(r.xmax == o.xmax);
    o.first = (int)lane_value((uint32_t)r.first, __builtin_ctzll(has));  // the first chunk's
    return o;
  }
  o.sum = wave_add(r.sum * (double)below(r.xmax, o.xmax, f));
  return o;
}
// The probability of token `col` with logit x
DEVI double prob(float x, int col, const Row& r, const Factor& f) {
  if (f.greedy) return r.xmax > -INFINITY && col == r.first ? 1.0 : 0.0;
  if (!(x > -INFINITY) || !(r.sum > 0.0)) return 0.0;
  if (r.xmax == INFINITY) return x == INFINITY ? 1.0 / r.sum : 0.0;
  return exp2((double)x * (double)f.c - ref_of(r.xmax, f)) / r.sum;
}

// What the token after the accepted ones is drawn from: max(p_n - q_n, 0), or p_n.
struct Rest {
  int n;         // accepted
  int skip;      // the refused draft; -1: none
  bool minus_q;  // p_n - q_n, of scaled weights; else p_n's weights without `skip`
  bool greedy;
  int first;     // greedy: the token
  float pmax, qmax, pref, qref, ap, aq;
};
// Scaled weights' difference, each rounded first: equal ones leave nothing.
DEVI float surplus(float p, float ap, float q, float aq) {
#pragma clang fp contract(off)
  return fmaxf(p * ap - q * aq, 0.0f);
}
struct RestSmem {
  Row row[2 * kMaxDrafts + 1];  // target rows, then the draft model's
};
// by all wavefronts of a workgroup
template <typename T>
DEVI Rest rest_of(const Args& a, const Rec* rec, int b, const Factor& f, RestSmem& sm) {
  constexpr int U = 3;  // rows of a wavefront whose records are asked for at once
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // a lane a draft: the drafts that are tokens, up to the first that is none, their
  // logits and random numbers
  const int mine = min(lane, a.k - 1);
  const long long d64 = a.drafts[(long)b * a.k + mine];
  const bool ok = lane < a.k && d64 >= 0 && d64 < a.cols;
  const u64 all = __ballot(ok);
  const int real = all == ~0ull ? 64 : __builtin_ctzll(~all);
  const int d = ok ? (int)d64 : 0;
  const float u = a.u[(long)b * (a.k + 1) + mine];
  const float x = (float)target_row<T>(a, b, mine)[d];
  const float y = a.draft ? (float)draft_row<T>(a, b, mine)[d] : 0.0f;
  // (all rows, whatever the drafts are: these loads do not wait for them)
  const int rows = a.k + 1 + (a.draft ? a.k : 0);
  for (int r0 = wave; r0 < rows; r0 += U * kWaves) {
    Rec r[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int t = r0 + i * kWaves;
      r[i] = Rec{0.0, -INFINITY, 0x7fffffff};
      if (t < rows && lane < a.n_ch)
        r[i] = (t <= a.k ? target_rec(a, rec, b, t) : draft_rec(a, rec, b, t - a.k - 1))[lane];
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (r0 + i * kWaves >= rows) break;
      const Row o = row_of(r[i], f);
      if (lane == 0) sm.row[r0 + i * kWaves] = o;
    }
  }
  __syncthreads();
  bool passed = false;
  if (lane < real) {
    const double q = a.draft ? prob(y, d, sm.row[a.k + 1 + lane], f) : 1.0;
    passed = (double)u * q < prob(x, d, sm.row[lane], f);
  }
  Rest r;
  const u64 yes = __ballot(passed);
  r.n = yes == ~0ull ? 64 : __builtin_ctzll(~yes);
  r.skip = r.n < real ? __builtin_amdgcn_readlane(d, r.n) : -1;
  const Row p = sm.row[r.n];
  r.greedy = f.greedy;
  r.first = p.xmax > -INFINITY ? p.first : -1;
  r.pmax = p.xmax;
  r.minus_q = a.draft && r.skip >= 0;
  r.ap = p.sum > 0.0 ? (float)(1.0 / p.sum) : 0.0f;
  r.qmax = 0.0f;
  r.aq = 0.0f;
  if (r.minus_q) {
    const Row q = sm.row[a.k + 1 + r.n];
    r.qmax = q.xmax;
    r.aq = q.sum > 0.0 ? (float)(1.0 / q.sum) : 0.0f;
  }
  r.pref = f.ref(r.pmax);
  r.qref = f.ref(r.qmax);
  return r;
}
// The weight of column c, logits x and y
DEVI float weigh_one(float x, float y, int c, const Rest& r, const Factor& f) {
  float z = weight(x, r.pmax, r.pref, f);
  if (r.minus_q) z = surplus(z, r.ap, weight(y, r.qmax, r.qref, f), r.aq);
  return c == r.skip ? 0.0f : z;
}
// The sum of a thread's 16 columns of a chunk: those from 16 tid on, in the draft's row
// wherever they lie in memory (rows of an odd number of columns: 48 sequences of 8 drafts
// of 128255 97 us with such columns one by one, 67 so)
typedef uint32_t u32x4any __attribute__((ext_vector_type(4), aligned(2)));
template <typename T>
DEVI double weigh(const T* prow, const T* qrow, int cols, int ch, const Rest& r, const Factor& f) {
  constexpr int VW = kTok / Vec16<T>::N;
  const int c0 = ch * kChunk - misaligned(prow) + 2 * kTok * (int)threadIdx.x;
  double sum = 0.0;
  if (c0 >= 0 && c0 + 2 * kTok <= cols && fused(r.pref) && fused(r.qref)) {
    u32x4 x[2 * VW], y[2 * VW];
#pragma unroll
    for (int v = 0; v < 2 * VW; ++v) x[v] = reinterpret_cast<const u32x4*>(prow + c0)[v];
    if (r.minus_q)
#pragma unroll
      for (int v = 0; v < 2 * VW; ++v) y[v] = reinterpret_cast<const u32x4any*>(qrow + c0)[v];
    auto at = [](const u32x4* z, int j) __attribute__((always_inline)) {
      const uint32_t w = VW == 2 ? z[j / 4][j % 4] : z[j / 8][j % 8 / 2];
      return VW == 2 ? __builtin_bit_cast(float, w) : j & 1 ? bf16hi(w) : bf16lo(w);
    };
    // sums of eight in fp32
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      float part = 0.0f;
      if (r.minus_q) {
#pragma unroll
        for (int j = v * kTok; j < (v + 1) * kTok; ++j) {
          const float z = surplus(weight(at(x, j), r.pref, f), r.ap,
                                  weight(at(y, j), r.qref, f), r.aq);
          part += c0 + j == r.skip ? 0.0f : z;
        }
      } else {
#pragma unroll
        for (int j = v * kTok; j < (v + 1) * kTok; ++j) {
          const float z = weight(at(x, j), r.pref, f);
          part += c0 + j == r.skip ? 0.0f : z;
        }
      }
      sum += (double)part;
    }
  } else {
    // a row's ends, and references too large to fuse: four columns' loads at a time
#pragma unroll 1
    for (int j = c0; j < c0 + 2 * kTok; j += 4) {
      float x[4], y[4] = {};
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = (float)prow[max(min(j + i, cols - 1), 0)];
      if (r.minus_q)
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = (float)qrow[max(min(j + i, cols - 1), 0)];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (j + i >= 0 && j + i < cols) sum += (double)weigh_one(x[i], y[i], j + i, r, f);
    }
  }
  return sum;
}

// grid (chunks, sequences)
template <typename T>
__device__ void verify_rest(const Args& a, const Rec* __restrict__ rec, double* __restrict__ part,
                            int* __restrict__ arrived, long long* __restrict__ tokens,
                            int* __restrict__ accepted) {
  __shared__ RestSmem sm;
  __shared__ double sums[kWaves];
  __shared__ int count, has[2][kWaves];
  const int tid = threadIdx.x, lane = tid & 63, b = blockIdx.y, n_ch = gridDim.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Factor f = factor_of(a, b);
  Rest r = rest_of<T>(a, rec, b, f, sm);
  long long* out = tokens + (long)b * (a.k + 1);
  if (blockIdx.x == 0) {
    if (tid <= a.k && (tid != r.n || r.greedy))
      out[tid] = tid < r.n ? a.drafts[(long)b * a.k + tid] : tid == r.n ? r.first : -1;
    if (tid == 0) accepted[b] = r.n;
  }
  if (r.greedy) return;
  // p_n's own weights: one workgroup draws, the scan has the sums of the chunks, but that of
  // the refused draft's chunk without it (1 sequence 8.1 -> 6.6 us)
  const bool alone = !r.minus_q;
  if (alone && blockIdx.x > 0) return;
  const T* prow = target_row<T>(a, b, r.n);
  const T* qrow = r.minus_q ? draft_row<T>(a, b, r.n) : prow;
  const Rec* prec = target_rec(a, rec, b, r.n) + min(lane, n_ch - 1);
  // Twice through one body (code that runs once is fetched from memory as it goes): the
  // workgroup's own chunk, then, by the last workgroup of the sequence, the drawn one.
  int ch = !alone ? blockIdx.x : r.skip < 0 ? -1 : (r.skip + misaligned(prow)) / kChunk;
  double target = 0.0;
#pragma unroll 1
  for (int pass = 0;; ++pass) {
    double mine = 0.0, run = 0.0;
    double before = 0.0, all = 0.0;  // sums before the wavefront's; of the chunk
    if (ch >= 0) {
      mine = weigh<T>(prow, qrow, a.cols, ch, r, f);
      run = wave_run(mine);
      if (lane == 63) sums[wave] = run;
      __syncthreads();
      for (int i = 0; i < kWaves; ++i) {
        before += i < wave ? sums[i] : 0.0;
        all += sums[i];
      }
    }
    if (pass == 1) {
      // the thread that the target falls into (rounding may leave none: the last that has any)
      const double lo = before + run - mine;
      const u64 at = __ballot(mine > 0.0 && lo + mine > target), any = __ballot(mine > 0.0);
      __syncthreads();
      if (lane == 0) has[0][wave] = at ? 1 : 0, has[1][wave] = any ? 1 : 0;
      __syncthreads();
      int w = -1, z = -1;
      for (int i = kWaves - 1; i >= 0; --i) {
        if (has[0][i]) w = i;
        if (has[1][i]) z = max(z, i);
      }
      if (wave != (w >= 0 ? w : z)) return;
      const int l = at ? __builtin_ctzll(at) : 63 - __builtin_clzll(any);
      const double t = target - lane_double(lo, l);
      const int c = ch * kChunk - misaligned(prow) + 2 * kTok * (wave * 64 + l) + lane;
      double v = 0.0;
      if (lane < 2 * kTok && c >= 0 && c < a.cols)
        v = (double)weigh_one((float)prow[c], (float)qrow[c], c, r, f);
      const double upto = wave_run(v);
      const u64 hit = __ballot(v > 0.0 && upto > t), some = __ballot(v > 0.0);
      if (lane == (hit ? __builtin_ctzll(hit) : 63 - __builtin_clzll(some))) out[r.n] = c;
      return;
    }
    if (tid == 0 && !alone) {
      // Store, count and the last one's loads are accesses of device scope, past the L2
      // caches; the store has been performed before the count is sent.  (Release and
      // acquire would write back and drop a whole L2 in every workgroup.)
      __hip_atomic_store(part + (long)b * kMaxChunks + ch, all, __ATOMIC_RELAXED,
                         __HIP_MEMORY_SCOPE_AGENT);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      count = __hip_atomic_fetch_add(arrived + b, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!alone && count != n_ch - 1) return;
    // every wavefront finds the chunk for itself
    auto scanned = [&] { return lane < n_ch ? prec->sum * (double)below(prec->xmax, r.pmax, f) : 0.0; };
    double s;
    if (alone)
      s = lane == ch ? all : scanned();
    else
      s = lane < n_ch ? __hip_atomic_load(part + (long)b * kMaxChunks + lane, __ATOMIC_RELAXED,
                                          __HIP_MEMORY_SCOPE_AGENT) : 0.0;
    double at = wave_run(s), whole = lane_double(at, 63);
    if (!(whole > 0.0)) {  // p_n lies below q_n everywhere: then p_n itself
      s = scanned();
      at = wave_run(s);
      whole = lane_double(at, 63);
      r.minus_q = false;
      r.skip = -1;
    }
    const float u = a.u[(long)b * (a.k + 1) + a.k];
    const double t = u > 0.0f ? (double)u * whole : 0.0;
    // the first chunk past it; u of 1: the last that has any
    const u64 yes = __ballot(s > 0.0 && at > t), any = __ballot(s > 0.0);
    if (!any) {  // no token to draw
      if (tid == 0) out[r.n] = -1;
      return;
    }
    ch = yes ? __builtin_ctzll(yes) : 63 - __builtin_clzll(any);
    target = t - lane_double(at - s, ch);
  }
}

}  // namespace

#define TEENY_VERIFY_INST(TN, T)                                                                 \
  extern "C" __global__ __launch_bounds__(256) void teeny_verify_scan_##TN(Args a, Rec* rec,      \
                                                                           int* arrived) {        \
    verify_scan<T>(a, rec, arrived);                                                             \
  }                                                                                              \
  extern "C" __global__ __launch_bounds__(512) void teeny_verify_rest_##TN(                      \
      Args a, const Rec* rec, double* part, int* arrived, long long* tokens, int* accepted) {     \
    verify_rest<T>(a, rec, part, arrived, tokens, accepted);                                     \
  }
TEENY_VERIFY_INST(f32, float)
TEENY_VERIFY_INST(bf16, bf16)
