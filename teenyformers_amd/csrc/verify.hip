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
// Numbers: weights are fp32 (2^((x - max) log2(e) / T), the factor in two parts:
// 1e-7 relative), sums of eight in fp32 and from there in fp64; what decides
// (acceptance, the place of u among running sums) is fp64.  A draw from one row sums
// unscaled weights, exact for equal logits.  No atomics: one order of sums.
//
//   scan   (chunk, row): the maximum of a chunk of 8192 columns and its weights' sum
//          below it.  Reading the rows bounds it; rows behind a sequence's last real
//          draft are not read.
//   rest   (chunk, sequence): each workgroup finds the sequence's accepted drafts from
//          the chunks' sums (a wavefront a draft, a lane a chunk) and sums its chunk of
//          what the next token is drawn from.
//   pick   (sequence): the chunk and the token.
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

// log2(e) / T (0: greedy) in two parts
struct Factor {
  double c;
  float hi, lo;
  bool greedy;
};
DEVI Factor factor_of(const Args& a, int b) {
  const double t = a.ts ? (double)a.ts[b] : a.t;
  Factor f;
  f.greedy = !(t > 0.0);  // (NaN too)
  f.c = f.greedy ? kLog2e : kLog2e / t;
  f.hi = (float)f.c;
  f.lo = (float)(f.c - (double)f.hi);
  return f;
}
// The weight of x below xmax, 0 .. 1
DEVI float weight(float x, float xmax, const Factor& f) {
  const float d = x - xmax;
  const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(d, f.hi, d * f.lo));
  return !(x > -INFINITY) ? 0.0f : x == xmax ? 1.0f : w == w ? w : 0.0f;
}

// The drafts of sequence b that are tokens, up to the first that is none.
DEVI int real_drafts(const Args& a, int b) {
  const int lane = threadIdx.x & 63;
  const long long d = lane < a.k ? a.drafts[(long)b * a.k + lane] : -1;
  const u64 ok = __ballot(d >= 0 && d < a.cols);
  return ok == ~0ull ? 64 : __builtin_ctzll(~ok);
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

DEVI double wave_add(double v) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// ---------------------------------------------------------------------------
template <typename T>
__device__ void verify_scan(const Args& a, Rec* __restrict__ rec) {
  __shared__ float red[kWaves];
  __shared__ double sums[kWaves];
  __shared__ int firsts[kWaves];
  const int tid = threadIdx.x, lane = tid & 63, ch = blockIdx.x, row_i = blockIdx.y;
  const int n_target = a.batch * (a.k + 1);
  const bool is_target = row_i < n_target;
  const int per = is_target ? a.k + 1 : a.k, at = is_target ? row_i : row_i - n_target;
  const int b = at / per, i = at - b * per;
  const T* row = is_target ? target_row<T>(a, b, i) : draft_row<T>(a, b, i);
  const int real = real_drafts(a, b);
  if (i > real || (!is_target && i == real)) return;  // (uniform)
  const int mis = misaligned(row);
  float x[2][kTok];
  int col[2];
#pragma unroll
  for (int v = 0; v < 2; ++v) col[v] = load8(row, a.cols, mis, ch, v * kThreads + tid, x[v]);
  const Factor f = factor_of(a, b);
  float mx = -INFINITY;
#pragma unroll
  for (int v = 0; v < 2; ++v)
#pragma unroll
    for (int j = 0; j < kTok; ++j) mx = fmaxf(mx, x[v][j]);
  mx = wave_max(mx);
  if (lane == 0) red[tid >> 6] = mx;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) mx = fmaxf(mx, red[w]);
  double sum = 0.0;
  int first = 0x7fffffff;
#pragma unroll
  for (int v = 0; v < 2; ++v) {
    if (f.greedy) {
#pragma unroll
      for (int j = kTok - 1; j >= 0; --j)
        if (x[v][j] == mx) first = min(first, col[v] + j);
    } else {
      float s = 0.0f;
#pragma unroll
      for (int j = 0; j < kTok; ++j) s += weight(x[v][j], mx, f);
      sum += (double)s;
    }
  }
  if (f.greedy) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) first = min(first, __shfl_xor(first, off, 64));
  } else {
    sum = wave_add(sum);
  }
  if (lane == 0) {
    sums[tid >> 6] = sum;
    firsts[tid >> 6] = first;
  }
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kWaves; ++w) {
      sum += sums[w];
      first = min(first, firsts[w]);
    }
    rec[(long)row_i * a.n_ch + ch] = Rec{sum, mx, first};
  }
}

// A row's maximum and sum of weights from its chunks' (by a wavefront, a lane a chunk).
struct Row {
  double sum;
  float xmax;
  int first;  // greedy: the token
};
DEVI Row row_of(const Rec* rec, int n_ch, const Factor& f) {
  const int lane = threadIdx.x & 63;
  Rec r{0.0, -INFINITY, 0x7fffffff};
  if (lane < n_ch) r = rec[lane];
  Row o;
  o.xmax = wave_max(r.xmax);
  o.first = 0x7fffffff;
  o.sum = 0.0;
  if (f.greedy) {
    const u64 has = __ballot(r.xmax == o.xmax);
    o.first = (int)lane_value((uint32_t)r.first, __builtin_ctzll(has));  // the first chunk's
    return o;
  }
  const double d = r.xmax == o.xmax ? 0.0 : ((double)r.xmax - (double)o.xmax) * f.c;
  o.sum = wave_add(r.xmax > -INFINITY && d == d ? r.sum * exp2(d) : 0.0);
  return o;
}
template <typename T>
DEVI double prob(const T* row, int col, const Row& r, const Factor& f) {
  if (f.greedy) return r.xmax > -INFINITY && col == r.first ? 1.0 : 0.0;
  const float x = (float)row[col];
  if (!(x > -INFINITY) || !(r.sum > 0.0)) return 0.0;
  const double w = x == r.xmax ? 1.0 : exp2(((double)x - (double)r.xmax) * f.c);
  return w == w ? w / r.sum : 0.0;
}

// What the token after the accepted ones is drawn from: max(p_n - q_n, 0), or p_n.
struct Rest {
  int n;         // accepted
  int skip;      // the refused draft; -1: none
  bool minus_q;  // p_n - q_n, of scaled weights; else p_n's weights without `skip`
  bool greedy;
  int first;     // greedy: the token
  float pmax, qmax;
  double ap, aq;
};
struct RestSmem {
  double sum[kMaxDrafts + 1], q_sum[kMaxDrafts];
  float xmax[kMaxDrafts + 1], q_xmax[kMaxDrafts];
  int first[kMaxDrafts + 1];
  int passed[kMaxDrafts + 1];
};
// by all wavefronts of a workgroup
template <typename T>
DEVI Rest rest_of(const Args& a, const Rec* rec, int b, const Factor& f, RestSmem& sm) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int real = real_drafts(a, b);
  for (int i = wave; i <= real; i += waves) {
    const Row p = row_of(target_rec(a, rec, b, i), a.n_ch, f);
    Row q{};
    int passed = 0;
    if (i < real) {
      const int d = (int)a.drafts[(long)b * a.k + i];
      double qd = 1.0;
      if (a.draft) {
        q = row_of(draft_rec(a, rec, b, i), a.n_ch, f);
        qd = prob(draft_row<T>(a, b, i), d, q, f);
      }
      passed = (double)a.u[(long)b * (a.k + 1) + i] * qd < prob(target_row<T>(a, b, i), d, p, f);
      if (lane == 0) {
        sm.q_sum[i] = q.sum;
        sm.q_xmax[i] = q.xmax;
      }
    }
    if (lane == 0) {
      sm.sum[i] = p.sum;
      sm.xmax[i] = p.xmax;
      sm.first[i] = p.first;
      sm.passed[i] = passed;
    }
  }
  __syncthreads();
  Rest r;
  r.n = 0;
  while (r.n < real && sm.passed[r.n]) ++r.n;
  r.skip = r.n < real ? (int)a.drafts[(long)b * a.k + r.n] : -1;
  r.greedy = f.greedy;
  r.first = sm.xmax[r.n] > -INFINITY ? sm.first[r.n] : -1;
  r.pmax = sm.xmax[r.n];
  r.minus_q = a.draft && r.skip >= 0;
  r.qmax = r.minus_q ? sm.q_xmax[r.n] : 0.0f;
  r.ap = sm.sum[r.n] > 0.0 ? 1.0 / sm.sum[r.n] : 0.0;
  r.aq = r.minus_q && sm.q_sum[r.n] > 0.0 ? 1.0 / sm.q_sum[r.n] : 0.0;
  return r;
}
// A thread's 16 columns of a chunk and their weights; their sum
template <typename T>
DEVI double weigh(const Args& a, int b, int ch, const Rest& r, const Factor& f, double (*w)[kTok],
                  int* col) {
  const T* prow = target_row<T>(a, b, r.n);
  const T* qrow = r.minus_q ? draft_row<T>(a, b, r.n) : prow;
  float x[2][kTok], y[2][kTok];
  // (vectors of the two rows begin at other columns where they are aligned otherwise:
  // q's columns are then read one by one)
  const int mis = misaligned(prow), qmis = r.minus_q ? misaligned(qrow) : mis;
#pragma unroll
  for (int v = 0; v < 2; ++v) col[v] = load8(prow, a.cols, mis, ch, 2 * (int)threadIdx.x + v, x[v]);
  if (r.minus_q) {
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      if (qmis == mis) {
        load8(qrow, a.cols, mis, ch, 2 * (int)threadIdx.x + v, y[v]);
      } else {
#pragma unroll
        for (int j = 0; j < kTok; ++j) {
          const int c = col[v] + j;
          y[v][j] = c >= 0 && c < a.cols ? fmaxf((float)qrow[c] + 0.0f, -INFINITY) : -INFINITY;
        }
      }
    }
  }
  double sum = 0.0;
#pragma unroll
  for (int v = 0; v < 2; ++v)
#pragma unroll
    for (int j = 0; j < kTok; ++j) {
      double z = (double)weight(x[v][j], r.pmax, f);
      if (r.minus_q) z = fmax(z * r.ap - (double)weight(y[v][j], r.qmax, f) * r.aq, 0.0);
      if (col[v] + j == r.skip) z = 0.0;
      w[v][j] = z;
      sum += z;
    }
  return sum;
}

template <typename T>
__device__ void verify_rest(const Args& a, const Rec* __restrict__ rec, double* __restrict__ part) {
  __shared__ RestSmem sm;
  __shared__ double sums[kWaves];
  const int tid = threadIdx.x, ch = blockIdx.x, b = blockIdx.y;
  const Factor f = factor_of(a, b);
  const Rest r = rest_of<T>(a, rec, b, f, sm);
  if (r.greedy) return;
  double w[2][kTok];
  int col[2];
  const double sum = wave_add(weigh<T>(a, b, ch, r, f, w, col));
  if ((tid & 63) == 0) sums[tid >> 6] = sum;
  __syncthreads();
  if (tid == 0) {
    double s = 0.0;
    for (int i = 0; i < kWaves; ++i) s += sums[i];
    part[(long)b * kMaxChunks + ch] = s;
  }
}

// inclusive over the wavefront
DEVI double wave_run(double v) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const double o = __shfl_up(v, off, 64);
    v += (int)(threadIdx.x & 63) >= off ? o : 0.0;
  }
  return v;
}

template <typename T>
__device__ void verify_pick(const Args& a, const Rec* __restrict__ rec,
                            const double* __restrict__ part, long long* __restrict__ tokens,
                            int* __restrict__ accepted) {
  __shared__ RestSmem sm;
  __shared__ double sums[kWaves];
  __shared__ int found, last, chunk;
  __shared__ double target;
  const int tid = threadIdx.x, lane = tid & 63, b = blockIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Factor f = factor_of(a, b);
  Rest r = rest_of<T>(a, rec, b, f, sm);
  long long* out = tokens + (long)b * (a.k + 1);
  if (tid <= a.k && tid != r.n) out[tid] = tid < r.n ? a.drafts[(long)b * a.k + tid] : -1;
  if (tid == 0) accepted[b] = r.n;
  if (r.greedy) {
    if (tid == 0) out[r.n] = r.first;
    return;
  }
  if (wave == 0) {
    double s = lane < a.n_ch ? part[(long)b * kMaxChunks + lane] : 0.0;
    double run = wave_run(s), all = __shfl(run, 63);
    const bool none = !(all > 0.0);
    if (none) {  // p_n lies below q_n everywhere: then p_n itself
      const Rec* t = target_rec(a, rec, b, r.n);
      const double d = lane < a.n_ch ? ((double)t[lane].xmax - (double)r.pmax) * f.c : 0.0;
      s = lane < a.n_ch && t[lane].xmax > -INFINITY
              ? t[lane].sum * (t[lane].xmax == r.pmax ? 1.0 : d == d ? exp2(d) : 0.0) : 0.0;
      run = wave_run(s);
      all = __shfl(run, 63);
    }
    const float u = a.u[(long)b * (a.k + 1) + a.k];
    const double t = u > 0.0f ? (double)u * all : 0.0;
    u64 at = __ballot(s > 0.0 && run > t);  // the first; u of 1: the last that has any
    const u64 any = __ballot(s > 0.0);
    const int ch = at ? __builtin_ctzll(at) : any ? 63 - __builtin_clzll(any) : -1;
    if (lane == 0) {
      chunk = ch | (none ? 1 << 16 : 0);
      found = 0x7fffffff;
      last = -1;
    }
    if (ch >= 0) {
      const double before = __shfl(run - s, ch);
      if (lane == 0) target = t - before;
    }
  }
  __syncthreads();
  if (chunk < 0) {  // no token to draw
    if (tid == 0) out[r.n] = -1;
    return;
  }
  if (chunk >> 16) {
    r.minus_q = false;
    r.skip = -1;
  }
  double w[2][kTok];
  int col[2];
  const double sum = weigh<T>(a, b, chunk & 0xffff, r, f, w, col), inc = wave_run(sum);
  if (lane == 63) sums[wave] = inc;
  __syncthreads();
  double run = inc - sum;
  for (int i = 0; i < wave; ++i) run += sums[i];
  int mine = 0x7fffffff, top = -1;
#pragma unroll
  for (int v = 0; v < 2; ++v)
#pragma unroll
    for (int j = 0; j < kTok; ++j) {
      run += w[v][j];
      if (w[v][j] > 0.0) {
        top = col[v] + j;
        if (run > target) mine = min(mine, top);
      }
    }
  if (mine < 0x7fffffff) atomicMin(&found, mine);
  if (top >= 0) atomicMax(&last, top);
  __syncthreads();
  if (tid == 0) out[r.n] = found < 0x7fffffff ? found : last;
}

}  // namespace

#define TEENY_VERIFY_INST(TN, T)                                                                 \
  extern "C" __global__ __launch_bounds__(512) void teeny_verify_scan_##TN(Args a, Rec* rec) {    \
    verify_scan<T>(a, rec);                                                                      \
  }                                                                                              \
  extern "C" __global__ __launch_bounds__(512) void teeny_verify_rest_##TN(Args a, const Rec* rec, \
                                                                           double* part) {        \
    verify_rest<T>(a, rec, part);                                                                \
  }                                                                                              \
  extern "C" __global__ __launch_bounds__(512) void teeny_verify_pick_##TN(                      \
      Args a, const Rec* rec, const double* part, long long* tokens, int* accepted) {             \
    verify_pick<T>(a, rec, part, tokens, accepted);                                              \
  }
TEENY_VERIFY_INST(f32, float)
TEENY_VERIFY_INST(bf16, bf16)
