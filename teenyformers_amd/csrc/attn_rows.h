// The running state of a wavefront's 32 query rows in bf16 attention over 32-key
// tiles in LDS, as the kernels with shares of the keys use it (prefix_attn.hip,
// paged.hip).
#pragma once
#include "cdna4.h"

constexpr int TK = 32;  // keys per tile
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kVmcnt0 = (7 << 4) | (15 << 8);
constexpr int kLgkmcnt0 = 15 | (3 << 14) | (7 << 4);

// The running state of a wavefront's 32 rows (one per lane % 32, as in the
// forward kernel: S^T = K Q^T, O^T += V^T P^T).
template <int D>
struct Rows {
  static constexpr int DC = D / 16, DT = D / 32, CPR = D / 8;
  bf16x8 q[DC];
  f32x16 acc[DT];
  float m, l;
  int k_off[DC], v_off[DT][2];

  DEVI void init() {
    const int lane = threadIdx.x & 63, l32 = lane & 31, g = lane >> 5;
#pragma unroll
    for (int t = 0; t < DT; ++t) acc[t] = f32x16{};
    m = -INFINITY;
    l = 0.0f;
#pragma unroll
    for (int c = 0; c < DC; ++c) k_off[c] = swz<SWZ_ROW, D>(l32 * CPR + 2 * c + g) * 16;
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = 8 * e + 4 * g + ((lane & 15) >> 2);
        const int col = 32 * t + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
        v_off[t][e] = swz<SWZ_DUAL, D>(row * CPR + col / 8) * 16 + (col % 8) * 2;
      }
  }
  // the lane's row of q, or zeros
  DEVI void load_q(const bf16* row, bool valid) {
    const int g = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int c = 0; c < DC; ++c)
      q[c] = valid ? as_bf16x8(*reinterpret_cast<const u32x4*>(row + 16 * c + 8 * g))
                   : as_bf16x8(u32x4{0, 0, 0, 0});
  }
  DEVI f32x16 scores(const char* kt) {
    u32x4 kr[DC];
#pragma unroll
    for (int c = 0; c < DC; ++c) kr[c] = *reinterpret_cast<const u32x4*>(kt + k_off[c]);
    f32x16 s = f32x16{};
#pragma unroll
    for (int c = 0; c < DC; ++c) s = mfma32(as_bf16x8(kr[c]), q[c], s);
    sched_group(kDsRead, DC);
    sched_group(kMfma, DC);
    return s;
  }
  // keys of the tile at or past lim (the lane's own) do not count
  DEVI void mask(f32x16& s, int lim) {
    const int g = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int r = 0; r < 16; ++r)
      if (8 * (r >> 2) + 4 * g + (r & 3) >= lim) s[r] = -INFINITY;
  }
  // P of the tile as the operand of its product with V
  DEVI void softmax(const f32x16& s, float sl2, uint32_t* pb) {
    float mx = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
    mx = fmaxf(mx, other_half(mx)) * sl2;
    if (__any(mx > m)) {  // wave-uniform
      const float m_new = fmaxf(m, mx);
      const float alpha = m_new == -INFINITY ? 1.0f : fast_exp2(m - m_new);
      m = m_new;
      l *= alpha;
#pragma unroll
      for (int t = 0; t < DT; ++t) acc[t] *= alpha;
    }
    const float ref = m == -INFINITY ? 0.0f : m;  // a row without a key so far
#pragma unroll
    for (int r = 0; r < 16; r += 2) {
      pb[r >> 1] = pack_bf16x2(fast_exp2(__builtin_fmaf(s[r], sl2, -ref)),
                               fast_exp2(__builtin_fmaf(s[r + 1], sl2, -ref)));
      l = add_bf16x2(pb[r >> 1], l);
    }
  }
  DEVI void read_v(const char* vt, u32x4 (*va)[DT]) {
#pragma unroll
    for (int hh = 0; hh < 2; ++hh)
#pragma unroll
      for (int t = 0; t < DT; ++t) {
        const char* p = vt + hh * 16 * D * 2;
        const u32x2 a0 = lds_read_tr(p + v_off[t][0]), a1 = lds_read_tr(p + v_off[t][1]);
        va[hh][t] = u32x4{a0[0], a0[1], a1[0], a1[1]};
      }
  }
  DEVI void product(const u32x4 (*va)[DT], const uint32_t* pb) {
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      const bf16x8 bop =
          as_bf16x8(u32x4{pb[4 * hh], pb[4 * hh + 1], pb[4 * hh + 2], pb[4 * hh + 3]});
#pragma unroll
      for (int t = 0; t < DT; ++t) acc[t] = mfma32(as_bf16x8(va[hh][t]), bop, acc[t]);
    }
  }
};
