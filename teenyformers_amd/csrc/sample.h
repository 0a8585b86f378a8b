// A row of logits in chunks, and wavefront sums: what the kernels that draw tokens
// share (sample.hip, verify.hip).
#pragma once
#include "chunks.h"
#include "common.h"

typedef unsigned long long u64;

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
