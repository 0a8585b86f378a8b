// A cache in pages: [n_pages, Hkv, 2^lg rows, D], key j of sequence b in row
// j % 2^lg of page table[b ld + (j >> lg)].  Entries outside [0, n_pages) are
// absent pages: nothing is read from them or written to them, and their keys do
// not count.  The new tokens of all sequences are packed: those of sequence b are
// tokens starts[b] .. starts[b + 1] - 1 (starts null: `each` tokens a sequence),
// token i of them at position past[b] + i (past null: past_all).
#pragma once
#include "cdna4.h"

struct Paged {
  const int *table, *starts, *past;
  int batch, tokens, each, past_all;
  int ld, width, n_pages, lg;  // table: row stride, pages of a sequence
  int hq, hkv;
};

// What a kernel knows of a sequence, bounded whatever the device arrays hold: tokens t0 ..
// t0 + n - 1 lie in the batch (none where its starts do not, or fall), and every count of
// keys in the table.
struct Seq {
  int t0, n, past, cap;
  // keys that the sequence's first i + 1 new tokens see
  DEVI int keys(int i) const { return min(max(past + i + 1, 0), cap); }
};
DEVI Seq seq_of(const Paged& a, int b) {
  Seq s;
  const int t0 = a.starts ? a.starts[b] : b * a.each;
  const int t1 = a.starts ? a.starts[b + 1] : t0 + a.each;
  const bool in = t0 >= 0 && t0 <= t1 && t1 <= a.tokens;
  s.t0 = in ? t0 : 0;
  s.n = in ? t1 - t0 : 0;
  s.cap = a.width << a.lg;
  s.past = min(max(a.past ? a.past[b] : a.past_all, -a.tokens), s.cap);
  return s;
}
// The sequence of token t (wave-uniform), the first that has it as seq_of sees it, whatever
// the starts of others are; -1: none.  A wavefront looks at 64 sequences at a time.
DEVI int seq_at(const Paged& a, int t) {
  if (!a.starts) return t < a.batch * a.each ? t / a.each : -1;
  const int lane = threadIdx.x & 63;
  for (int i = 0; i < a.batch; i += 64) {
    const int b = min(i + lane, a.batch - 1), t0 = a.starts[b], t1 = a.starts[b + 1];
    const uint64_t has = __ballot(t0 >= 0 && t0 <= t && t < t1 && t1 <= a.tokens);
    if (has) return i + (int)__builtin_ctzll(has);
  }
  return -1;
}

// A wavefront's way along a sequence's table: 64 entries in a register, the first ones
// asked for at once (a short sequence's, beside the loads of its length).
struct PageWalk {
  const int* row;
  int width, n_pages, first, mine;
  DEVI PageWalk(const Paged& a, int b)
      : row(a.table + (long)b * a.ld), width(a.width), n_pages(a.n_pages), first(0) {
    const int j = threadIdx.x & 63;
    mine = row[min(j, width - 1)];
    if (j >= width || (unsigned)mine >= (unsigned)n_pages) mine = -1;
  }
  // the page of table entry i (wave-uniform); -1: absent
  DEVI int at(int i) {
    if ((unsigned)(i - first) >= 64u) {
      first = i;
      const int j = i + lane_now();
      mine = j < width ? row[j] : -1;
      if ((unsigned)mine >= (unsigned)n_pages) mine = -1;
      pin(mine);  // waited for here: after the branch every use would wait for the tiles in flight
    }
    return __builtin_amdgcn_readlane(mine, i - first);
  }
};

// The kv head of a workgroup and its place among per_head of that head; false: none.
// XCDs take heads of their own, or groups of 2, 4 or 8 share some, and their heads' places
// in turn: a head's keys pass few L2 caches, and where a head's long rows come first, every
// XCD and CU gets long and short ones.  us of bf16 chunks with runs of a head's places by
// XCD and so: 2048 tokens behind 6144, Hq32 Hkv4 296, 254, Hq16 Hkv16 175, 163; 3548 behind
// 0, Hq32 Hkv4 168, 129, Hq24 Hkv6 108, 103, Hq32 Hkv8 120, 120.
DEVI bool paged_place(int hkv, int per_head, int* hk, int* in) {
  const int lg = min(__builtin_ctz(hkv), 3), share = 3 - lg, heads = hkv >> lg;
  const int x = blockIdx.x & 7, at = (blockIdx.x >> 3 << share) + (x & ((1 << share) - 1));
  *in = at / heads;
  *hk = (x >> share) * heads + at - *in * heads;
  return *in < per_head;
}

// How a launch of the attention shares its work out.  The rows of a sequence and kv
// head are r = i G + g: token i, q head g of the group.
struct PagedPlan {
  float scale;
  int keys, splits;            // of sequences with up to `few` rows: keys of a share, shares
  int keys_many, splits_many;  // of the others
  int few;
  int groups;                  // row tiles of a sequence in the few rows' grid
  int tiles;                   // row tiles of all sequences with more, at most
  int stride;                  // rows of partials kept for each (sequence, kv head); 0: for all
                               // heads of all tokens
};
// Partials; m in the log2 domain, -inf: no key.  Sequences of one share write their output
// instead.  Sequences of few rows: share i of row r at [i][b][kv head][r] (stride > 0) or
// at [i][token][head]; of many rows, at [i][token][head] of arrays of their own.
struct PagedParts {
  float *m, *l, *o;
  float *m_many, *l_many, *o_many;
};
DEVI long few_row(const Paged& a, const PagedPlan& pl, int split, int b, int hk, int r, long row) {
  return pl.stride ? (((long)split * a.batch + b) * a.hkv + hk) * pl.stride + r
                   : (long)split * a.tokens * a.hq + row;
}
// (the last share of the grid takes all that is left)
DEVI int paged_shares(const Seq& s, int keys, int most) {
  return min(max(1, (s.keys(s.n - 1) + keys - 1) / keys), most);
}

// Values in V that are not finite and that some query must not see: 0 times such a
// value would be NaN, so their tile is not multiplied but added key by key to the rows
// that see it.  acc, lane: a wavefront's 32 rows as O^T accumulators; vt: 32 keys of a
// tile in the SWZ_DUAL order; pb: their P; lim: the lane's keys, relative to vt's first.
template <int D>
DEVI void add_keys(f32x16* acc, const char* vt, const uint32_t* pb, int lim) {
  typedef uint32_t u32x8 __attribute__((ext_vector_type(8)));
  const int g = lane_now() >> 5;
  const u32x8 p8 = {pb[0], pb[1], pb[2], pb[3], pb[4], pb[5], pb[6], pb[7]};
  // (looped: it hardly ever runs, and code in the way of what does costs its fetches)
#pragma unroll 1
  for (int r = 0; r < 16; ++r) {
    const uint32_t two = p8[r >> 1];
    const float mine = r & 1 ? bf16hi(two) : bf16lo(two), other = other_half(mine);
#pragma unroll 1
    for (int gg = 0; gg < 2; ++gg) {
      const int key = 8 * (r >> 2) + 4 * gg + (r & 3);
      const float p = gg == g ? mine : other;
      if (key >= lim) continue;
#pragma unroll
      for (int t = 0; t < D / 32; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const u32x2 w = *reinterpret_cast<const u32x2*>(
              vt + swz<SWZ_DUAL, D>(key * (D / 8) + 4 * t + j) * 16 + 8 * g);
          acc[t][4 * j] += p * bf16lo(w[0]);
          acc[t][4 * j + 1] += p * bf16hi(w[0]);
          acc[t][4 * j + 2] += p * bf16lo(w[1]);
          acc[t][4 * j + 3] += p * bf16hi(w[1]);
        }
    }
  }
}
// whether either bf16 of w is not finite
DEVI uint32_t bf16_bad(uint32_t w) {
  return (w & 0x7f800000u) == 0x7f800000u || (w & 0x7f80u) == 0x7f80u;
}
