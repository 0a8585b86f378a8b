// A cache in pages: [n_pages, Hkv, 2^lg rows, D], key j of sequence b in row
// j % 2^lg of page table[b ld + (j >> lg)].  Entries outside [0, n_pages) are
// absent pages: nothing is read from them or written to them, and their keys do
// not count.  The new tokens of all sequences are packed: those of sequence b are
// tokens starts[b] .. starts[b + 1] - 1 (starts null: `each` tokens a sequence),
// token i of them at position past[b] + i (past null: past_all).
#pragma once
#include "common.h"

struct Paged {
  const int *table, *starts, *past;
  int batch, tokens, each, past_all;
  int ld, width, n_pages, lg;  // table: row stride, pages of a sequence
  int hq, hkv;
};

// What a kernel knows of a sequence, bounded whatever the device arrays hold:
// tokens t0 .. t0 + n - 1 lie in the batch, and every count of keys in the table.
struct Seq {
  int t0, n, past, cap;
  // keys that the sequence's first i + 1 new tokens see
  DEVI int keys(int i) const { return min(max(past + i + 1, 0), cap); }
};
DEVI Seq seq_of(const Paged& a, int b) {
  Seq s;
  const int t0 = a.starts ? a.starts[b] : b * a.each;
  const int t1 = a.starts ? a.starts[b + 1] : t0 + a.each;
  s.t0 = min(max(t0, 0), a.tokens);
  s.n = max(min(t1, a.tokens) - s.t0, 0);
  s.cap = a.width << a.lg;
  s.past = min(max(a.past ? a.past[b] : a.past_all, -a.tokens), s.cap);
  return s;
}
// The sequence of token t (wave-uniform): the last one that starts at or before it;
// -1: none.  A wavefront looks at 64 starts at a time.
DEVI int seq_at(const Paged& a, int t) {
  if (!a.starts) return t < a.batch * a.each ? t / a.each : -1;
  const int lane = threadIdx.x & 63;
  int n = 0;
  for (int i = 0; i <= a.batch; i += 64) {
    const bool yes = i + lane <= a.batch && a.starts[min(i + lane, a.batch)] <= t;
    const uint64_t all = __ballot(yes);
    n += __builtin_popcountll(all);
    if (~all) break;
  }
  return n > 0 && n <= a.batch ? n - 1 : -1;
}

// A wavefront's way along a sequence's table: 64 entries in a register.
struct PageWalk {
  const int* row;
  int width, n_pages, first, mine;
  DEVI PageWalk(const Paged& a, int b)
      : row(a.table + (long)b * a.ld), width(a.width), n_pages(a.n_pages), first(-1 << 20), mine(-1) {}
  // the page of table entry i (wave-uniform); -1: absent
  DEVI int at(int i) {
    if ((unsigned)(i - first) >= 64u) {
      first = i;
      const int j = i + (int)(threadIdx.x & 63);
      mine = j < width ? row[j] : -1;
      if ((unsigned)mine >= (unsigned)n_pages) mine = -1;
    }
    return __builtin_amdgcn_readlane(mine, i - first);
  }
};
