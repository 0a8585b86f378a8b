// A row of logits in chunks: where a thread's vectors lie (host and device).
#pragma once

constexpr int kTok = 8;         // tokens of a thread's vector
constexpr int kChunk = 8192;    // columns per chunk
constexpr int kMaxChunks = 64;  // a lane each

// The column of the vector that is loaded for columns c .. c + 7 of a row of cols >= 2 kTok:
// c itself where all of them lie in the row, else (whatever it holds is not used) the row's
// first that is as aligned.  A chunk starts at an aligned address, at or before a column of
// the row, so c is a multiple of kTok from one.
constexpr int vector_col(int c, int cols) {
  return c >= 0 && c + kTok <= cols ? c : c & (kTok - 1);
}
