// Where the new tokens' rows of a call lie in the paged cache: shared by the kernels that write, read and move them.
#pragma once

#include "tri_common.h"

namespace tri {
namespace {

// The sequence of a row (the same in every lane): the last one whose first row is not behind it; -1 if none has the row.  A wave
// probes 64 of the ascending starts at once: one load for up to 64 sequences, two for up to 4096.
__device__ __forceinline__ int sequence_of_row(const int32_t* row_starts, int B, int row, int lane) {
  int lo = 0, n = B;
  while (true) {
    const int step = ceil_div(n, kWave), i = lane * step;
    const int count = __popcll(__ballot(i < n && row_starts[lo + min(i, n - 1)] <= row));
    if (count == 0) return -1;
    lo += (count - 1) * step;
    n = min(step, n - (count - 1) * step);
    if (n <= 1) break;
  }
  return row < row_starts[lo + 1] ? lo : -1;
}

// The token that row `row` of sequence b is: its rows are the last ones of its tokens.  Negative: the sequence has fewer tokens than rows.
__device__ __forceinline__ int token_of_row(const int32_t* row_starts, const int32_t* seq_lens, int Tmax, int b, int row) {
  const int T = min(max(seq_lens[b], 0), Tmax);
  return row_starts ? T - (row_starts[b + 1] - row) : T - 1;
}

// The physical block of token t >= 0, -1 if it lies outside the pool.
__device__ __forceinline__ int page_of_token(const int32_t* block_table, int pitch, int block_size, int num_blocks, int b, int t) {
  const int page = block_table ? block_table[(int64_t)b * pitch + t / block_size] : b;
  return page >= 0 && page < num_blocks ? page : -1;
}

}  // namespace
}  // namespace tri
