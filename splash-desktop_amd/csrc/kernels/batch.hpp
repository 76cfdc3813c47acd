// What the cache and attention kernels read of a batch that only the device holds: row starts, lengths, page ids. Every
// value is bounded here, so that nothing outside the views is addressed whatever the buffers hold.
#pragma once
#include "kernels.hpp"

namespace sq::kern {

// A sequence of the batch: its rows [first, first + rows) of the head rows, and its keys with them. keys is at most
// the sequence's pages hold, and rows lie within the batch's.
struct Sequence {
  uint32_t first, rows;
  int keys;
};
__device__ __forceinline__ Sequence sequence_of(const KvArgs &kv, uint32_t s) {
  const uint32_t a = min(kv.row_starts[s], kv.rows), b = min(kv.row_starts[s + 1], kv.rows);
  const uint32_t most = kv.pages_per_sequence << kv.page_shift;   // the host keeps it below 2^31
  return {a, b > a ? b - a : 0u, (int)min(kv.lengths[s], most)};
}

// Where a row of the batch lies: its sequence's index and its position, or no sequence (sequence ~0u) for a row
// outside all of them. A wave counts the row starts up to the row, 64 at a time: one round trip, where a search would
// make one a step.
struct RowPlace {
  uint32_t sequence;
  int position;
};
__device__ __forceinline__ RowPlace place_of(const KvArgs &kv, uint32_t row) {
  uint32_t count = 0;
  for (uint32_t i = threadIdx.x & 63; i - (threadIdx.x & 63) < kv.sequences; i += 64)
    count += (uint32_t)__popcll(__ballot(i < kv.sequences && kv.row_starts[i] <= row));
  if (!count) return {~0u, 0};
  const Sequence q = sequence_of(kv, count - 1);
  if (row - q.first >= q.rows) return {~0u, 0};
  return {count - 1, q.keys - (int)(q.first + q.rows - row)};
}

// The page of token `position` (at least 0, below the sequence's keys), or ~0u for a hole.
__device__ __forceinline__ uint32_t page_of(const KvArgs &kv, uint32_t sequence, int position) {
  const uint32_t page =
      kv.page_table[(size_t)sequence * kv.pages_per_sequence + ((uint32_t)position >> kv.page_shift)];
  return page < kv.pages ? page : ~0u;
}

}  // namespace sq::kern
