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

// Pages of 4 bits: byte `pair` (0..3) of w holds two e2m1 codes, the first in its low half; as two bf16 under a scale whose
// exponent alone counts (the byte b of a group shifted to a float's exponent, b << 23: 2^(b - 127), and NaN for 255).
// Exact: a code has one bit behind its first, and a product past bf16's range is infinite.
__device__ __forceinline__ uint32_t fp4_pair(uint32_t w, uint32_t scale, int pair) {
  const float s = __uint_as_float(scale);
  switch (pair) {
    case 0: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0));
    case 1: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1));
    case 2: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2));
    default: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3));
  }
}
// Group g's scale of a word of them.
__device__ __forceinline__ uint32_t fp4_scale(uint32_t word, uint32_t g) { return (word >> (8 * g) & 0xFFu) << 23; }
// Scales of bytes above 252, under which values are not finite, or may not be.
__device__ __forceinline__ bool fp4_unbounded(uint32_t scale) { return scale > (252u << 23); }

}  // namespace sq::kern
