// What both kinds of few-row tiles share (attend_rows.hpp; attend_rows_four.hpp, 4-bit pages).
#pragma once
#include "attend.hpp"
#include "device.hpp"

namespace sq::kern {

constexpr int kStep = 32;      // keys a wave takes a step
// What all weights are multiplied by on their way into the second product, so that the rest of one that bf16 holds exactly
// is 2^-18 of it and not zero. The outputs grow by as much, a 2^-10 of their own rounding. (The rest of a weight below
// 2^-108 leaves bf16's normal range: an infinite value under it may give NaN, as it does in fp32 where e^x has become 0.)
constexpr float kMore = 1 + 0x1p-18f;

// The maximum over the four lanes that hold one row's keys.
__device__ __forceinline__ float row_max(float v) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float row_sum(float v) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Sixteen keys of one page: the first one's place in the cache, and how many there are to read (none in a hole).
struct Keys16 {
  size_t at;
  uint32_t count;
};
// A part's keys, and of them those that every row of the unit sees.
struct KeySpan {
  int begin, end, clear_begin, clear_end;
};

}  // namespace sq::kern
