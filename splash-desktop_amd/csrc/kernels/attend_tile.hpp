// Attention of many rows a key head (tiles of 128 rows times query heads): chunks of prompts, bound by the matrix units
// and by the softmax between the two products.
//
// Four waves of 32 rows share tiles of 64 keys in LDS, two tiles deep: while one is multiplied the next arrives. Both
// products run transposed on 32x32x16 MFMAs: S^T = K Q^T leaves 16 of each 32 keys of one row in a lane (lane (h, r), l =
// 32 h + r, holds keys 8 j + 4 h + i of row r), so a row's maximum and sum are the lane's own but for one exchange with
// the lane 32 away, and the eight weights of 16 keys that the second product O^T = V^T P^T wants of a lane are eight that
// it already holds: the contraction takes its keys in that order, 4 h .. + 3 and 8 + 4 h .. + 3 of 16. V^T in that order
// comes from ds_read_b64_tr_b16, which reads four keys' rows and gives each lane one value of them.
//
// LDS holds both tiles as bf16, a key a row, its 16-byte chunks exchanged by the row (chunk c of row k at c ^ swap(k)) so
// that 16 rows of one chunk (K's reads) and four rows of four chunks (V's) fall on all 64 banks. bf16 pages are copied
// straight into LDS (the exchange is in the addresses that the lanes read from); codes pass through registers and become
// bf16 once for all four waves, exactly. Scales multiply the scores, and the weights before they are rounded.
//
// The weights enter the second product as one bf16 each, half a step of which is as much as the output's own rounding: 0.0022
// to 0.0024 from 64 bits, where two (attend_rows.hip) give 0.0017. Two make half as many products again, which nothing hides here: a chunk at 16384
// keys takes 708 us for 518 (int8 794 for 648), prompts of 500 to 900 keys 7% more, 8 rows of heads of 256 6%.
//
// What it reaches: 2048 bf16 rows of 32 heads of 128 at 16384 keys of 8 in 520 us, 0.99 PFLOP/s where a large matrix product
// of the library reaches 1.34: the matrix units are busy 53% of the cycles and the VALU (mostly the exponentials' 32 a lane
// and tile) 48%, at clocks that the power limit holds near 1.75 GHz. The same with 8-bit pages takes 620 to 660 us (the
// scales' and codes' VALU). Narrow heads have half the products for the same exponentials, 380 VALU instructions a wave and
// tile, and keep neither pipe busy: 24 GFLOP of int8 prompts take 81 us, of whose cycles the VALU issues 44% and the matrix
// units work 14%; the rest goes to the barriers and to the start of units of 17 tiles, a chain of loads that nothing covers.
//
// 4-bit pages: a lane's eight codes and the byte of their group become eight bf16 on the way to LDS, scales and all, so no
// scale is left for scores or weights: the chunk at 16384 keys in 3% more than a bf16 one, heads of 256 in 47% more (their codes
// wait in registers that are full; VALU 45% of the cycles, matrix units 42%, heads of 128).
//
// Scored calls are their own instances, so that plain ones compile as if there were none. A cap that is all there is has one
// more (CappedArgs): where a tile's scores are below 0.4 of the cap, cap tanh(t / cap) is an odd polynomial of the seventh
// degree beside the second product, and no exponential or quotient. 2048 rows at 16384 keys of 8, in one run: 16 heads of 256
// with a cap of 50 so 779 us, with the exponential form (a cap of 10) 965, with slopes 836, with neither 693; 32 heads of 128 638,
// 814, 645 and 545 (slopes over int8 keys 728); 32 of 64 452 with the cap and 346 without. (Between cards and runs 5%.)
//
// The registers are full: bf16 heads of 256 spill 13 of them (40 bytes a lane), int8 ones of 128 and 256 4 and 12 (12 and 0
// bytes: accumulation registers hold the others), e4m3 ones 13 and 20 (40 and 24), 4-bit ones of 256 38 (140). Scored ones of
// 256 spill 21 to 50 (72 to 168 bytes) and of bf16 64 4 (12), capped ones of 256 24 to 48 (48 to 180) and of e4m3 128 13 (40).
// No others any.
//
// Keys past the sequence's end and holes read as zeros (buffer resources end there). Only tiles that some row does not
// see whole compare positions.
#pragma once
#include "attend.hpp"
#include "device.hpp"

#include <utility>

namespace sq::kern {
namespace {

constexpr int kWaves = 4, kThreads = 64 * kWaves, kRows = 32 * kWaves;

typedef __attribute__((__vector_size__(16 * sizeof(float)))) float f32x16;

__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                 0);
}
// op over the two lanes that hold a row's keys.
__device__ __forceinline__ float other_max(float v) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float other_sum(float v) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}
// A vector a lane from a buffer straight into LDS: lane l's lands at lds + 16 l.
__device__ __forceinline__ void copy_to_lds(__amdgpu_buffer_rsrc_t from, uint8_t *lds, uint32_t at) {
  const auto to = (__attribute__((address_space(3))) void *)lds;
  __builtin_amdgcn_raw_ptr_buffer_load_lds(from, to, 16, at, 0, 0, 0);
}
// Four keys' values, transposed (lane i of 16 gives the address of key i / 4's values 4 (i % 4) .. + 3 and gets value i
// of the four keys).
__device__ __forceinline__ u32x2 read_transposed(const uint8_t *lds) {
  typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4 *)lds));
}
// Every wave's stores to LDS have landed, and (unless codes are on their way to registers) its copies into it.
template <bool CODES>
__device__ __forceinline__ void tile_barrier() {
  __builtin_amdgcn_s_waitcnt(CODES ? 0xC07F : 0);   // lgkmcnt(0), and vmcnt(0)
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// f of 0 .. N - 1, each a constant.
template <int N, typename F, int... I>
__device__ __forceinline__ void static_for(F &&f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void static_for(F &&f) {
  static_for<N>(f, std::make_integer_sequence<int, N>{});
}

// A head row in LDS: DIM bf16 values, CHUNKS 16-byte chunks. Where chunk c of key k lies.
template <int DIM>
struct Tile {
  static constexpr int kRowBytes = 2 * DIM, kChunks = DIM / 8, kBytes = kKeyTile * kRowBytes;
  // 128-byte rows (DIM 64) lie two to a round of the banks, so the pair's number takes the row's place.
  static __device__ __forceinline__ uint32_t key_swap(uint32_t k) { return DIM == 64 ? (k >> 1) & 7u : k & 15u; }
  static __device__ __forceinline__ uint32_t value_swap(uint32_t k) {
    return DIM == 64 ? 4u * ((k >> 1) & 1u) : 4u * (k & 3u);
  }
};

template <uint32_t FMT, int DIM, typename A>
__global__ __launch_bounds__(kThreads, attend_tile_resident(DIM, FMT)) void attend_tile_kernel(A a) {
  constexpr bool kScored = kScoredCall<A>, kCapped = std::is_same_v<A, CappedArgs>;
  // The score of a hidden key where a cap's polynomial passes over it: no weight, and no infinity among its products.
  constexpr float kHidden = -1e15f;
  using T = Tile<DIM>;
  constexpr bool kFour = FMT == SQ_KV_E2M1;
  constexpr bool kCodes = FMT != SQ_KV_BF16;   // they pass through registers
  constexpr bool kScaled = kCodes && !kFour;   // and have a scale a token, which the tile keeps
  constexpr int kSteps = DIM / 16, kBlocks = DIM / 32, kBits = kFour ? 4 : kCodes ? 8 : 16;
  constexpr int kBlockFloats = 32 * (DIM + 2);   // of a part in the workspace
  // A wave fetches 16 keys of the tile, kLoads vectors a lane of K and of V (of 16 bytes; of 8, heads of 64 in 4 bits).
  constexpr int kVector = DIM * kBits < 512 ? 8 : 16, kLoads = 2 * DIM * kBits / 64 / kVector;
  constexpr int kRowLanes = DIM * kBits / 8 / kVector, kLoadRows = 64 / kRowLanes;
  constexpr uint32_t kGroups = DIM / 32;   // scale bytes of a head row in 4 bits
  __shared__ __attribute__((aligned(1024))) uint8_t tiles[2][2][T::kBytes];   // [tile % 2][K, V]
  __shared__ f32x4 scales[kScaled ? 4 : 1][2][kKeyTile / 4];   // [tile % 4][K, V]
  // [tile % 4][wave]: whether its 16 keys' values hold a NaN code (4 bits: a scale byte above 252)
  __shared__ u32x4 nans[FMT == SQ_KV_E4M3 || kFour ? 4 : 1];
  __shared__ LineShared<kThreads, A> shared;
  const uint32_t lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
  const uint32_t wave = uniform(threadIdx.x >> 6);
  const Cut cut{kRows / (int)a.group, 4 * kKeyTile, kUnitSlack + 192, attend_tile_resident(DIM, FMT), 1152, DIM <= 128 ? 0 : 16};
  const float by_group = 1.0f / (float)a.group;
  const uint32_t dim = a.kv.head_dim, row_bytes = kFour ? dim / 2 : dim * (kBits / 8);
  Part<A> next;
  constexpr bool kWhole = kScored || kFour;   // (the others keep the shares, and so the bits, that they have)
  Work<kThreads, A, kWhole> work = make_work<kThreads, kWhole>(a, cut, shared, next);
  UnitNote began{};

  // Where this lane's vectors lie in 16 keys of a page, and (codes) in the LDS tile.
  uint32_t key_from[kLoads], value_from[kLoads], code_to[kLoads], group_from[kFour ? kLoads : 1];
#pragma unroll
  for (int j = 0; j < kLoads; ++j) {
    const uint32_t k = kLoadRows * j + lane / kRowLanes, c = lane % kRowLanes;
    if constexpr (kFour) {
      // A vector of 32 codes is a group, and four chunks of LDS, 4 c and the next (one of 16 half a group, and two of them).
      key_from[j] = value_from[j] = kVector * c < row_bytes ? k * row_bytes + kVector * c : kNowhere;
      group_from[j] = kVector * c < row_bytes ? k * kGroups + kVector * c / 16 : kNowhere;
      code_to[j] = (16 * wave + k) * T::kRowBytes;
    } else if constexpr (kCodes) {
      // A vector of 16 codes is two chunks of LDS, 2 c and 2 c + 1.
      key_from[j] = value_from[j] = 16 * c < dim ? k * row_bytes + 16 * c : kNowhere;
      code_to[j] = (16 * wave + k) * T::kRowBytes;
    } else {
      // LDS takes the lanes' vectors in lane order, so the lane reads the chunk that its place holds.
      const uint32_t kc = c ^ T::key_swap(k), vc = c ^ T::value_swap(k);
      key_from[j] = 8 * kc < dim ? k * row_bytes + 16 * kc : kNowhere;
      value_from[j] = 8 * vc < dim ? k * row_bytes + 16 * vc : kNowhere;
      code_to[j] = 0;
    }
  }
  // The K operand's row (key r of a block of 32) and the V operand's (keys 4 h + i / 4 of 16, i = lane % 16), chunk 0.
  const uint32_t key_at = r * T::kRowBytes + 16 * (h ^ T::key_swap(r));
  const uint32_t vi = lane & 15, vk = 4 * h + vi / 4;
  const uint32_t value_at = vk * T::kRowBytes + 8 * (vi % 2) + 16 * ((2 * (lane / 16 % 2) + vi % 4 / 2) ^ T::value_swap(vk));

  while (work.next(a, cut, shared, next)) {
    const Part<A> part = settled(a, cut, next);
    const Units<A> &u = part.units;
    const int row0 = cut.fit * part.m, rows = min(cut.fit, u.rows - row0), live = rows * (int)a.group;
    int unit_end = u.causal ? min(u.keys, u.base + row0 + rows) : u.keys;   // keys that any row sees
    if constexpr (kScored) unit_end = max(unit_end, u.bounds.prefix);
    const int tile0 = u.first_tile(part.m);
    const int k_begin = kKeyTile * (tile0 + part.t0), k_end = min(unit_end, kKeyTile * (tile0 + part.t1));
    int clear_begin = u.window ? u.base + row0 + rows - u.window : 0;
    int clear_end = u.causal ? u.base + row0 + 1 : u.keys;
    if constexpr (kScored) {
      clear_begin = max(clear_begin, u.bounds.begin);
      if (u.base + row0 >= 0) clear_end = max(clear_end, u.bounds.prefix);
    }

    // This lane's row.
    const int p = 32 * (int)wave + (int)r, pi = row_of(p, by_group), pg = p - pi * (int)a.group;
    const bool on = p < live;
    const int at = u.base + row0 + pi;
    int low = u.window ? at - u.window + 1 : 0;
    int high = u.causal ? min(at + 1, u.keys) : u.keys;
    [[maybe_unused]] float slope = 0.0f;   // scored: of the row's head, in powers of two
    if constexpr (kScored) {
      low = max(low, u.bounds.begin);
      if (at >= 0) high = max(high, u.bounds.prefix);
      if (on && a.slopes) slope = a.slopes[part.head * a.group + pg] * 1.44269504089f;
    }
    [[maybe_unused]] float cap_scale = 0.0f;   // of a score as the product leaves it, to its share of the cap
    if constexpr (kCapped) cap_scale = a.scale * a.cap_over;
    const float unit = kScored ? 1.0f : a.scale;   // what scores are still to be multiplied by once they are settled
    const bool busy = 32 * (int)wave < live;   // waves past the unit's rows only fetch
    // The page table's entries of the tile at k, lanes 0..3 those of its four 16 keys (~0u past the part's keys); and what
    // they say: the page of this wave's 16 keys (~0u for none), and which of the four have none.
    struct Pages {
      uint32_t own, holes;
    };
    const auto entries_at = [&](int k) __attribute__((always_inline)) {
      const int from = k + 16 * (int)min(lane, 3u);
      return from < k_end ? a.kv.page_table[(size_t)part.sequence * a.kv.pages_per_sequence +
                                            ((uint32_t)from >> a.kv.page_shift)]
                          : ~0u;
    };
    const auto pages_of = [&](uint32_t entries) __attribute__((always_inline)) {
      const uint32_t own = from_lane(entries, wave);
      return Pages{own < a.kv.pages ? own : ~0u, (uint32_t)__ballot(entries >= a.kv.pages) & 15u};
    };
    const int tiles_n = max(part.t1 - part.t0, 0);
    const auto at_tile = [&](int i) __attribute__((always_inline)) { return k_begin + kKeyTile * i; };
    uint32_t entries[3];   // on their way before the queries, which nothing wants before the first keys
#pragma unroll
    for (int i = 0; i < 3; ++i) entries[i] = entries_at(at_tile(i));
    u32x4 q[kSteps];
    {
      const uint16_t *row = a.query + (size_t)(part.first_row + row0 + (on ? pi : 0)) * a.query_stride +
                            (part.head * a.group + (on ? pg : 0)) * dim;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const uint32_t d = 16 * s + 8 * h;
        q[s] = on && d < dim ? (*(const u32x4 *)(row + d) & a.keep) ^ a.flip : u32x4{0u, 0u, 0u, 0u};
      }
    }
    float m = -INFINITY, l = 0.0f;
    f32x16 o[kBlocks];
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[b][i] = 0.0f;

    // Copies of the tile at k into stage `to`, K or V: bf16 straight into LDS, codes into registers until place() converts
    // them.
    u32x4 code_k[kCodes ? kLoads : 1], code_v[kCodes ? kLoads : 1];
    float code_scale[2] = {0.0f, 0.0f};
    uint32_t group_k[kFour ? kLoads : 1], group_v[kFour ? kLoads : 1];   // the vectors' scale bytes
    const auto fetch = [&](int k, uint32_t page, int to, auto of_values) __attribute__((always_inline)) {
      constexpr bool kValues = decltype(of_values)::value;
      const int from = k + 16 * (int)wave, n = page == ~0u ? 0 : min(16, k_end - from);
      const size_t base = ((((size_t)(page == ~0u ? 0 : page) * a.kv.kv_heads + part.head) << a.kv.page_shift) +
                           ((uint32_t)from & ((1u << a.kv.page_shift) - 1)));
      const __amdgpu_buffer_rsrc_t rows =
          buffer_rsrc((kValues ? a.kv.values : a.kv.keys) + base * row_bytes, (uint32_t)n * row_bytes);
      if constexpr (kFour) {
        const __amdgpu_buffer_rsrc_t by = buffer_rsrc(
            (const uint8_t *)(kValues ? a.kv.value_scales : a.kv.key_scales) + base * kGroups, (uint32_t)n * kGroups);
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
          u32x4 &v = (kValues ? code_v : code_k)[j];
          if constexpr (kVector == 8) {
            const u32x2 two = buffer_b64<0>(rows, key_from[j], 0);
            v = u32x4{two[0], two[1], 0u, 0u};
          } else {
            v = buffer_b128<0>(rows, key_from[j], 0);
          }
          (kValues ? group_v : group_k)[j] = buffer_b8<0>(by, group_from[j], 0);
        }
      } else if constexpr (kCodes) {
#pragma unroll
        for (int j = 0; j < kLoads; ++j)
          (kValues ? code_v : code_k)[j] = buffer_b128<0>(rows, (kValues ? value_from : key_from)[j], 0);
        const __amdgpu_buffer_rsrc_t by =
            buffer_rsrc((kValues ? a.kv.value_scales : a.kv.key_scales) + base, (uint32_t)n * 4);
        code_scale[kValues] = __uint_as_float(buffer_b32<0>(by, 4 * (lane & 15), 0));
      } else {
        uint8_t *lds = &tiles[to][kValues][16 * wave * T::kRowBytes];
#pragma unroll
        for (int j = 0; j < kLoads; ++j) copy_to_lds(rows, lds + 1024 * j, (kValues ? value_from : key_from)[j]);
      }
    };
    // Whether rows of the unit see other keys than others among the 64 from k on (not for their holes or the sequence's end).
    const auto differs = [&](int k) __attribute__((always_inline)) {
      return k < clear_begin || k + kKeyTile > clear_end;
    };
    const auto place = [&](int tile, auto of_values) __attribute__((always_inline)) {
      constexpr bool kValues = decltype(of_values)::value;
      if constexpr (FMT == SQ_KV_E4M3 && kValues) {
        // Looked at here, where the codes are at hand, for 2 to 4% of a chunk; a pass over the tile in LDS and its barrier took
        // 1 to 8 (most where a window begins in the middle of every unit).
        if (differs(at_tile(tile))) {
          uint32_t any = 0;
#pragma unroll
          for (int j = 0; j < kLoads; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) any |= nan_codes(code_v[j][i]);
          const bool some = __any(any != 0);
          if (lane == 0) ((uint32_t *)&nans[tile % 4])[wave] = some;
        }
      }
      if constexpr (kFour) {
        if constexpr (kValues)
          if (differs(at_tile(tile))) {
            bool any = false;
#pragma unroll
            for (int j = 0; j < kLoads; ++j) any |= group_v[j] > 252u;
            const bool some = __any(any);
            if (lane == 0) ((uint32_t *)&nans[tile % 4])[wave] = some;
          }
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
          const uint32_t k = kLoadRows * j + lane / kRowLanes, c = kVector / 4 * (lane % kRowLanes);
          const u32x4 w = (kValues ? code_v : code_k)[j];
          const uint32_t by = (kValues ? group_v : group_k)[j] << 23;
#pragma unroll
          for (int i = 0; i < kVector / 4; ++i)
            *(u32x4 *)&tiles[tile % 2][kValues][code_to[j] + 16 * ((c + i) ^ (kValues ? T::value_swap(k) : T::key_swap(k)))] =
                u32x4{fp4_pair(w[i], by, 0), fp4_pair(w[i], by, 1), fp4_pair(w[i], by, 2), fp4_pair(w[i], by, 3)};
        }
      } else if constexpr (kCodes) {
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
          const uint32_t k = kLoadRows * j + lane / kRowLanes, c = 2 * (lane % kRowLanes);
          const u32x4 w = (kValues ? code_v : code_k)[j];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const u32x2 lo = code_pairs4<FMT>(w[2 * i]), hi = code_pairs4<FMT>(w[2 * i + 1]);
            *(u32x4 *)&tiles[tile % 2][kValues][code_to[j] + 16 * ((c + i) ^ (kValues ? T::value_swap(k) : T::key_swap(k)))] =
                u32x4{lo[0], lo[1], hi[0], hi[1]};
          }
        }
        if (lane < 16) ((float *)&scales[tile % 4][kValues][4 * wave])[lane] = code_scale[kValues];
      }
    };
    constexpr std::false_type kOfKeys{};
    constexpr std::true_type kOfValues{};

    f32x16 s[2];   // the scores of the tile at hand
    constexpr f32x16 kZero{};
    const auto key_operand = [&](int tile, int c, int b) __attribute__((always_inline)) {
      return *(const u32x4 *)&tiles[tile % 2][0][32 * b * T::kRowBytes + (key_at ^ (32 * c))];
    };
    const auto value_operand = [&](int tile, int t, int b) __attribute__((always_inline)) {
      const uint8_t *from = &tiles[tile % 2][1][16 * t * T::kRowBytes + (value_at ^ (64 * b))];
      const u32x2 v0 = read_transposed(from), v1 = read_transposed(from + 8 * T::kRowBytes);
      return u32x4{v0[0], v0[1], v1[0], v1[1]};
    };

    // The running maximum above a tile's largest score but kRaise.
    const auto raise = [&](float top) __attribute__((always_inline)) {
      if (__any(top > m + kRaise)) {
        const float next = fmaxf(m, other_max(top));
        const float shrink = exp2_fast(m - finite_max(next));
        m = next;
        l *= shrink;
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) o[b] *= shrink;
      }
    };
    // A tile's scores to their final form but for the exponential: scaled (codes), hidden where the row does not see the
    // key, the running maximum above all of them but kRaise. Returns whether a cap is left for finish() to do (a cap keeps the
    // order of scores, so the maximum is the largest one's).
    const auto settle = [&](int tile, int k, uint32_t holes, bool clear) __attribute__((always_inline)) {
      if constexpr (kScaled) {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          f32x4 by[4];   // together, so that one wait serves the four
#pragma unroll
          for (int j = 0; j < 4; ++j) by[j] = scales[tile % 4][0][8 * b + 2 * j + h];
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int i = 0; i < 16; ++i) s[b][i] *= by[i / 4][i % 4];
        }
      }
      float top = -INFINITY;
      [[maybe_unused]] bool small = false;   // all of them, of a call with a cap: the cap is finish()'s
      if constexpr (kCapped) {
        if (clear) {
          float bottom = INFINITY;
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              top = fmaxf(top, s[b][i]);
              bottom = fminf(bottom, s[b][i]);
            }
          small = !__any(fmaxf(top, -bottom) * cap_scale > kTanhSmall);
          top = small ? capped(a, top * a.scale) : -INFINITY;
        }
      }
      if (!small) {
        if constexpr (kScored) {
          const float ahead = (float)(k + 4 * (int)h - at);   // of the lane's first key
          if (kCapped || a.cap != 0.0f) {
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
              for (int i = 0; i < 16; ++i) s[b][i] = capped(a, s[b][i] * a.scale);
          } else {
            s[0] *= a.scale;
            s[1] *= a.scale;
          }
          if (!kCapped && a.slopes) {
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
              for (int i = 0; i < 16; ++i)
                s[b][i] = fmaf(-slope, fabsf(ahead + (float)(32 * b + 8 * (i / 4) + i % 4)), s[b][i]);
          }
        }
        if (!clear) {
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int key = k + 32 * b + 8 * (i / 4) + 4 * (int)h + i % 4;
              const bool sees = key >= low && key < high && !(holes >> (2 * b + i / 8) & 1);
              s[b][i] = sees ? s[b][i] : kCapped ? kHidden : -INFINITY;
            }
        }
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int i = 0; i < 16; ++i) top = fmaxf(top, s[b][i]);
        if constexpr (kCapped) top = top == kHidden ? -INFINITY : top;
      }
      if constexpr (!kScored) top *= a.scale;   // not negative (the queries carry its sign), and not zero
      raise(top);
      return small;
    };

    // Infinities and NaNs among a tile's values must not reach rows that do not see them through 0 * inf: the rows that do
    // see them take their products apart, and they leave the tile. Only tiles that are not clear can have such rows.
    const auto set_apart = [&](int tile, int k, uint32_t holes) __attribute__((always_inline)) {
      if constexpr (kFour) {
        if (!differs(k)) return;
        const u32x4 any = nans[tile % 4];
        if (!uniform(any[0] | any[1] | any[2] | any[3])) return;
      }
      if constexpr (kScaled) {
        // The scale of a head row that was not finite is a NaN, and all of it is.
        float *by = (float *)scales[tile % 4][1];
        const bool bad = !(fabsf(by[lane]) < INFINITY);
        uint64_t rows_bad = __ballot(bad);
        if (rows_bad) {
          while (busy && rows_bad) {
            const int key = __ffsll((unsigned long long)rows_bad) - 1, j = k + key;
            rows_bad &= rows_bad - 1;
            if (on && j >= low && j < high && !(holes >> (key / 16) & 1)) {
#pragma unroll
              for (int b = 0; b < kBlocks; ++b) o[b] += __uint_as_float(0x7FC00000u);
            }
          }
          __syncthreads();
          if (bad && wave == 0) by[lane] = 0.0f;
          __syncthreads();
        }
        // int8 codes are finite, and so are e4m3's that a write has made; pages may hold its NaN that have not been written
        // yet, or by another.
        if constexpr (FMT == SQ_KV_INT8) return;
        if (!differs(k)) return;
        const u32x4 any = nans[tile % 4];
        if (!uniform(any[0] | any[1] | any[2] | any[3])) return;
      }
      constexpr int kMine = T::kBytes / 16 / kThreads;
      uint8_t *vt = tiles[tile % 2][1];
      if constexpr (!kCodes) {
        uint32_t any = 0;
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
          const u32x4 v = *(const u32x4 *)&vt[16 * (threadIdx.x + kThreads * i)];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            any |= (uint32_t)((v[e] & 0x7F80u) == 0x7F80u) | (uint32_t)((v[e] & 0x7F800000u) == 0x7F800000u);
        }
        if (!__syncthreads_or((int)any)) return;
      }
      if constexpr (kScaled) {
        // All of them are NaNs, whatever the weights. Products of kHuge in their places and in those of keys seen, which
        // overflow, once to infinity and once below it, leave NaNs, and add zeros to all other accumulators.
        constexpr uint32_t kHuge = 0x7F00u;   // bf16's 2^127
        if (busy) {
#pragma unroll 1
          for (int t = 0; t < 4; ++t) {
            u32x4 sees;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int j = k + 16 * t + 8 * (i / 2) + 4 * (int)h + 2 * (i % 2);   // and the next key
              sees[i] = (on && j >= low && j < high ? kHuge : 0u) | (on && j + 1 >= low && j + 1 < high ? kHuge << 16 : 0u);
            }
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
              u32x4 at = value_operand(tile, t, b);
#pragma unroll
              for (int i = 0; i < 4; ++i)
                at[i] = ((at[i] & 0x7F80u) == 0x7F80u ? kHuge : 0u) | ((at[i] & 0x7F800000u) == 0x7F800000u ? kHuge << 16 : 0u);
              o[b] = mfma32(at, sees, o[b]);
              o[b] = mfma32(at ^ 0x80008000u, sees, o[b]);
              __builtin_amdgcn_sched_barrier(0);
            }
          }
        }
      } else if (busy) {
#pragma unroll 1
        for (uint32_t key = 0; key < kKeyTile; ++key) {
          // Key `key` is score 4 (key % 32 / 8) + key % 4 of block key / 32 in the lanes with h = key / 4 % 2.
          const uint32_t i = 4 * (key % 32 / 8) + key % 4;
          const float score = key & 32 ? s[1][i] : s[0][i];
          const float mine = bf16_to_f32(f32_to_bf16(exp2_fast(fmaf(score, unit, -finite_max(m)))));
          const float weight = __shfl(mine, (int)(r + 32 * (key / 4 % 2)));
          const int j = k + (int)key;
          const bool sees = on && j >= low && j < high && !(holes >> (key / 16) & 1);
#pragma unroll
          for (int b = 0; b < kBlocks; ++b)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const uint32_t chunk = (4 * b + c) ^ T::value_swap(key);
              const u32x2 v = *(const u32x2 *)&vt[key * T::kRowBytes + 16 * chunk + 8 * h];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const uint32_t bits = e & 1 ? v[e / 2] >> 16 : v[e / 2] & 0xFFFFu;
                if (sees && (bits & 0x7F80u) == 0x7F80u) o[b][4 * c + e] += weight * bf16_to_f32(bits);
              }
            }
        }
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        u32x4 *v = (u32x4 *)&vt[16 * (threadIdx.x + kThreads * i)];
        u32x4 clean = *v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if ((clean[e] & 0x7F80u) == 0x7F80u) clean[e] &= 0xFFFF0000u;
          if ((clean[e] & 0x7F800000u) == 0x7F800000u) clean[e] &= 0x0000FFFFu;
        }
        *v = clean;
      }
      __syncthreads();
    };

    // The rest of a tile, and the next one's first product: each block of 32 scores gives its registers to the next tile's
    // as it becomes weights. The products go out in slots, scores and values in turn, operands read from LDS kAhead slots
    // before, the second block's exponentials between the first ones' products; a barrier to the compiler's scheduling
    // keeps them so (left to itself it gathers the products, each behind a wait for its operand).
    // A call's cap is a polynomial here where the tile's scores are small, four instructions more a score, which the products
    // partly hide. Scores that are settled go through the polynomial 1, as the registers hold no second form of this code. The
    // share of the cap goes into the coefficients, or, one more instruction, is taken first: bf16 heads of 256 spill less so, 6%
    // less time (int8 ones would take 1% more, heads of 128 2%).
    const auto finish = [&](int tile, [[maybe_unused]] bool to_cap) __attribute__((always_inline)) {
      constexpr bool kShareFirst = FMT == SQ_KV_BF16 && DIM == 256;
      [[maybe_unused]] float by_y = 1.0f, p0 = 1.0f, p1 = 0.0f, p2 = 0.0f, p3 = 0.0f;
      if constexpr (kCapped) {
        if (to_cap) {
          const float by = kShareFirst ? a.cap : a.scale, two = kShareFirst ? 1.0f : cap_scale * cap_scale;
          if constexpr (kShareFirst) by_y = cap_scale;
          p0 = kTanh0 * by;
          p1 = kTanh1 * by * two;
          p2 = kTanh2 * by * (two * two);
          p3 = kTanh3 * by * (two * two * two);
        }
      }
      constexpr int kSlots = 4 * kSteps, kAhead = 4;
      // Slot i's product: a score (step of a block of 32 keys), or values (16 keys into a block of 32 values).
      struct Slot {
        bool score;
        int major, minor;
      };
      constexpr auto slot = [](int i) {
        const int half = i / (2 * kSteps), j = i % (2 * kSteps) / 2;
        return i % 2 == 0 ? Slot{true, j, half} : Slot{false, 2 * half + j / kBlocks, j % kBlocks};
      };
      u32x4 w[4];   // the weights of 16 keys each
      u32x4 operand[kSlots];
      const float from = -finite_max(m);
      float sum[2] = {0.0f, 0.0f};
      f32x4 by{}, by_next{};   // four weights' scales of values, read four weights before
      if constexpr (kScaled) by_next = scales[tile % 4][1][h];
      float even = 0.0f;
      const auto read = [&](auto index) __attribute__((always_inline)) {
        constexpr Slot at = slot(decltype(index)::value);
        operand[index] = at.score ? key_operand(tile + 1, at.major, at.minor) : value_operand(tile, at.major, at.minor);
      };
      // The weight of score i of block b.
      const auto weigh = [&](int b, int i) __attribute__((always_inline)) {
        if constexpr (kScaled)
          if (i % 4 == 0) {
            by = by_next;
            const int group = 4 * b + i / 4 + 1;
            if (group < 8) by_next = scales[tile % 4][1][2 * group + h];
          }
        float v;
        if constexpr (kCapped) {
          const float y = kShareFirst ? s[b][i] * by_y : s[b][i], z = y * y;
          v = exp2_fast(fmaf(y, fmaf(z, fmaf(z, fmaf(z, p3, p2), p1), p0), from));
        } else {
          v = exp2_fast(fmaf(s[b][i], unit, from));
        }
        sum[i % 2] += v;
        if constexpr (kScaled) v *= by[i % 4];
        if (i % 2) w[2 * b + i / 8][i % 8 / 2] = bf16_pair(even, v);
        else even = v;
      };
      static_for<kAhead>([&](auto i) __attribute__((always_inline)) { read(i); });
#pragma unroll
      for (int i = 0; i < 16; ++i) weigh(0, i);
      static_for<kSlots>([&](auto index) __attribute__((always_inline)) {
        constexpr int i = decltype(index)::value;
        if constexpr (i + kAhead < kSlots) read(std::integral_constant<int, i + kAhead>{});
        constexpr Slot at = slot(i);
        if constexpr (at.score) s[at.minor] = mfma32(operand[i], q[at.major], at.major ? s[at.minor] : kZero);
        else o[at.minor] = mfma32(operand[i], w[at.major], o[at.minor]);
        if constexpr (i < 2 * kSteps)
          for (int e = 8 * i / kSteps; e < 8 * (i + 1) / kSteps; ++e) weigh(1, e);
        __builtin_amdgcn_sched_barrier(0);
      });
      l += sum[0] + sum[1];
    };

    // K runs a tile ahead of V: while a tile is finished and the next one's scores are made, the copies of K two tiles on
    // and V one tile on are under way, into the stages that the last tile has left. Codes wait in registers one tile
    // more, and the page table's entries are fetched a tile before the copies that want them.
    __syncthreads();   // the last part's tiles have been read
    Pages pages[4];    // of the tiles from the one at hand on
#pragma unroll
    for (int i = 0; i < 3; ++i) pages[i] = pages_of(entries[i]);
    uint32_t later = entries_at(at_tile(3));
    fetch(at_tile(0), pages[0].own, 0, kOfKeys);
    fetch(at_tile(0), pages[0].own, 0, kOfValues);
    place(0, kOfKeys);
    place(0, kOfValues);
    fetch(at_tile(1), pages[1].own, 1, kOfKeys);
    if constexpr (kCodes) {
      place(1, kOfKeys);
      fetch(at_tile(2), pages[2].own, 0, kOfKeys);
      fetch(at_tile(1), pages[1].own, 1, kOfValues);
    }
    tile_barrier<kCodes>();
    if (busy) {
#pragma unroll
      for (int c = 0; c < kSteps; ++c)
#pragma unroll
        for (int b = 0; b < 2; ++b) s[b] = mfma32(key_operand(0, c, b), q[c], c ? s[b] : kZero);
    }
    tile_barrier<kCodes>();   // K's first stage has been read
    for (int tile = 0; tile < tiles_n; ++tile) {
      const int k = at_tile(tile);
      // Of two workgroups' waves on a SIMD the older goes first, and finishes long before the other: they take turns
      // instead (2048 rows at 16384 keys: 372 and 468 us without the turns, 408 and 417 with them).
      if (tile & 1) __builtin_amdgcn_s_setprio(1);
      else __builtin_amdgcn_s_setprio(0);
      pages[3] = pages_of(later);
      later = entries_at(at_tile(tile + 4));
      if constexpr (kCodes) {
        if (tile + 1 < tiles_n) {
          place(tile + 2, kOfKeys);
          place(tile + 1, kOfValues);
        }
        if (tile + 2 < tiles_n) {
          fetch(at_tile(tile + 3), pages[3].own, 0, kOfKeys);
          fetch(at_tile(tile + 2), pages[2].own, 0, kOfValues);
        }
      } else {
        if (tile + 2 < tiles_n) fetch(at_tile(tile + 2), pages[2].own, tile % 2, kOfKeys);
        if (tile + 1 < tiles_n) fetch(at_tile(tile + 1), pages[1].own, (tile + 1) % 2, kOfValues);
      }
      const uint32_t holes = pages[0].holes;
      const bool clear = k >= clear_begin && k + kKeyTile <= clear_end && k + kKeyTile <= k_end && !holes;
      bool to_cap = false;
      if (busy) to_cap = settle(tile, k, holes, clear);
      if (!clear) set_apart(tile, k, holes);
      if (busy) finish(tile, to_cap);
      tile_barrier<kCodes>();
#pragma unroll
      for (int i = 0; i < 3; ++i) pages[i] = pages[i + 1];
    }
    l = other_sum(l);

    if (part.parts > 1) {
      if (part.part == 0) began = {part.parts, (uint32_t)live, part.first_row + (uint32_t)row0, part.head};
      if (busy) {
        float *mine = a.partials + part_block(a, part.first_piece, part.part, wave) * kBlockFloats;
        if (on) {
#pragma unroll
          for (int b = 0; b < kBlocks; ++b)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              *(f32x4 *)(mine + ((4 * b + j) * 64 + lane) * 4) =
                  f32x4{o[b][4 * j], o[b][4 * j + 1], o[b][4 * j + 2], o[b][4 * j + 3]};
        }
        if (h == 0) {
          mine[32 * DIM + 2 * lane] = m;
          mine[32 * DIM + 2 * lane + 1] = l;
        }
      }
      continue;
    }
    if (on) {
      const float by = l == 0.0f ? 0.0f : 1.0f / l;
      uint16_t *out = a.output + (size_t)(part.first_row + row0 + pi) * a.output_stride + (part.head * a.group + pg) * dim;
#pragma unroll
      for (int b = 0; b < kBlocks; ++b)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t d = 32 * b + 8 * j + 4 * h;
          if (d < dim)
            *(u32x2 *)(out + d) = u32x2{bf16_pair(o[b][4 * j] * by, o[b][4 * j + 1] * by),
                                        bf16_pair(o[b][4 * j + 2] * by, o[b][4 * j + 3] * by)};
        }
    }
  }
  work.leave(a, began);
}

template <uint32_t FMT, typename A>
hipError_t launch_dim(const A &a, hipStream_t stream) {
  const dim3 grid(a.workgroups), block(kThreads);
  if (a.kv.head_dim <= 64) hipLaunchKernelGGL((attend_tile_kernel<FMT, 64, A>), grid, block, 0, stream, a);
  else if (a.kv.head_dim <= 128) hipLaunchKernelGGL((attend_tile_kernel<FMT, 128, A>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((attend_tile_kernel<FMT, 256, A>), grid, block, 0, stream, a);
  return hipGetLastError();
}
template <typename A>
hipError_t launch_tile(const A &a, hipStream_t stream) {
  if (a.kv.format == SQ_KV_BF16) return launch_dim<SQ_KV_BF16>(a, stream);
  if (a.kv.format == SQ_KV_INT8) return launch_dim<SQ_KV_INT8>(a, stream);
  if (a.kv.format == SQ_KV_E2M1) return launch_dim<SQ_KV_E2M1>(a, stream);
  return launch_dim<SQ_KV_E4M3>(a, stream);
}

}  // namespace
}  // namespace sq::kern
