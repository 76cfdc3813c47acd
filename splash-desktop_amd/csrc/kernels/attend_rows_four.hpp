// The few-row tiles' keys and values of 4 bits. The products, weights and outputs are those of attend_rows.hpp: a wave takes 32
// keys a step, A and B of 16, and no shared memory lies between the cache and the matrix units. A group's scale is a power of
// two, which the conversion to bf16 takes with the code: the operands are the values themselves, exactly, and no scale is left
// for scores or weights. A vector of 16 bytes is a group of one key, so chain c of the first product takes values 128 (c / 4) +
// 32 kq + 8 (c % 4) + e of a lane's vector, and the queries lie in that order.
//
// A step is half the bytes of 8-bit codes and as many instructions, so two things bind it that do not bind them. Its bytes: one
// step ahead is too few in flight, so where registers allow a wave keeps two (a token over 131072 keys of 8 heads of 128, with
// the join: 50 us with one, 41 with two), and every path loads alike, past the end from empty resources: where paths with fewer
// loads meet, or after a store to memory that may be LDS's, the compiler waits for all loads at each step. Its VALU (52% of
// a launch's cycles, the matrix units 17%): 64 conversions and 32 transposes a step stay; scales come by one rotation, and no
// selects are made where all keys are seen.
//
// What it reaches: a token of 40 heads over 131072 keys of 8 heads of 128 (143 MB) in 35 us, 4.1 TB/s, where int8 takes 54; a
// token each of 64 sequences of 200 to 8000 keys (151 MB) in 52, 2.9 TB/s, four of a tile's 16 rows live, and a
// start and a join of the waves for each of some 1000 parts.
// Tiles of 32 rows and heads of 256 keep one step in flight. With the join, one / two steps: eight rows each of those 64 sequences
// 77 / 77 us (int8 95), four rows of 64 heads over 131072 keys 53 / 53; of heads of 64, where two spill 19 registers, 54 / 60;
// heads of 256 (37 spilled), a token over 131072 keys 64 / 78, 4.4 TB/s with one (int8 108), of each of 64 sequences 83 / 103
// (int8 128).
#pragma once
#include "attend_few.hpp"

namespace sq::kern {
namespace {

// Ones in the places of a word's codes whose values are finite under a scale byte above 252: none under 255, magnitudes up to
// 1.5 (codes with no bit of 4) under 254, and up to 3 (codes without bits 4 and 2 together) under 253.
__device__ __forceinline__ uint32_t finite_codes4(uint32_t w, uint32_t by) {
  const uint32_t infinite = (by == 254 ? w : w & w << 1) & 0x44444444u;
  return by == 255 ? 0u : ~((infinite >> 2) * 15);
}

template <int DIM, int MB>
struct Rows4 {
  static constexpr int kRun = DIM / 16, kChains = DIM / 32;
  // Vectors of keys a lane loads of 16 keys (heads of 64: of 8 bytes), words of values a key (heads of 64: half of it is the
  // lane's), and words of scale bytes for four keys.
  static constexpr int kKeyLoads = DIM <= 128 ? 1 : 2, kValueWords = DIM <= 128 ? 1 : 2, kGroupWords = DIM == 64 ? 2 : 4;
  static constexpr uint32_t kGroups = DIM / 32;   // scale bytes of a head row

  struct KeyTile {
    u32x4 w[2][kKeyLoads];
    uint32_t group[2][kKeyLoads];   // the word with each vector's scale byte
  };
  struct ValueTile {
    uint32_t w[2][4][kValueWords];
    uint32_t groups[2][kGroupWords];
  };

  u32x4 q[MB][kChains];
  float m[MB], l[MB];
  f32x4 o[MB][kRun];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int b = 0; b < MB; ++b) {
      m[b] = -INFINITY;
      l[b] = 0.0f;
#pragma unroll
      for (int d = 0; d < kRun; ++d) o[b][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }

  // Whole words of scale bytes, here and of the values: what is loaded of a byte or two the compiler zero-extends at the loop's
  // end, where it waits for it. All 16 keys' bytes are there to read (a page holds whole sixteens); those of keys past the last
  // one belong to none, and their codes read as zeros.
  static __device__ __forceinline__ void load_keys(KeyTile &t, const KvArgs &kv, const Keys16 &k, int half,
                                                   uint32_t row_bytes, uint32_t lane) {
    const uint32_t r = lane & 15, kq = lane >> 4;
    const __amdgpu_buffer_rsrc_t codes = buffer_rsrc(kv.keys + k.at * row_bytes, k.count * row_bytes);
    const __amdgpu_buffer_rsrc_t by =
        buffer_rsrc((const uint8_t *)kv.key_scales + k.at * kGroups, k.count ? 16 * kGroups : 0);
#pragma unroll
    for (int j = 0; j < kKeyLoads; ++j) {
      const uint32_t at = DIM == 64 ? 8 * kq : 64 * j + 16 * kq, from = at < row_bytes ? r * row_bytes + at : kNowhere;
      if constexpr (DIM == 64) {
        const u32x2 v = buffer_b64(codes, from, 0);
        t.w[half][j] = u32x4{v[0], v[1], 0u, 0u};
      } else {
        t.w[half][j] = buffer_b128(codes, from, 0);
      }
      t.group[half][j] = buffer_b32(by, at < row_bytes ? (r * kGroups & ~3u) + 4 * j : kNowhere, 0);
    }
  }
  static __device__ __forceinline__ void load_values(ValueTile &t, const KvArgs &kv, const Keys16 &k, int half,
                                                     uint32_t row_bytes, uint32_t lane) {
    const uint32_t i = lane & 15, kq = lane >> 4, at = i * kRun / 2;
    const __amdgpu_buffer_rsrc_t codes = buffer_rsrc(kv.values + k.at * row_bytes, k.count * row_bytes);
    const __amdgpu_buffer_rsrc_t by =
        buffer_rsrc((const uint8_t *)kv.value_scales + k.at * kGroups, k.count ? 16 * kGroups : 0);
    // One select for the four keys: with one each the compiler branches round the loads.
    const uint32_t first = at < row_bytes ? 4 * kq * row_bytes + (at & ~3u) : kNowhere;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (kValueWords == 1) {
        t.w[half][e][0] = buffer_b32(codes, first + e * row_bytes, 0);
      } else {
        const u32x2 v = buffer_b64(codes, first + e * row_bytes, 0);
        t.w[half][e][0] = v[0];
        t.w[half][e][1] = v[1];
      }
    }
    const uint32_t scales = at < row_bytes ? 4 * kq * kGroups : kNowhere;
    if constexpr (DIM == 64) {
      const u32x2 v = buffer_b64(by, scales, 0);
      t.groups[half][0] = v[0];
      t.groups[half][1] = v[1];
    } else if constexpr (DIM == 128) {
      const u32x4 v = buffer_b128(by, scales, 0);
#pragma unroll
      for (int e = 0; e < 4; ++e) t.groups[half][e] = v[e];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) t.groups[half][e] = buffer_b32(by, scales + kGroups * e + 4 * (i / 8), 0);
    }
  }

  // Byte g of a word where fp4_pair reads it, the exponent's bits, among others that it does not: one instruction.
  static __device__ __forceinline__ uint32_t turned(uint32_t word, uint32_t g) {
    return __builtin_amdgcn_alignbit(word, word, 8 * g + 9);
  }
  // The scale of half h's key 4 kq + e for the lane's values (kRun of one group), in its place among others (TURNED) or alone.
  template <bool TURNED = false>
  static __device__ __forceinline__ uint32_t value_scale(const ValueTile &t, int h, int e, uint32_t lane) {
    const uint32_t i = lane & 15, word = t.groups[h][DIM == 64 ? e / 2 : e];
    const uint32_t g = DIM == 64 ? 2 * (e % 2) + i / 8 : DIM == 128 ? i / 4 : i / 2 % 4;
    return TURNED ? turned(word, g) : fp4_scale(word, g);
  }

  static __device__ __forceinline__ uint32_t query_at(int chain, uint32_t lane) {
    return DIM == 64 ? 16 * (lane >> 4) + 8 * chain : 128 * (chain / 4) + 32 * (lane >> 4) + 8 * (chain % 4);
  }

  // s = the raw products of 32 keys for block b's rows: half h's value i is key 16 h + 4 kq + i.
  __device__ __forceinline__ void scores(const KeyTile &t, f32x4 (&s)[MB][2], uint32_t lane) const {
    const uint32_t kq = lane >> 4;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int b = 0; b < MB; ++b) s[b][h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < kChains; ++c) {
        const uint32_t w = t.w[h][c / 4][c % 4], by = turned(t.group[h][c / 4], DIM == 64 ? 2 * (lane & 1) + kq / 2 : kq);
        const u32x4 k{fp4_pair(w, by, 0), fp4_pair(w, by, 1), fp4_pair(w, by, 2), fp4_pair(w, by, 3)};
#pragma unroll
        for (int b = 0; b < MB; ++b) s[b][h] = mfma_bf16(k, q[b][c], s[b][h]);
      }
    }
  }

  // Adds the weights' product with 32 keys' values, two values of a run at a time. rest: what the weights lost to their rounding.
  __device__ __forceinline__ void accumulate(const ValueTile &t, const u32x4 (&p)[MB], const u32x4 (&rest)[MB], uint32_t lane) {
    uint32_t by[2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 4; ++e) by[h][e] = value_scale<true>(t, h, e, lane);
#pragma unroll
    for (int j = 0; j < kRun / 2; ++j) {
      uint32_t w[2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          w[h][e] = fp4_pair(DIM == 64 ? t.w[h][e][0] >> (16 * (lane & 1)) : t.w[h][e][j / 4], by[h][e], j % 4);
      const u32x4 even{low_halves(w[0][0], w[0][1]), low_halves(w[0][2], w[0][3]), low_halves(w[1][0], w[1][1]),
                       low_halves(w[1][2], w[1][3])};
      const u32x4 odd{high_halves(w[0][0], w[0][1]), high_halves(w[0][2], w[0][3]), high_halves(w[1][0], w[1][1]),
                      high_halves(w[1][2], w[1][3])};
#pragma unroll
      for (int b = 0; b < MB; ++b) {
        o[b][2 * j] = mfma_bf16(even, p[b], o[b][2 * j]);
        o[b][2 * j + 1] = mfma_bf16(odd, p[b], o[b][2 * j + 1]);
      }
#pragma unroll
      for (int b = 0; b < MB; ++b) {
        o[b][2 * j] = mfma_bf16(even, rest[b], o[b][2 * j]);
        o[b][2 * j + 1] = mfma_bf16(odd, rest[b], o[b][2 * j + 1]);
      }
    }
  }

  // Whether a value of the tile may be an infinity or NaN, by its keys' scales.
  static __device__ __forceinline__ bool unbounded(const ValueTile &t, uint32_t lane) {
    bool any = false;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 4; ++e) any |= fp4_unbounded(value_scale(t, h, e, lane));
    return any;
  }

  // Infinities and NaNs (under bytes above 252) leave the tile where some rows see a key of it and others do not (they must not
  // reach the others through 0 * inf), and the rows that see them add their products one by one. Finite values under such bytes
  // stay, for the products with both halves of a weight. Bit 4 h + i of seen: key 16 h + 4 kq + i.
  __device__ __forceinline__ void set_apart(ValueTile &t, const KvArgs &kv, const Keys16 (&at)[2], const u32x4 (&p)[MB],
                                            const uint32_t (&seen)[MB], uint32_t row_bytes, uint32_t lane) {
    const uint32_t r = lane & 15, kq = lane >> 4;
#pragma unroll
    for (int b = 0; b < MB; ++b)
      for (int key = 0; key < kStep; ++key) {
        const int h = key / 16, i = key % 4, source = 16 * (key % 16 / 4) + (int)r;
        // By selects: an index known only at run time would put the weights in scratch memory.
        const uint32_t first = h ? p[b][2] : p[b][0], second = h ? p[b][3] : p[b][1];
        const uint32_t word = i / 2 ? second : first;
        const float weight = __uint_as_float((uint32_t)__shfl((int)(i % 2 ? word & 0xFFFF0000u : word << 16), source));
        const bool sees = (__shfl((int)seen[b], source) >> (4 * h + i)) & 1;
        const size_t place = h ? at[1].at : at[0].at;
        const uint32_t count = h ? at[1].count : at[0].count;
        const __amdgpu_buffer_rsrc_t codes = buffer_rsrc(kv.values + place * row_bytes, count * row_bytes);
        const __amdgpu_buffer_rsrc_t groups =
            buffer_rsrc((const uint8_t *)kv.value_scales + place * kGroups, count * kGroups);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int d = 0; d < kRun; d += 2) {
            const uint32_t value = kRun * (4 * kq + j) + d;
            if (value / 2 >= row_bytes) continue;
            const uint32_t by = buffer_b8(groups, (key % 16) * kGroups + value / 32, 0) << 23;
            if (!sees || !fp4_unbounded(by)) continue;
            const uint32_t two = fp4_pair(buffer_b8(codes, (key % 16) * row_bytes + value / 2, 0), by, 0);
            if ((two & 0x7F80u) == 0x7F80u) o[b][d][j] += weight * bf16_to_f32(two & 0xFFFFu);
            if ((two & 0x7F800000u) == 0x7F800000u) o[b][d + 1][j] += weight * __uint_as_float(two & 0xFFFF0000u);
          }
      }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t by = value_scale(t, h, e, lane) >> 23;
        if (by > 252)
#pragma unroll
          for (int i = 0; i < kValueWords; ++i) t.w[h][e][i] &= finite_codes4(t.w[h][e][i], by);
      }
      // The scales of NaNs too, whichever lane's they are: a byte of zero.
#pragma unroll
      for (int e = 0; e < kGroupWords; ++e)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          if (fp4_scale(t.groups[h][e], g) >> 23 == 255) t.groups[h][e] &= ~(0xFFu << (8 * g));
    }
  }
};

// A part's keys through the wave's state. low, high: the keys that the lane's rows see; slope, position: of its rows (scored).
template <int WAVES, int DIM, int MB, typename A>
__device__ __forceinline__ void run_four(const A &a, const Part<A> &part, Rows4<DIM, MB> &state, const KeySpan &span,
                                         const int (&low)[MB], const int (&high)[MB], const float (&slope)[MB],
                                         const int (&position)[MB], uint32_t wave, uint32_t lane) {
  using R = Rows4<DIM, MB>;
  constexpr int kDepth = attend_rows_depth(16 * MB, DIM, SQ_KV_E2M1), kStride = kStep * WAVES;
  const uint32_t kq = lane >> 4, row_bytes = a.kv.head_dim / 2;
  // The page table's entry of the 16 keys from k on (past the end the last key's), and their place: none there or in a hole.
  const auto page_at = [&](int k) __attribute__((always_inline)) {
    return a.kv.page_table[(size_t)part.sequence * a.kv.pages_per_sequence +
                           ((uint32_t)max(min(k, span.end - 1), 0) >> a.kv.page_shift)];
  };
  const auto keys_at = [&](int k, uint32_t entry) __attribute__((always_inline)) {
    const uint32_t page = uniform(entry);
    if (page >= a.kv.pages || k >= span.end) return Keys16{0, 0u};
    return Keys16{(((size_t)page * a.kv.kv_heads + part.head) << a.kv.page_shift) +
                      ((uint32_t)k & ((1u << a.kv.page_shift) - 1)),
                  (uint32_t)min(16, span.end - k)};
  };
  typename R::KeyTile keys[kDepth];
  typename R::ValueTile values[kDepth];
  Keys16 places[kDepth][2];
  int k = span.begin + kStep * (int)wave;
  const auto fetch_keys = [&](typename R::KeyTile &t, const Keys16 (&at)[2]) __attribute__((always_inline)) {
    R::load_keys(t, a.kv, at[0], 0, row_bytes, lane);
    R::load_keys(t, a.kv, at[1], 1, row_bytes, lane);
  };
  const auto fetch_values = [&](typename R::ValueTile &t, const Keys16 (&at)[2]) __attribute__((always_inline)) {
    R::load_values(t, a.kv, at[0], 0, row_bytes, lane);
    R::load_values(t, a.kv, at[1], 1, row_bytes, lane);
  };
  __builtin_amdgcn_s_waitcnt(0);   // nothing is pending, a store of the last part's that may be LDS's among it
  // Fetches run kDepth steps ahead of the products, and the page table's entries a step ahead of the fetches.
  uint32_t entry_a = page_at(k), entry_b = page_at(k + 16);
#pragma unroll
  for (int d = 0; d < kDepth; ++d) {
    const int at = k + d * kStride;
    places[d][0] = keys_at(at, entry_a);
    places[d][1] = keys_at(at + 16, entry_b);
    entry_a = page_at(at + kStride);
    entry_b = page_at(at + kStride + 16);
    __builtin_amdgcn_sched_barrier(0);   // the order of loads that a step counts on
    fetch_keys(keys[d], places[d]);
    fetch_values(values[d], places[d]);
  }
  const auto step = [&](typename R::KeyTile &kt, typename R::ValueTile &vt, Keys16 (&at)[2]) __attribute__((always_inline)) {
    const uint32_t hole = (at[0].count ? 0u : 1u) | (at[1].count ? 0u : 2u);
    const Keys16 next[2] = {keys_at(k + kDepth * kStride, entry_a), keys_at(k + kDepth * kStride + 16, entry_b)};
    entry_a = page_at(k + (kDepth + 1) * kStride);
    entry_b = page_at(k + (kDepth + 1) * kStride + 16);
    f32x4 s[MB][2];
    state.scores(kt, s, lane);
    fetch_keys(kt, next);

    const bool clear = k >= span.clear_begin && k + kStep <= span.clear_end && k + kStep <= span.end && !hole;
    uint32_t seen[MB];   // bit 4 h + i: key 16 h + 4 kq + i
#pragma unroll
    for (int b = 0; b < MB; ++b) {
      seen[b] = 0xFFu;
      if (!clear) {
        seen[b] = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int key = k + 16 * (i / 4) + 4 * (int)kq + i % 4;
          seen[b] |= (uint32_t)(key >= low[b] && key < high[b] && key < span.end && !(hole >> (i / 4) & 1)) << i;
        }
      }
    }
    u32x4 p[MB], rest[MB];
#pragma unroll
    for (int b = 0; b < MB; ++b) {
      float v[8], w[8], top = -INFINITY;
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = s[b][i / 4][i % 4] * a.scale;
      if constexpr (kScoredCall<A>) {
        if (a.cap != 0.0f)
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = capped(a, v[i]);
        if (a.slopes) {
          const float ahead = (float)(k + 4 * (int)kq - position[b]);   // of the lane's first key
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = fmaf(-slope[b], fabsf(ahead + (float)(16 * (i / 4) + i % 4)), v[i]);
        }
      }
      if (!clear)
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = seen[b] >> i & 1 ? v[i] : -INFINITY;
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmaxf(top, v[i]);
      if (__any(top > state.m[b] + kRaise)) {
        const float next_m = fmaxf(state.m[b], row_max(top));
        const float shrink = exp2_fast(state.m[b] - finite_max(next_m));
        state.m[b] = next_m;
        state.l[b] *= shrink;
#pragma unroll
        for (int d = 0; d < R::kRun; ++d) state.o[b][d] *= shrink;
      }
      const float from = finite_max(state.m[b]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        w[i] = exp2_fast(v[i] - from);
        state.l[b] += w[i];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[b][i] = high_halves(__float_as_uint(w[2 * i]), __float_as_uint(w[2 * i + 1]));
        rest[b][i] = bf16_pair(fmaf(w[2 * i], kMore, -__uint_as_float(p[b][i] << 16)),
                               fmaf(w[2 * i + 1], kMore, -__uint_as_float(p[b][i] & 0xFFFF0000u)));
      }
    }
    if (!clear && __any(R::unbounded(vt, lane))) state.set_apart(vt, a.kv, at, p, seen, row_bytes, lane);
    state.accumulate(vt, p, rest, lane);
    fetch_values(vt, next);
    at[0] = next[0];
    at[1] = next[1];
    k += kStride;
  };
  while (k < span.end) {
#pragma unroll
    for (int d = 0; d < kDepth; ++d)
      if (d == 0 || k < span.end) step(keys[d], values[d], places[d]);
  }
}

}  // namespace
}  // namespace sq::kern
