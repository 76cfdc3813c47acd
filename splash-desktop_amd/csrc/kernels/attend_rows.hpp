// Attention of few rows a key head (tiles of 16 or 32 rows times query heads): single tokens and verify lanes,
// bound by reading the cache once.
//
// No shared memory lies between the cache and the matrix units. A wave takes 32 keys a step, 16 of them (A) and the next
// 16 (B): S^T = K Q^T puts four keys of each row in a lane, 4 kq + i of A and of B for lane (kq, r) (l = 16 kq + r), and
// those eight are the contraction slots that the second product O^T = V^T P^T wants of the lane's weights, so P never
// moves. V^T then wants, in lane (kq, i), the keys 4 kq + e of A and B of one output value: the lane loads these eight
// keys' values c i .. c i + c - 1 (c = head_dim / 16, one vector a key), and the 2 x 2 transposes of v_perm make from
// them the operands of c matrix products, product d taking value c i + d of every lane: half an instruction a value, in
// the place of a pass through LDS. Products' rows i then hold values c i + d, so a lane's outputs are runs of c values.
// 8-bit codes become bf16 operands exactly (127 and e4m3's four bits both fit its eight); the scales of their tokens
// multiply the scores, and the weights before they are rounded.
//
// Heads of 256 of e4m3 spill 2 or 6 registers (12 or 28 bytes a lane), no others any.
//
// Loads go through buffer resources of 16 keys of one page (pages are whole multiples of 16 tokens): a key past the
// sequence, a page that is a hole and a value past head_dim all read zero, with no instruction spent on them.
//
// The matrix units take the weights in bf16, half a step of which is 2^-9 to 2^-8 of a weight, as much as the output's own
// rounding: where a few weights outweigh the rest, all of it shows. They go in as two, the weight rounded down and the rest
// (2^-16 of it is lost). Reading the cache hides the second products: a token over 131072 int8 keys takes 54 us either way,
// and is 0.0017 from 64 bits (its own rounding) for 0.0027. An infinite value meets both, so neither may be zero or
// negative where the weight is not (0 inf and inf - inf are NaN): hence down, and hence kMore.
//
// What it reaches: a token of 40 heads over 131072 int8 keys of 8 heads of 128 (277 MB) in 54 us, 5.1 TB/s (a large copy
// reaches 4.9); a token each of 64 sequences of 200 to 8000 e4m3 keys (291 MB) in 63 us, 4.6 TB/s; one over 700 bf16 keys,
// which is a chain of round trips (lengths, page table, keys, the waves' join), in 14 us.
//
// Softmax: each wave keeps its own running maximum, lane sums and accumulators, and raises the maximum (which costs
// lane exchanges and a pass over the accumulators) only when a score exceeds it by 8 (a factor of 256, which fp32 sums
// and bf16's exponent hold without loss); the waves of a workgroup join at the end of a part, through LDS.
#pragma once
#include "attend.hpp"
#include "device.hpp"

namespace sq::kern {
namespace {

constexpr int kStep = 32;      // keys a wave takes a step
// What all weights are multiplied by on their way into the second product, so that the rest of one that bf16 holds exactly
// is 2^-18 of it and not zero. The outputs grow by as much, a 2^-10 of their own rounding. (The rest of a weight below
// 2^-108 leaves bf16's normal range: an infinite value under it may give NaN, as it does in fp32 where e^x has become 0.)
constexpr float kMore = 1 + 0x1p-18f;

// Four e4m3 codes, NaNs as zeros.
__device__ __forceinline__ uint32_t finite_codes(uint32_t w) {
  const uint32_t nan = nan_codes(w);
  return w & ~(nan | (nan - (nan >> 7)));
}
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

// DIM: the head's values as computed (64, 128 or 256; values past head_dim are zero). MB: blocks of 16 rows.
template <uint32_t FMT, int DIM, int MB>
struct Rows {
  static constexpr bool kFour = FMT == SQ_KV_E2M1;
  static constexpr bool kScaled = FMT == SQ_KV_INT8 || FMT == SQ_KV_E4M3;   // a scale a token
  static constexpr int kBits = kFour ? 4 : kScaled ? 8 : 16, kRun = DIM / 16, kChains = DIM / 32;
  // Vectors a lane loads for its share of 16 keys: K 16 bytes each (heads of 64 in 4 bits: 8 of them), V kRun values a key
  // (the same: 2 bytes).
  static constexpr int kKeyLoads = DIM * kBits < 512 ? 1 : DIM * kBits / 512;
  static constexpr int kValueWords = kRun * kBits < 32 ? 1 : kRun * kBits / 32;
  static constexpr uint32_t kGroups = DIM / 32;   // scale bytes of a head row in 4 bits
  static constexpr int kGroupWords = DIM == 64 ? 2 : 4;
  static __device__ __forceinline__ uint32_t bytes_of(uint32_t values) { return values * kBits / 8; }

  struct KeyTile {
    u32x4 w[2][kKeyLoads];
    f32x4 scale[2];
    uint32_t group[kFour ? 2 : 1][kKeyLoads];   // the word with each vector's scale byte
  };
  struct ValueTile {
    uint32_t w[2][4][kValueWords];   // (heads of 64 in 4 bits: the lane's half of it)
    f32x4 scale[2];
    uint32_t groups[kFour ? 2 : 1][kGroupWords];   // the lane's four keys' scale bytes (two keys a word: heads of 64)
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

  static __device__ __forceinline__ void load_keys(KeyTile &t, const KvArgs &kv, const Keys16 &k, int half,
                                                   uint32_t row_bytes, uint32_t lane) {
    const __amdgpu_buffer_rsrc_t r = buffer_rsrc(kv.keys + k.at * row_bytes, k.count * row_bytes);
    if constexpr (kFour) {
      // A vector is one group's (half of one's, heads of 64). Whole words, here and of the values: the compiler zero-extends
      // what it loads of a byte or two at the loop's end, where it waits for it.
      const __amdgpu_buffer_rsrc_t by =
          buffer_rsrc((const uint8_t *)kv.key_scales + k.at * kGroups, k.count ? 16 * kGroups : 0);
#pragma unroll
      for (int j = 0; j < kKeyLoads; ++j) {
        const uint32_t at = DIM == 64 ? 8 * (lane >> 4) : 64 * j + 16 * (lane >> 4);
        const uint32_t from = at < row_bytes ? (lane & 15) * row_bytes + at : kNowhere;
        if constexpr (DIM == 64) {
          const u32x2 v = buffer_b64(r, from, 0);
          t.w[half][j] = u32x4{v[0], v[1], 0u, 0u};
        } else {
          t.w[half][j] = buffer_b128(r, from, 0);
        }
        t.group[half][j] = buffer_b32(by, at < row_bytes ? ((lane & 15) * kGroups & ~3u) + 4 * j : kNowhere, 0);
      }
      return;
    }
#pragma unroll
    for (int j = 0; j < kKeyLoads; ++j) {
      const uint32_t at = 64 * j + 16 * (lane >> 4);
      t.w[half][j] = buffer_b128(r, at < row_bytes ? (lane & 15) * row_bytes + at : kNowhere, 0);
    }
    if constexpr (kScaled)
      t.scale[half] = __builtin_bit_cast(f32x4, buffer_b128(buffer_rsrc(kv.key_scales + k.at, k.count ? 64 : 0), 16 * (lane >> 4), 0));
  }
  static __device__ __forceinline__ void load_values(ValueTile &t, const KvArgs &kv, const Keys16 &k, int half,
                                                     uint32_t row_bytes, uint32_t lane) {
    const __amdgpu_buffer_rsrc_t r = buffer_rsrc(kv.values + k.at * row_bytes, k.count * row_bytes);
    const uint32_t at = (lane & 15) * kRun * kBits / 8;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      uint32_t from = at < row_bytes ? (4 * (lane >> 4) + e) * row_bytes + at : kNowhere;
      // One select for the four keys, or the compiler branches round each of these loads and waits for all of them.
      if constexpr (kFour) from = (at < row_bytes ? 4 * (lane >> 4) * row_bytes + at : kNowhere) + e * row_bytes;
      if constexpr (kRun * kBits == 16) {
        t.w[half][e][0] = buffer_b32(r, from & ~3u, 0);
      } else if constexpr (kValueWords == 1) {
        t.w[half][e][0] = buffer_b32(r, from, 0);
      } else if constexpr (kValueWords == 2) {
        const u32x2 v = buffer_b64(r, from, 0);
        t.w[half][e][0] = v[0];
        t.w[half][e][1] = v[1];
      } else {
#pragma unroll
        for (int i = 0; i < kValueWords / 4; ++i) {
          const u32x4 v = buffer_b128(r, from + 16 * i, 0);
#pragma unroll
          for (int j = 0; j < 4; ++j) t.w[half][e][4 * i + j] = v[j];
        }
      }
    }
    if constexpr (kFour) {
      // All 16 keys' bytes are there to read (a page holds whole sixteens): those of keys past the last one belong to none.
      const __amdgpu_buffer_rsrc_t by =
          buffer_rsrc((const uint8_t *)kv.value_scales + k.at * kGroups, k.count ? 16 * kGroups : 0);
      const uint32_t first = at < row_bytes ? 4 * (lane >> 4) * kGroups : kNowhere;
      if constexpr (DIM == 64) {
        const u32x2 v = buffer_b64(by, first, 0);
        t.groups[half][0] = v[0];
        t.groups[half][1] = v[1];
      } else if constexpr (DIM == 128) {
        const u32x4 v = buffer_b128(by, first, 0);
#pragma unroll
        for (int e = 0; e < 4; ++e) t.groups[half][e] = v[e];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) t.groups[half][e] = buffer_b32(by, first + kGroups * e + 4 * ((lane & 15) / 8), 0);
      }
    }
    if constexpr (kScaled)
      t.scale[half] =
          __builtin_bit_cast(f32x4, buffer_b128(buffer_rsrc(kv.value_scales + k.at, k.count ? 64 : 0), 16 * (lane >> 4), 0));
  }

  // Byte g of a word where fp4_pair reads it, the exponent's bits, among others that it does not: one instruction.
  static __device__ __forceinline__ uint32_t turned(uint32_t word, uint32_t g) {
    return __builtin_amdgcn_alignbit(word, word, 8 * g + 9);
  }
  // The scale of half h's key 4 kq + e for the lane's values (kRun of one group), in its place (turned) or alone.
  template <bool TURNED = false>
  static __device__ __forceinline__ uint32_t value_scale(const ValueTile &t, int h, int e, uint32_t lane) {
    const uint32_t i = lane & 15, word = t.groups[h][DIM == 64 ? e / 2 : e];
    const uint32_t g = DIM == 64 ? 2 * (e % 2) + i / 8 : DIM == 128 ? i / 4 : i / 2 % 4;
    return TURNED ? turned(word, g) : fp4_scale(word, g);
  }

  // The rows' values in the K operand's order: bf16 chain j takes values 32 j + 8 kq + e; of codes, whose 16-byte vector
  // holds 16 values, chains 2 j and 2 j + 1 take values 64 j + 16 kq + e and + 8 + e; in 4 bits, of whose 32 a vector chains
  // 4 j to 4 j + 3 take 8 each, values 128 j + 32 kq + 8 (chain - 4 j) + e.
  static __device__ __forceinline__ uint32_t query_at(int chain, uint32_t lane) {
    if constexpr (kFour)
      return DIM == 64 ? 16 * (lane >> 4) + 8 * chain : 128 * (chain / 4) + 32 * (lane >> 4) + 8 * (chain % 4);
    return kScaled ? 64 * (chain / 2) + 16 * (lane >> 4) + 8 * (chain % 2) : 32 * chain + 8 * (lane >> 4);
  }

  // The scale of a lane's vector j of half h's keys.
  static __device__ __forceinline__ uint32_t key_scale(const KeyTile &t, int h, int j, uint32_t lane) {
    const uint32_t kq = lane >> 4;
    return turned(t.group[h][j], DIM == 64 ? 2 * (lane & 1) + kq / 2 : kq);
  }
  static __device__ __forceinline__ u32x4 key_operand(const KeyTile &t, int half, int chain, uint32_t lane) {
    if constexpr (kFour) {
      const uint32_t w = t.w[half][chain / 4][chain % 4], by = key_scale(t, half, chain / 4, lane);
      return u32x4{fp4_pair(w, by, 0), fp4_pair(w, by, 1), fp4_pair(w, by, 2), fp4_pair(w, by, 3)};
    } else if constexpr (!kScaled) {
      return t.w[half][chain];
    } else {
      const u32x4 w = t.w[half][chain / 2];
      const u32x2 a = code_pairs4<FMT>(w[2 * (chain % 2)]), b = code_pairs4<FMT>(w[2 * (chain % 2) + 1]);
      return u32x4{a[0], a[1], b[0], b[1]};
    }
  }

  // s = the raw products of 32 keys for block b's rows: half h's value i is key 16 h + 4 kq + i.
  __device__ __forceinline__ void scores(const KeyTile &t, f32x4 (&s)[MB][2], uint32_t lane) const {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int b = 0; b < MB; ++b) s[b][h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < kChains; ++c) {
        const u32x4 k = key_operand(t, h, c, lane);
#pragma unroll
        for (int b = 0; b < MB; ++b) s[b][h] = mfma_bf16(k, q[b][c], s[b][h]);
      }
    }
  }

  // The operands of values 2 j and 2 j + 1 of a run, from each key's word of them as bf16.
  static __device__ __forceinline__ void value_operands(const uint32_t (&w)[2][4], u32x4 &even, u32x4 &odd) {
    even = u32x4{low_halves(w[0][0], w[0][1]), low_halves(w[0][2], w[0][3]), low_halves(w[1][0], w[1][1]),
                 low_halves(w[1][2], w[1][3])};
    odd = u32x4{high_halves(w[0][0], w[0][1]), high_halves(w[0][2], w[0][3]), high_halves(w[1][0], w[1][1]),
                high_halves(w[1][2], w[1][3])};
  }

  // Adds the weights' product with 32 keys' values. Two values of a run at a time. rest: what the weights lost to their
  // rounding.
  __device__ __forceinline__ void accumulate(const ValueTile &t, const u32x4 (&p)[MB], const u32x4 (&rest)[MB], uint32_t lane) {
    uint32_t by[2][4];
    if constexpr (kFour)
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
        for (int e = 0; e < 4; ++e) {
          if constexpr (kFour) w[h][e] = fp4_pair(DIM == 64 ? t.w[h][e][0] >> (16 * (lane & 1)) : t.w[h][e][j / 4], by[h][e], j % 4);
          else if constexpr (!kScaled) w[h][e] = t.w[h][e][j];
          else w[h][e] = code_pairs4<FMT>(t.w[h][e][j / 2])[j % 2];
        }
      u32x4 even, odd;
      value_operands(w, even, odd);
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

  // e4m3's NaN codes leave the tile, and the accumulators of the rows that see them become NaN: products of large values in
  // the places of such codes and of keys seen, which overflow, once to infinity and once below it, leave NaNs, and add zeros
  // to all other accumulators. (Bit 4 h + i of seen: key 16 h + 4 kq + i.) A word of each key at a time: this hardly ever
  // runs, and takes no more registers than the kernel has.
  __device__ __forceinline__ void take_nans(ValueTile &t, const uint32_t (&seen)[MB]) {
    constexpr uint32_t kLarge = 0x7Eu, kHuge = 0x7F00u;   // e4m3's 448, bf16's 2^127
#pragma unroll
    for (int i = 0; i < kValueWords; ++i) {
      uint32_t at[2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t &word = t.w[h][e][i];
          asm volatile("" : "+v"(word));   // or the terms of the check before would wait in registers for their use here
          at[h][e] = (nan_codes(word) >> 7) * kLarge;
          word = finite_codes(word);
        }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint32_t w[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) w[h][e] = code_pairs4<FMT>(at[h][e])[j];
        u32x4 even, odd;
        value_operands(w, even, odd);
#pragma unroll
        for (int b = 0; b < MB; ++b) {
          uint32_t bits = seen[b];
          asm volatile("" : "+v"(bits));
          u32x4 sees;
#pragma unroll
          for (int n = 0; n < 4; ++n) sees[n] = (bits >> (2 * n) & 1) * kHuge | (bits >> (2 * n + 1) & 1) * (kHuge << 16);
          f32x4 &first = o[b][4 * i + 2 * j], &second = o[b][4 * i + 2 * j + 1];
          first = mfma_bf16(even, sees, first);
          second = mfma_bf16(odd, sees, second);
          sees ^= 0x80008000u;
          first = mfma_bf16(even, sees, first);
          second = mfma_bf16(odd, sees, second);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
};

// Whether any value of a tile is an infinity or NaN (e4m3's: its NaN code).
template <uint32_t FMT, int N>
__device__ __forceinline__ bool unbounded(const uint32_t (&w)[2][4][N]) {
  uint32_t any = 0;
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if constexpr (FMT == SQ_KV_E4M3) any |= nan_codes(w[h][e][i]);
        else any |= (uint32_t)((w[h][e][i] & 0x7F80u) == 0x7F80u) | (uint32_t)((w[h][e][i] & 0x7F800000u) == 0x7F800000u);
      }
  return any != 0;
}

// The same of a tile in 4 bits, by its keys' scales: whether a value may be one.
template <typename R>
__device__ __forceinline__ bool unbounded4(const typename R::ValueTile &t, uint32_t lane) {
  bool any = false;
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int e = 0; e < 4; ++e) any |= fp4_unbounded(R::value_scale(t, h, e, lane));
  return any;
}

template <int MB, int WAVES, typename A>
struct Shared {
  LineShared<64 * WAVES, A> line;
  f32x4 waves[WAVES][WAVES][64];   // of each wave 4 WAVES accumulators at once, a vector of four for each to sum
  float maxima[WAVES][MB][16], sums[WAVES][MB][16];
};

template <uint32_t FMT, int DIM, int MB, int WAVES, typename A>
__global__ __launch_bounds__(64 * WAVES, (WAVES == 8 ? 2 : attend_rows_resident(16 * MB, DIM, FMT))) void
attend_rows_kernel(A a) {
  constexpr bool kScored = kScoredCall<A>;
  using R = Rows<FMT, DIM, MB>;
  constexpr int kWaves = WAVES, kThreads = 64 * WAVES, kJoin = 4 * WAVES;
  constexpr bool kScaled = R::kScaled;
  // Accumulator t = kRun j + d of a block is value d of run j.
  constexpr int kRun = R::kRun, kRegs = 4 * kRun, kChunks = (kRegs + kJoin - 1) / kJoin;
  constexpr int kVectors = kRegs < kJoin ? kRegs / 4 : kJoin / 4;   // of four accumulators, in a chunk
  constexpr int kBlockFloats = 16 * (DIM + 2);   // of a part in the workspace
  __shared__ Shared<MB, WAVES, A> shared;
  const uint32_t lane = threadIdx.x & 63, r = lane & 15, kq = lane >> 4;
  const uint32_t wave = uniform(threadIdx.x >> 6);
  const Cut cut{16 * MB / (int)a.group, (int)kAttendLeast, kUnitSlack + 256};
  const float by_group = 1.0f / (float)a.group;
  const uint32_t dim = a.kv.head_dim, row_bytes = R::bytes_of(dim);
  Part<A> next;
  Work<kThreads, A> work = make_work<kThreads>(a, cut, shared.line, next);
  UnitNote began{};
  while (work.next(a, cut, shared.line, next)) {
    const Part<A> part = settled(a, cut, next);
    const Units<A> &u = part.units;
    const int row0 = cut.fit * part.m, rows = min(cut.fit, u.rows - row0), live = rows * (int)a.group;
    int unit_end = u.causal ? min(u.keys, u.base + row0 + rows) : u.keys;   // keys that any row sees
    if constexpr (kScored) unit_end = max(unit_end, u.bounds.prefix);
    const int tile0 = u.first_tile(part.m);
    const int k_begin = kKeyTile * (tile0 + part.t0), k_end = min(unit_end, kKeyTile * (tile0 + part.t1));
    // Keys [clear_begin, clear_end) are seen by every row of the unit.
    int clear_begin = u.window ? u.base + row0 + rows - u.window : 0;
    int clear_end = u.causal ? u.base + row0 + 1 : u.keys;
    if constexpr (kScored) {
      clear_begin = max(clear_begin, u.bounds.begin);
      if (u.base + row0 >= 0) clear_end = max(clear_end, u.bounds.prefix);
    }

    R state;
    state.clear();
    int low[MB], high[MB];   // the keys this lane's rows see
    float slope[MB];         // scored: of the lane's heads, in powers of two
    int position[MB];
#pragma unroll
    for (int b = 0; b < MB; ++b) {
      const int p = 16 * b + (int)r, i = row_of(p, by_group), g = p - i * (int)a.group;
      const int at = u.base + row0 + i;
      low[b] = u.window ? at - u.window + 1 : 0;
      high[b] = u.causal ? min(at + 1, u.keys) : u.keys;
      const bool on = p < live;
      if constexpr (kScored) {
        low[b] = max(low[b], u.bounds.begin);
        if (at >= 0) high[b] = max(high[b], u.bounds.prefix);
        slope[b] = on && a.slopes ? a.slopes[part.head * a.group + g] * 1.44269504089f : 0.0f;
        position[b] = at;
      }
      const uint16_t *row = a.query + (size_t)(part.first_row + row0 + (on ? i : 0)) * a.query_stride +
                            (part.head * a.group + (on ? g : 0)) * dim;
#pragma unroll
      for (int c = 0; c < R::kChains; ++c) {
        const uint32_t d = R::query_at(c, lane);
        state.q[b][c] = on && d < dim ? (*(const u32x4 *)(row + d) & a.keep) ^ a.flip : u32x4{0u, 0u, 0u, 0u};
      }
    }

    // The page of the 16 keys from k on as the table has it (~0u past the part's keys), and their place: none in a hole.
    constexpr int kDepth = attend_rows_depth(16 * MB, DIM, FMT);   // steps in flight
    const auto page_at = [&](int k) __attribute__((always_inline)) {
      // Several steps in flight: loads on every path alike (past the end the last key's entry, and no keys), so that a step
      // waits for its own tile and not, as where paths with fewer loads meet, for all of them.
      if constexpr (kDepth > 1)
        return a.kv.page_table[(size_t)part.sequence * a.kv.pages_per_sequence +
                               ((uint32_t)max(min(k, k_end - 1), 0) >> a.kv.page_shift)];
      return k < k_end ? a.kv.page_table[(size_t)part.sequence * a.kv.pages_per_sequence +
                                         ((uint32_t)k >> a.kv.page_shift)]
                       : ~0u;
    };
    const auto keys_at = [&](int k, uint32_t entry) __attribute__((always_inline)) {
      const uint32_t page = uniform(entry);
      if (page >= a.kv.pages || (kDepth > 1 && k >= k_end)) return Keys16{0, 0u};
      return Keys16{(((size_t)page * a.kv.kv_heads + part.head) << a.kv.page_shift) +
                        ((uint32_t)k & ((1u << a.kv.page_shift) - 1)),
                    (uint32_t)min(16, k_end - k)};
    };

    typename R::KeyTile kts[kDepth];
    typename R::ValueTile vts[kDepth];
    Keys16 kas[kDepth], kbs[kDepth];
    int k = k_begin + kStep * (int)wave;
    const auto fetch_keys = [&](typename R::KeyTile &kt, const Keys16 &ka, const Keys16 &kb) __attribute__((always_inline)) {
      R::load_keys(kt, a.kv, ka, 0, row_bytes, lane);
      R::load_keys(kt, a.kv, kb, 1, row_bytes, lane);
    };
    const auto fetch_values = [&](typename R::ValueTile &vt, const Keys16 &ka, const Keys16 &kb) __attribute__((always_inline)) {
      R::load_values(vt, a.kv, ka, 0, row_bytes, lane);
      R::load_values(vt, a.kv, kb, 1, row_bytes, lane);
    };
    // Nothing is pending here: a store to memory that the compiler takes for LDS's too, left from the last part, would make each
    // step wait for every load.
    if constexpr (kDepth > 1) __builtin_amdgcn_s_waitcnt(0);
    // Fetches run kDepth steps ahead of the products, and the page table's entries a step ahead of the fetches.
    constexpr int kStride = kStep * kWaves;
    uint32_t entry_a = page_at(k), entry_b = page_at(k + 16);
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      const int at = k + d * kStride;
      kas[d] = keys_at(at, entry_a);
      kbs[d] = keys_at(at + 16, entry_b);
      entry_a = page_at(at + kStride);
      entry_b = page_at(at + kStride + 16);
      if constexpr (kDepth > 1) __builtin_amdgcn_sched_barrier(0);   // the order of loads that a step counts on
      if (kDepth > 1 || at < k_end) {
        fetch_keys(kts[d], kas[d], kbs[d]);
        fetch_values(vts[d], kas[d], kbs[d]);
      }
    }
    const auto step = [&](typename R::KeyTile &kt, typename R::ValueTile &vt, Keys16 &ka, Keys16 &kb)
                          __attribute__((always_inline)) {
      const bool more = kDepth > 1 || k + kStride < k_end;
      const uint32_t hole = (ka.count ? 0u : 1u) | (kb.count ? 0u : 2u);
      const Keys16 na = keys_at(k + kDepth * kStride, entry_a), nb = keys_at(k + kDepth * kStride + 16, entry_b);
      entry_a = page_at(k + (kDepth + 1) * kStride);
      entry_b = page_at(k + (kDepth + 1) * kStride + 16);
      f32x4 s[MB][2];
      state.scores(kt, s, lane);
      f32x4 key_scale[2], value_scale[2];
      if constexpr (kScaled) {
        key_scale[0] = kt.scale[0] * a.scale;
        key_scale[1] = kt.scale[1] * a.scale;
        value_scale[0] = vt.scale[0];
        value_scale[1] = vt.scale[1];
      }
      if (more) fetch_keys(kt, na, nb);

      const bool clear = k >= clear_begin && k + kStep <= clear_end && k + kStep <= k_end && !hole;
      uint32_t seen[MB];   // bit 4 h + i: key 16 h + 4 kq + i
#pragma unroll
      for (int b = 0; b < MB; ++b) {
        seen[b] = 0xFFu;
        if (!clear) {
          seen[b] = 0;
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int key = k + 16 * h + 4 * (int)kq + i;
              seen[b] |= (uint32_t)(key >= low[b] && key < high[b] && key < k_end && !(hole >> h & 1)) << (4 * h + i);
            }
        }
      }
      u32x4 p[MB], rest[MB];
#pragma unroll
      for (int b = 0; b < MB; ++b) {
        float v[8], top = -INFINITY;
        if constexpr (kScored) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float t = s[b][i / 4][i % 4];
            s[b][i / 4][i % 4] = kScaled ? t * key_scale[i / 4][i % 4] : t * a.scale;
          }
          if (a.cap != 0.0f)
#pragma unroll
            for (int i = 0; i < 8; ++i) s[b][i / 4][i % 4] = capped(a, s[b][i / 4][i % 4]);
          if (a.slopes) {
            const float ahead = (float)(k + 4 * (int)kq - position[b]);   // of the lane's first key
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float away = fabsf(ahead + (float)(16 * (i / 4) + i % 4));
              s[b][i / 4][i % 4] = fmaf(-slope[b], away, s[b][i / 4][i % 4]);
            }
          }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float t = kScored   ? s[b][h][i]
                            : kScaled ? s[b][h][i] * key_scale[h][i]
                                      : s[b][h][i] * a.scale;
            v[4 * h + i] = (R::kFour && kDepth > 1) || clear || (seen[b] >> (4 * h + i) & 1) ? t : -INFINITY;
            if constexpr (!R::kFour || kDepth == 1) top = fmaxf(top, v[4 * h + i]);
          }
        if constexpr (R::kFour && kDepth > 1) {   // in 4 bits the VALU counts: no selects where all keys are seen
          if (!clear)
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = seen[b] >> i & 1 ? v[i] : -INFINITY;
#pragma unroll
          for (int i = 0; i < 8; ++i) top = fmaxf(top, v[i]);
        }
        if (__any(top > state.m[b] + kRaise)) {
          const float next = fmaxf(state.m[b], row_max(top));
          const float shrink = exp2_fast(state.m[b] - finite_max(next));
          state.m[b] = next;
          state.l[b] *= shrink;
#pragma unroll
          for (int d = 0; d < kRun; ++d) state.o[b][d] *= shrink;
        }
        const float from = finite_max(state.m[b]);
        float w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          w[i] = exp2_fast(v[i] - from);
          state.l[b] += w[i];
        }
        if constexpr (kScaled) {
          // A scale past the row's keys may be anything (a NaN of its own row among it): no product with it there.
#pragma unroll
          for (int i = 0; i < 8; ++i)
            w[i] = clear || (seen[b] >> i & 1) ? w[i] * value_scale[i / 4][i % 4] : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p[b][i] = high_halves(__float_as_uint(w[2 * i]), __float_as_uint(w[2 * i + 1]));
          rest[b][i] = bf16_pair(fmaf(w[2 * i], kMore, -__uint_as_float(p[b][i] << 16)),
                                 fmaf(w[2 * i + 1], kMore, -__uint_as_float(p[b][i] & 0xFFFF0000u)));
        }
      }
      if constexpr (!kScaled) {
        // Where some rows see a key and others do not, its values must not reach the others through 0 * inf: infinities
        // and NaNs leave the tile, and the rows that see them add their products one by one.
        bool some = false;
        if (!clear) {
          if constexpr (R::kFour) some = unbounded4<R>(vt, lane);
          else some = unbounded<FMT>(vt.w);
        }
        if (!clear && __any(some)) {
#pragma unroll
          for (int b = 0; b < MB; ++b)
            for (int key = 0; key < kStep; ++key) {
              const int h = key / 16, i = key % 4, source = 16 * (key % 16 / 4) + (int)r;
              // By selects: an index known only at run time would put the weights in scratch memory.
              const uint32_t first = h ? p[b][2] : p[b][0], second = h ? p[b][3] : p[b][1];
              const uint32_t word = i / 2 ? second : first;
              const float weight = __uint_as_float((uint32_t)__shfl((int)(i % 2 ? word & 0xFFFF0000u : word << 16), source));
              const bool sees = (__shfl((int)seen[b], source) >> (4 * h + i)) & 1;
              const Keys16 &from = h ? kb : ka;
              const __amdgpu_buffer_rsrc_t values =
                  buffer_rsrc(a.kv.values + from.at * row_bytes, from.count * row_bytes);
              const __amdgpu_buffer_rsrc_t groups = buffer_rsrc(
                  (const uint8_t *)a.kv.value_scales + from.at * R::kGroups, R::kFour ? from.count * R::kGroups : 0);
#pragma unroll
              for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int d = 0; d < kRun; d += 2) {
                  const uint32_t at = kRun * (4 * kq + j) + d;
                  if constexpr (R::kFour) {
                    // All of a group under a byte above 252, of 253 and 254 the finite ones too.
                    const uint32_t by =
                        at < dim ? buffer_b8(groups, (key % 16) * R::kGroups + at / 32, 0) << 23 : 0u;
                    if (sees && fp4_unbounded(by)) {
                      const uint32_t two = fp4_pair(buffer_b8(values, (key % 16) * row_bytes + at / 2, 0), by, 0);
                      state.o[b][d][j] += weight * bf16_to_f32(two & 0xFFFFu);
                      state.o[b][d + 1][j] += weight * __uint_as_float(two & 0xFFFF0000u);
                    }
                    continue;
                  }
                  const uint32_t two = at < dim ? buffer_b32(values, (key % 16) * row_bytes + 2 * at, 0) : 0u;
                  if (sees && (two & 0x7F80u) == 0x7F80u) state.o[b][d][j] += weight * bf16_to_f32(two & 0xFFFFu);
                  if (sees && (two & 0x7F800000u) == 0x7F800000u)
                    state.o[b][d + 1][j] += weight * __uint_as_float(two & 0xFFFF0000u);
                }
            }
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
              for (int i = 0; i < R::kValueWords; ++i) {
                uint32_t &word = vt.w[h][e][i];
                if constexpr (R::kFour) {
                  if (fp4_unbounded(R::value_scale(vt, h, e, lane))) word = 0;
                } else {
                  if ((word & 0x7F80u) == 0x7F80u) word &= 0xFFFF0000u;
                  if ((word & 0x7F800000u) == 0x7F800000u) word &= 0x0000FFFFu;
                }
              }
          if constexpr (R::kFour) {
            // Their scales too, whichever lane's they are: a byte of zero.
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int e = 0; e < R::kGroupWords; ++e) {
                uint32_t &word = vt.groups[h][e];
#pragma unroll
                for (int g = 0; g < 4; ++g)
                  if (fp4_unbounded(fp4_scale(word, g))) word &= ~(0xFFu << (8 * g));
              }
          }
        }
      }
      if constexpr (FMT == SQ_KV_E4M3) {
        // The same of NaN codes. (No write makes one, but pages may hold them that have not been written yet, or by another.)
        if (!clear && __any(unbounded<FMT>(vt.w))) state.take_nans(vt, seen);
      }
      state.accumulate(vt, p, rest, lane);
      if (more) fetch_values(vt, na, nb);
      ka = na;
      kb = nb;
      k += kStride;
    };
    while (k < k_end) {
#pragma unroll
      for (int d = 0; d < kDepth; ++d)
        if (d == 0 || k < k_end) step(kts[d], vts[d], kas[d], kbs[d]);
    }
#pragma unroll
    for (int b = 0; b < MB; ++b) state.l[b] = row_sum(state.l[b]);

    // finish(b, c, sum): accumulators kJoin c + 4 wave .. + 3 of block b over every wave, for waves below kVectors.
    const auto write = [&](int b, int c, f32x4 sum, float total) __attribute__((always_inline)) {
      const int p = 16 * b + (int)r, i = row_of(p, by_group), g = p - i * (int)a.group;
      const uint32_t acc = kJoin * c + 4 * wave, value = kRun * (4 * kq + acc / kRun) + acc % kRun;
      if (p >= live || value >= dim) return;
      const float by = total == 0.0f ? 0.0f : 1.0f / total;
      uint16_t *out = a.output + (size_t)(part.first_row + row0 + i) * a.output_stride +
                      (part.head * a.group + g) * dim + value;
      *(u32x2 *)out = u32x2{bf16_pair(sum[0] * by, sum[1] * by), bf16_pair(sum[2] * by, sum[3] * by)};
    };
    if (part.parts > 1 && part.part == 0) began = {part.parts, (uint32_t)live, part.first_row + (uint32_t)row0, part.head};
    __syncthreads();   // the last join has been read
    if (lane < 16) {
#pragma unroll
      for (int b = 0; b < MB; ++b) {
        shared.maxima[wave][b][lane] = state.m[b];
        shared.sums[wave][b][lane] = state.l[b];
      }
    }
#pragma unroll
    for (int b = 0; b < MB; ++b) {
      float top = -INFINITY, total = 0.0f, by[kWaves];
      float *mine = a.partials + part_block(a, part.first_piece, part.part, b) * kBlockFloats;
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        if (b || c) __syncthreads();
#pragma unroll
        for (int v = 0; v < kVectors; ++v) {
          f32x4 four;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int acc = kJoin * c + 4 * v + i;
            four[i] = state.o[b][acc % kRun][acc / kRun];
          }
          shared.waves[wave][v][lane] = four;
        }
        __syncthreads();
        if (c == 0) {
#pragma unroll
          for (int w = 0; w < kWaves; ++w) top = fmaxf(top, shared.maxima[w][b][r]);
#pragma unroll
          for (int w = 0; w < kWaves; ++w) {
            // A wave that saw nothing adds nothing, even to a row whose maximum is infinite.
            const float l = shared.sums[w][b][r];
            by[w] = l == 0.0f ? 0.0f : exp2_fast(shared.maxima[w][b][r] - finite_max(top));
            total += l * by[w];
          }
        }
        if ((int)wave >= kVectors) continue;
        f32x4 sum = shared.waves[0][wave][lane] * by[0];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) sum += shared.waves[w][wave][lane] * by[w];
        if (part.parts == 1) {
          write(b, c, sum, total);
        } else if (16 * b + (int)r < live) {
          *(f32x4 *)(mine + ((c * kVectors + wave) * 64 + lane) * 4) = sum;
        }
      }
      if (part.parts > 1 && wave == 0 && lane < 16) {
        float *row = mine + 16 * DIM + 2 * lane;
        row[0] = top;
        row[1] = total;
      }
    }
  }
  work.leave(a, began);
}

template <uint32_t FMT, int DIM, int MB, typename A>
hipError_t launch_one(uint32_t waves, const A &a, hipStream_t stream) {
  if constexpr (attend_rows_resident(16 * MB, DIM, FMT) > 1) {
    if (waves == 8) {
      hipLaunchKernelGGL((attend_rows_kernel<FMT, DIM, MB, 8, A>), dim3(a.workgroups), dim3(512), 0, stream, a);
      return hipGetLastError();
    }
  }
  if (waves != 4) return hipErrorInvalidValue;
  hipLaunchKernelGGL((attend_rows_kernel<FMT, DIM, MB, 4, A>), dim3(a.workgroups), dim3(256), 0, stream, a);
  return hipGetLastError();
}
template <uint32_t FMT, int DIM, typename A>
hipError_t launch_blocks(uint32_t tile_rows, uint32_t waves, const A &a, hipStream_t stream) {
  if (tile_rows == 16) return launch_one<FMT, DIM, 1>(waves, a, stream);
  if constexpr (attend_few_rows(DIM) >= 32)
    if (tile_rows == 32) return launch_one<FMT, DIM, 2>(waves, a, stream);
  return hipErrorInvalidValue;
}
template <uint32_t FMT, typename A>
hipError_t launch_dim(uint32_t tile_rows, uint32_t waves, const A &a, hipStream_t stream) {
  if (a.kv.head_dim <= 64) return launch_blocks<FMT, 64>(tile_rows, waves, a, stream);
  if (a.kv.head_dim <= 128) return launch_blocks<FMT, 128>(tile_rows, waves, a, stream);
  return launch_blocks<FMT, 256>(tile_rows, waves, a, stream);
}
template <typename A>
hipError_t launch_rows(uint32_t tile_rows, uint32_t waves, const A &a, hipStream_t stream) {
  if (a.kv.format == SQ_KV_BF16) return launch_dim<SQ_KV_BF16>(tile_rows, waves, a, stream);
  if (a.kv.format == SQ_KV_INT8) return launch_dim<SQ_KV_INT8>(tile_rows, waves, a, stream);
  if (a.kv.format == SQ_KV_E2M1) return launch_dim<SQ_KV_E2M1>(tile_rows, waves, a, stream);
  return launch_dim<SQ_KV_E4M3>(tile_rows, waves, a, stream);
}

}  // namespace
}  // namespace sq::kern
