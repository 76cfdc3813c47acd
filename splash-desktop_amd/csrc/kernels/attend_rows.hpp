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
// Heads of 256 of e4m3 spill 2 or 6 registers (12 or 28 bytes a lane; scored ones 8 or 14, 36 or 60), scored 8-bit heads of 64
// in tiles of 32 rows 4 or 5 (20 or 24), no others any.
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
#include <type_traits>

#include "attend_few.hpp"
#include "attend_rows_four.hpp"

namespace sq::kern {
namespace {

// Four e4m3 codes, NaNs as zeros.
__device__ __forceinline__ uint32_t finite_codes(uint32_t w) {
  const uint32_t nan = nan_codes(w);
  return w & ~(nan | (nan - (nan >> 7)));
}
// DIM: the head's values as computed (64, 128 or 256; values past head_dim are zero). MB: blocks of 16 rows.
template <uint32_t FMT, int DIM, int MB>
struct Rows {
  static constexpr bool kCodes = FMT != SQ_KV_BF16;
  static constexpr int kBytes = kCodes ? 1 : 2, kRun = DIM / 16, kChains = DIM / 32;
  // Vectors a lane loads for its share of 16 keys: K 16 bytes each, V kRun values a key.
  static constexpr int kKeyLoads = DIM * kBytes / 64, kValueWords = kRun * kBytes / 4;

  struct KeyTile {
    u32x4 w[2][kKeyLoads];
    f32x4 scale[2];
  };
  struct ValueTile {
    uint32_t w[2][4][kValueWords];
    f32x4 scale[2];
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
#pragma unroll
    for (int j = 0; j < kKeyLoads; ++j) {
      const uint32_t at = 64 * j + 16 * (lane >> 4);
      t.w[half][j] = buffer_b128(r, at < row_bytes ? (lane & 15) * row_bytes + at : kNowhere, 0);
    }
    if constexpr (kCodes)
      t.scale[half] = __builtin_bit_cast(f32x4, buffer_b128(buffer_rsrc(kv.key_scales + k.at, k.count ? 64 : 0), 16 * (lane >> 4), 0));
  }
  static __device__ __forceinline__ void load_values(ValueTile &t, const KvArgs &kv, const Keys16 &k, int half,
                                                     uint32_t row_bytes, uint32_t lane) {
    const __amdgpu_buffer_rsrc_t r = buffer_rsrc(kv.values + k.at * row_bytes, k.count * row_bytes);
    const uint32_t at = (lane & 15) * kRun * kBytes;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t from = at < row_bytes ? (4 * (lane >> 4) + e) * row_bytes + at : kNowhere;
      if constexpr (kValueWords == 1) {
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
    if constexpr (kCodes)
      t.scale[half] =
          __builtin_bit_cast(f32x4, buffer_b128(buffer_rsrc(kv.value_scales + k.at, k.count ? 64 : 0), 16 * (lane >> 4), 0));
  }

  // The rows' values in the K operand's order: bf16 chain j takes values 32 j + 8 kq + e; of codes, whose 16-byte vector
  // holds 16 values, chains 2 j and 2 j + 1 take values 64 j + 16 kq + e and + 8 + e.
  static __device__ __forceinline__ uint32_t query_at(int chain, uint32_t lane) {
    return kCodes ? 64 * (chain / 2) + 16 * (lane >> 4) + 8 * (chain % 2) : 32 * chain + 8 * (lane >> 4);
  }

  static __device__ __forceinline__ u32x4 key_operand(const KeyTile &t, int half, int chain) {
    if constexpr (!kCodes) {
      return t.w[half][chain];
    } else {
      const u32x4 w = t.w[half][chain / 2];
      const u32x2 a = code_pairs4<FMT>(w[2 * (chain % 2)]), b = code_pairs4<FMT>(w[2 * (chain % 2) + 1]);
      return u32x4{a[0], a[1], b[0], b[1]};
    }
  }

  // s = the raw products of 32 keys for block b's rows: half h's value i is key 16 h + 4 kq + i.
  __device__ __forceinline__ void scores(const KeyTile &t, f32x4 (&s)[MB][2]) const {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int b = 0; b < MB; ++b) s[b][h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < kChains; ++c) {
        const u32x4 k = key_operand(t, h, c);
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
  __device__ __forceinline__ void accumulate(const ValueTile &t, const u32x4 (&p)[MB], const u32x4 (&rest)[MB]) {
#pragma unroll
    for (int j = 0; j < kRun / 2; ++j) {
      uint32_t w[2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (!kCodes) w[h][e] = t.w[h][e][j];
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
  constexpr bool kFour = FMT == SQ_KV_E2M1;
  using R = std::conditional_t<kFour, Rows4<DIM, MB>, Rows<FMT, DIM, MB>>;
  constexpr int kWaves = WAVES, kThreads = 64 * WAVES, kJoin = 4 * WAVES;
  constexpr bool kCodes = FMT == SQ_KV_INT8 || FMT == SQ_KV_E4M3;
  // Accumulator t = kRun j + d of a block is value d of run j.
  constexpr int kRun = R::kRun, kRegs = 4 * kRun, kChunks = (kRegs + kJoin - 1) / kJoin;
  constexpr int kVectors = kRegs < kJoin ? kRegs / 4 : kJoin / 4;   // of four accumulators, in a chunk
  constexpr int kBlockFloats = 16 * (DIM + 2);   // of a part in the workspace
  __shared__ Shared<MB, WAVES, A> shared;
  const uint32_t lane = threadIdx.x & 63, r = lane & 15, kq = lane >> 4;
  const uint32_t wave = uniform(threadIdx.x >> 6);
  constexpr bool kWhole = kScored || kFour;   // (the others keep the shares, and so the bits, that they have)
  const Cut cut{16 * MB / (int)a.group, (int)attend_least(DIM, FMT, kScored), kUnitSlack + 256,
                attend_resident(16 * MB, WAVES, DIM, FMT), 640, 0};
  const float by_group = 1.0f / (float)a.group;
  const uint32_t dim = a.kv.head_dim, row_bytes = kFour ? dim / 2 : dim * (kCodes ? 1 : 2);
  Part<A> next;
  Work<kThreads, A, kWhole> work = make_work<kThreads, kWhole>(a, cut, shared.line, next);
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

    if constexpr (kFour) {
      run_four<kWaves>(a, part, state, KeySpan{k_begin, k_end, clear_begin, clear_end}, low, high, slope, position, wave, lane);
    } else {
      // The page of the 16 keys from k on as the table has it (~0u past the part's keys), and their place: none in a hole.
      const auto page_at = [&](int k) __attribute__((always_inline)) {
        return k < k_end ? a.kv.page_table[(size_t)part.sequence * a.kv.pages_per_sequence +
                                           ((uint32_t)k >> a.kv.page_shift)]
                         : ~0u;
      };
      const auto keys_at = [&](int k, uint32_t entry) __attribute__((always_inline)) {
        const uint32_t page = uniform(entry);
        if (page >= a.kv.pages) return Keys16{0, 0u};
        return Keys16{(((size_t)page * a.kv.kv_heads + part.head) << a.kv.page_shift) +
                          ((uint32_t)k & ((1u << a.kv.page_shift) - 1)),
                      (uint32_t)min(16, k_end - k)};
      };

      typename R::KeyTile kt;
      typename R::ValueTile vt;
      int k = k_begin + kStep * (int)wave;
      const auto fetch_keys = [&](const Keys16 &ka, const Keys16 &kb) __attribute__((always_inline)) {
        R::load_keys(kt, a.kv, ka, 0, row_bytes, lane);
        R::load_keys(kt, a.kv, kb, 1, row_bytes, lane);
      };
      const auto fetch_values = [&](const Keys16 &ka, const Keys16 &kb) __attribute__((always_inline)) {
        R::load_values(vt, a.kv, ka, 0, row_bytes, lane);
        R::load_values(vt, a.kv, kb, 1, row_bytes, lane);
      };
      // Fetches run a step ahead of the products, and the page table's entries a step ahead of the fetches.
      constexpr int kStride = kStep * kWaves;
      uint32_t entry_a = page_at(k), entry_b = page_at(k + 16);
      Keys16 ka = keys_at(k, entry_a), kb = keys_at(k + 16, entry_b);
      entry_a = page_at(k + kStride);
      entry_b = page_at(k + kStride + 16);
      if (k < k_end) {
        fetch_keys(ka, kb);
        fetch_values(ka, kb);
      }
      for (; k < k_end; k += kStride) {
        const bool more = k + kStride < k_end;
        const uint32_t hole = (ka.count ? 0u : 1u) | (kb.count ? 0u : 2u);
        const Keys16 na = keys_at(k + kStride, entry_a), nb = keys_at(k + kStride + 16, entry_b);
        entry_a = page_at(k + 2 * kStride);
        entry_b = page_at(k + 2 * kStride + 16);
        f32x4 s[MB][2];
        state.scores(kt, s);
        f32x4 key_scale[2], value_scale[2];
        if constexpr (kCodes) {
          key_scale[0] = kt.scale[0] * a.scale;
          key_scale[1] = kt.scale[1] * a.scale;
          value_scale[0] = vt.scale[0];
          value_scale[1] = vt.scale[1];
        }
        if (more) fetch_keys(na, nb);

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
              s[b][i / 4][i % 4] = kCodes ? t * key_scale[i / 4][i % 4] : t * a.scale;
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
                              : kCodes ? s[b][h][i] * key_scale[h][i]
                                        : s[b][h][i] * a.scale;
              v[4 * h + i] = clear || (seen[b] >> (4 * h + i) & 1) ? t : -INFINITY;
              top = fmaxf(top, v[4 * h + i]);
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
          if constexpr (kCodes) {
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
        if constexpr (!kCodes) {
          // Where some rows see a key and others do not, its values must not reach the others through 0 * inf: infinities
          // and NaNs leave the tile, and the rows that see them add their products one by one.
          if (!clear && __any(unbounded<FMT>(vt.w))) {
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
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                  for (int d = 0; d < kRun; d += 2) {
                    const uint32_t at = kRun * (4 * kq + j) + d;
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
                  if ((word & 0x7F80u) == 0x7F80u) word &= 0xFFFF0000u;
                  if ((word & 0x7F800000u) == 0x7F800000u) word &= 0x0000FFFFu;
                }
          }
        }
        if constexpr (FMT == SQ_KV_E4M3) {
          // The same of NaN codes. (No write makes one, but pages may hold them that have not been written yet, or by another.)
          if (!clear && __any(unbounded<FMT>(vt.w))) state.take_nans(vt, seen);
        }
        state.accumulate(vt, p, rest);
        if (more) fetch_values(na, nb);
        ka = na;
        kb = nb;
      }
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
