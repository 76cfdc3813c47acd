// Attention of few rows a key head (tiles of 16, 32 or 64 rows times query heads): single tokens and verify lanes,
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
// Loads go through buffer resources of 16 keys of one page (pages are whole multiples of 16 tokens): a key past the
// sequence, a page that is a hole and a value past head_dim all read zero, with no instruction spent on them.
//
// Softmax: each wave keeps its own running maximum, lane sums and accumulators, and raises the maximum (which costs
// lane exchanges and a pass over the accumulators) only when a score exceeds it by 8 (a factor of 256, which fp32 sums
// and bf16's exponent hold without loss); the four waves of a workgroup join at the end of a part.
#include "attend.hpp"
#include "device.hpp"

namespace sq::kern {
namespace {

constexpr int kWaves = 4, kThreads = 64 * kWaves, kStep = 32;   // keys a wave takes a step
constexpr float kRaise = 8.0f;
constexpr uint32_t kNowhere = 0x7FFFFFF0u;   // past every resource's range: reads zero

// Two of a key's values for each of two keys, regrouped: two keys of each of two values.
__device__ __forceinline__ uint32_t low_halves(uint32_t k0, uint32_t k1) {
  return __builtin_amdgcn_perm(k1, k0, 0x05040100u);
}
__device__ __forceinline__ uint32_t high_halves(uint32_t k0, uint32_t k1) {
  return __builtin_amdgcn_perm(k1, k0, 0x07060302u);
}
typedef __attribute__((__vector_size__(2 * sizeof(__bf16)))) __bf16 bf16x2;
__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
  return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)a, (__bf16)b});
}
// Four codes as bf16, in their order.
template <uint32_t FMT>
__device__ __forceinline__ u32x2 code_pairs4(uint32_t w) {
  if constexpr (FMT == SQ_KV_E4M3) {
    return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true))};
  } else {
    uint32_t f[4];   // whole numbers of at most 8 bits: their fp32 words' high halves are their bf16
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = __float_as_uint((float)(int8_t)(w >> (8 * e)));
    return u32x2{high_halves(f[0], f[1]), high_halves(f[2], f[3])};
  }
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

// Sixteen keys of one page: where their values lie, and how many bytes of them there are to read.
struct Keys16 {
  const uint8_t *keys, *values;
  const float *key_scales, *value_scales;
  uint32_t bytes, scale_bytes;
};

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

  static __device__ __forceinline__ void load_keys(KeyTile &t, const Keys16 &k, int half, uint32_t row_bytes,
                                                   uint32_t lane) {
    const __amdgpu_buffer_rsrc_t r = buffer_rsrc(k.keys, k.bytes);
#pragma unroll
    for (int j = 0; j < kKeyLoads; ++j) {
      const uint32_t at = 64 * j + 16 * (lane >> 4);
      t.w[half][j] = buffer_b128(r, at < row_bytes ? (lane & 15) * row_bytes + at : kNowhere, 0);
    }
    if constexpr (kCodes)
      t.scale[half] = __builtin_bit_cast(f32x4, buffer_b128(buffer_rsrc(k.key_scales, k.scale_bytes), 16 * (lane >> 4), 0));
  }
  static __device__ __forceinline__ void load_values(ValueTile &t, const Keys16 &k, int half, uint32_t row_bytes,
                                                     uint32_t lane) {
    const __amdgpu_buffer_rsrc_t r = buffer_rsrc(k.values, k.bytes);
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
          __builtin_bit_cast(f32x4, buffer_b128(buffer_rsrc(k.value_scales, k.scale_bytes), 16 * (lane >> 4), 0));
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

  // Adds the weights' product with 32 keys' values. Two values of a run at a time.
  __device__ __forceinline__ void accumulate(const ValueTile &t, const u32x4 (&p)[MB]) {
#pragma unroll
    for (int j = 0; j < kRun / 2; ++j) {
      uint32_t w[2][4];   // values 2 j and 2 j + 1 of each key as bf16
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (!kCodes) w[h][e] = t.w[h][e][j];
          else w[h][e] = code_pairs4<FMT>(t.w[h][e][j / 2])[j % 2];
        }
      const u32x4 even{low_halves(w[0][0], w[0][1]), low_halves(w[0][2], w[0][3]), low_halves(w[1][0], w[1][1]),
                       low_halves(w[1][2], w[1][3])};
      const u32x4 odd{high_halves(w[0][0], w[0][1]), high_halves(w[0][2], w[0][3]), high_halves(w[1][0], w[1][1]),
                      high_halves(w[1][2], w[1][3])};
#pragma unroll
      for (int b = 0; b < MB; ++b) {
        o[b][2 * j] = mfma_bf16(even, p[b], o[b][2 * j]);
        o[b][2 * j + 1] = mfma_bf16(odd, p[b], o[b][2 * j + 1]);
      }
    }
  }
};

// Whether any value of a bf16 tile is an infinity or NaN.
template <int N>
__device__ __forceinline__ bool unbounded(const uint32_t (&w)[2][4][N]) {
  uint32_t any = 0;
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int i = 0; i < N; ++i)
        any |= (uint32_t)((w[h][e][i] & 0x7F80u) == 0x7F80u) | (uint32_t)((w[h][e][i] & 0x7F800000u) == 0x7F800000u);
  return any != 0;
}

template <uint32_t FMT, int DIM, int MB>
__global__ __launch_bounds__(kThreads, DIM * MB <= (DIM == 256 ? 0 : FMT == SQ_KV_BF16 ? 128 : 256) ? 2 : 1) void attend_rows_kernel(AttendArgs a) {
  using R = Rows<FMT, DIM, MB>;
  constexpr bool kCodes = R::kCodes;
  constexpr int kRun = R::kRun, kRegs = 4 * kRun, kChunk = 8, kChunks = kRegs / kChunk;
  // A part in the workspace: its accumulators in the waves' register order, then its rows' maxima and sums.
  constexpr int kPartFloats = MB * (kRegs * 64 + 32);
  __shared__ int64_t prefix[kMaxSequences + 1], scan[kWaves];
  __shared__ float joined[kWaves][kChunk][64], maxima[kWaves][MB][16], sums[kWaves][MB][16];
  __shared__ uint32_t arrival;
  const uint32_t lane = threadIdx.x & 63, r = lane & 15, kq = lane >> 4;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int fit = 16 * MB / (int)a.group;
  const uint32_t dim = a.kv.head_dim, row_bytes = dim * R::kBytes;
  const Line line = make_line<kThreads>(a, fit, 2 * kWaves * kStep, prefix, scan);
  const uint32_t piece = piece_of(line, blockIdx.x);
  if (blockIdx.x / 8 >= (line.active + 7) / 8 || piece >= line.active) return;
  int64_t x = line.share * piece;
  const int64_t end = x + line.share < line.total ? x + line.share : line.total;

  while (x < end) {
    const Part part = next_part(a, line, fit, x, end, piece);
    if (part.t1 <= part.t0) continue;
    const Units &u = part.units;
    const int row0 = fit * part.m, rows = min(fit, u.rows - row0), live = rows * (int)a.group;
    const int unit_end = u.causal ? min(u.keys, u.base + row0 + rows) : u.keys;   // keys that any row sees
    const int tile0 = u.first_tile(part.m);
    const int k_begin = kKeyTile * (tile0 + part.t0), k_end = min(unit_end, kKeyTile * (tile0 + part.t1));
    // Keys [clear_begin, clear_end) are seen by every row of the unit.
    const int clear_begin = u.window ? u.base + row0 + rows - u.window : 0;
    const int clear_end = u.causal ? u.base + row0 + 1 : u.keys;

    R state;
    state.clear();
    int low[MB], high[MB];   // the keys this lane's rows see
#pragma unroll
    for (int b = 0; b < MB; ++b) {
      const int p = 16 * b + (int)r, i = p / (int)a.group, g = p - i * (int)a.group;
      const int at = u.base + row0 + i;
      low[b] = u.window ? at - u.window + 1 : 0;
      high[b] = u.causal ? min(at + 1, u.keys) : u.keys;
      const bool on = p < live;
      const uint16_t *row = a.query + (size_t)(part.first_row + row0 + (on ? i : 0)) * a.query_stride +
                            (part.head * a.group + (on ? g : 0)) * dim;
#pragma unroll
      for (int c = 0; c < R::kChains; ++c) {
        const uint32_t d = R::query_at(c, lane);
        state.q[b][c] = on && d < dim ? *(const u32x4 *)(row + d) : u32x4{0u, 0u, 0u, 0u};
      }
    }

    // The 16 keys from k on: none if they lie past the unit's keys or in a hole.
    const auto keys_at = [&](int k) __attribute__((always_inline)) {
      const int n = min(16, k_end - k);
      const uint32_t page =
          n > 0 ? (uint32_t)__builtin_amdgcn_readfirstlane((int)page_of(a.kv, part.sequence, k)) : ~0u;
      const bool there = page != ~0u;
      const size_t at = (((size_t)(there ? page : 0) * a.kv.kv_heads + part.head) << a.kv.page_shift) +
                        ((uint32_t)k & ((1u << a.kv.page_shift) - 1));
      return Keys16{a.kv.keys + at * row_bytes, a.kv.values + at * row_bytes, a.kv.key_scales + at,
                    a.kv.value_scales + at, there ? (uint32_t)n * row_bytes : 0u, there ? 64u : 0u};
    };

    typename R::KeyTile kt;
    typename R::ValueTile vt;
    int k = k_begin + kStep * (int)wave;
    const auto fetch_keys = [&](const Keys16 &ka, const Keys16 &kb) __attribute__((always_inline)) {
      R::load_keys(kt, ka, 0, row_bytes, lane);
      R::load_keys(kt, kb, 1, row_bytes, lane);
    };
    const auto fetch_values = [&](const Keys16 &ka, const Keys16 &kb) __attribute__((always_inline)) {
      R::load_values(vt, ka, 0, row_bytes, lane);
      R::load_values(vt, kb, 1, row_bytes, lane);
    };
    Keys16 ka = keys_at(k), kb = keys_at(k + 16);
    fetch_keys(ka, kb);
    fetch_values(ka, kb);
    for (; k < k_end; k += kStep * kWaves) {
      const uint32_t hole = (ka.bytes ? 0u : 1u) | (kb.bytes ? 0u : 2u);
      const Keys16 na = keys_at(k + kStep * kWaves), nb = keys_at(k + kStep * kWaves + 16);
      f32x4 s[MB][2];
      state.scores(kt, s);
      f32x4 key_scale[2], value_scale[2];
      if constexpr (kCodes) {
        key_scale[0] = kt.scale[0] * a.scale;
        key_scale[1] = kt.scale[1] * a.scale;
        value_scale[0] = vt.scale[0];
        value_scale[1] = vt.scale[1];
      }
      fetch_keys(na, nb);

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
      u32x4 p[MB];
#pragma unroll
      for (int b = 0; b < MB; ++b) {
        float v[8], top = -INFINITY;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float t = kCodes ? s[b][h][i] * key_scale[h][i] : s[b][h][i] * a.scale;
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
        p[b] = u32x4{bf16_pair(w[0], w[1]), bf16_pair(w[2], w[3]), bf16_pair(w[4], w[5]), bf16_pair(w[6], w[7])};
      }
      if constexpr (!kCodes) {
        // Where some rows see a key and others do not, its values must not reach the others through 0 * inf: infinities
        // and NaNs leave the tile, and the rows that see them add their products one by one.
        if (!clear && __any(unbounded(vt.w))) {
#pragma unroll
          for (int b = 0; b < MB; ++b)
            for (int key = 0; key < kStep; ++key) {
              const int h = key / 16, i = key % 4, source = 16 * (key % 16 / 4) + (int)r;
              // By selects: an index known only at run time would put the weights in scratch memory.
              const uint32_t first = h ? p[b][2] : p[b][0], second = h ? p[b][3] : p[b][1];
              const uint32_t word = i / 2 ? second : first;
              const float weight = __uint_as_float((uint32_t)__shfl((int)(i % 2 ? word & 0xFFFF0000u : word << 16), source));
              const bool sees = (__shfl((int)seen[b], source) >> (4 * h + i)) & 1;
              const __amdgpu_buffer_rsrc_t values = buffer_rsrc(h ? kb.values : ka.values, h ? kb.bytes : ka.bytes);
#pragma unroll
              for (int d = 0; d < kRun; ++d)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  const uint32_t at = kRun * (4 * kq + j) + d;
                  const uint32_t bits = at < dim ? __builtin_amdgcn_raw_buffer_load_b16(
                                                       values, (key % 16) * row_bytes + 2 * at, 0, 0)
                                                 : 0u;
                  if (sees && (bits & 0x7F80u) == 0x7F80u) state.o[b][d][j] += weight * bf16_to_f32(bits);
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
      state.accumulate(vt, p);
      fetch_values(na, nb);
      ka = na;
      kb = nb;
    }
#pragma unroll
    for (int b = 0; b < MB; ++b) state.l[b] = row_sum(state.l[b]);

    // Joins the waves' states, eight accumulators at a time, into finish(b, chunk, factor, pair): wave w holds sums of
    // accumulators 8 chunk + 2 w and + 1 (accumulator kRun j + d: value d of run j). total_l and top as the lane's row's.
    const auto join = [&](auto &&finish, float (&top)[MB], float (&total)[MB]) __attribute__((always_inline)) {
      __syncthreads();
      if (lane < 16) {
#pragma unroll
        for (int b = 0; b < MB; ++b) {
          maxima[wave][b][lane] = state.m[b];
          sums[wave][b][lane] = state.l[b];
        }
      }
      __syncthreads();
      float mine[MB];
#pragma unroll
      for (int b = 0; b < MB; ++b) {
        top[b] = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) top[b] = fmaxf(top[b], maxima[w][b][r]);
        total[b] = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
          // A wave that saw nothing adds nothing, even to a row whose maximum is infinite.
          const float s = sums[w][b][r];
          if (s != 0.0f) total[b] += s * exp2_fast(maxima[w][b][r] - finite_max(top[b]));
        }
        mine[b] = state.l[b] != 0.0f ? exp2_fast(state.m[b] - finite_max(top[b])) : 0.0f;
      }
#pragma unroll
      for (int b = 0; b < MB; ++b)
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          if (b || c) __syncthreads();
#pragma unroll
          for (int t = 0; t < kChunk; ++t) {
            const int acc = kChunk * c + t;
            joined[wave][t][lane] = state.o[b][acc % kRun][acc / kRun] * mine[b];
          }
          __syncthreads();
          float sum[2] = {0.0f, 0.0f};
#pragma unroll
          for (int w = 0; w < kWaves; ++w) {
            sum[0] += joined[w][2 * wave][lane];
            sum[1] += joined[w][2 * wave + 1][lane];
          }
          finish(b, c, sum);
        }
    };
    const auto write = [&](const float (&total)[MB]) __attribute__((always_inline)) {
      return [&](int b, int c, const float (&sum)[2]) __attribute__((always_inline)) {
        const int p = 16 * b + (int)r, i = p / (int)a.group, g = p - i * (int)a.group;
        const uint32_t acc = kChunk * c + 2 * wave, value = kRun * (4 * kq + acc / kRun) + acc % kRun;
        if (p >= live || value >= dim) return;
        const float by = total[b] == 0.0f ? 0.0f : 1.0f / total[b];
        uint16_t *out = a.output + (size_t)(part.first_row + row0 + i) * a.output_stride +
                        (part.head * a.group + g) * dim + value;
        *(uint32_t *)out = bf16_pair(sum[0] * by, sum[1] * by);
      };
    };

    float top[MB], total[MB];
    if (part.parts == 1) {
      join(write(total), top, total);
      continue;
    }
    float *mine = a.partials + (size_t)part_slot(part.first_piece, part.part) * kPartFloats;
    join([&](int b, int c, const float (&sum)[2])
             __attribute__((always_inline)) {
               store_pair(mine + ((b * kChunks + c) * kWaves + wave) * 128 + 2 * lane, sum[0], sum[1]);
             },
         top, total);
    if (wave == 0 && lane < 16) {
#pragma unroll
      for (int b = 0; b < MB; ++b)
        store_pair(mine + MB * kRegs * 64 + 32 * b + 2 * lane, top[b], total[b]);
    }
    if (!last_part(a.counters + part.first_piece, part.parts, &arrival)) continue;
    // The last to arrive: each wave joins every fourth part into a state of its own, in key order, and the waves join as
    // above.
    state.clear();
    for (uint32_t j = wave; j < part.parts; j += kWaves) {
      const float *from = a.partials + (size_t)part_slot(part.first_piece, j) * kPartFloats;
#pragma unroll
      for (int b = 0; b < MB; ++b) {
        float m, l, v[kRegs];
        load_pair(from + MB * kRegs * 64 + 32 * b + 2 * r, m, l);
#pragma unroll
        for (int t = 0; t < kRegs / 2; ++t) load_pair(from + (b * (kRegs / 2) + t) * 128 + 2 * lane, v[2 * t], v[2 * t + 1]);
        if (l == 0.0f) m = -INFINITY;
        const float next = fmaxf(state.m[b], m);
        const float keep = state.l[b] != 0.0f ? exp2_fast(state.m[b] - finite_max(next)) : 0.0f;
        const float take = l != 0.0f ? exp2_fast(m - finite_max(next)) : 0.0f;
        state.m[b] = next;
        state.l[b] = state.l[b] * keep + l * take;
#pragma unroll
        for (int t = 0; t < kRegs; ++t) {
          const float acc = state.o[b][t % kRun][t / kRun];
          state.o[b][t % kRun][t / kRun] = acc * keep + v[t] * take;
        }
      }
    }
    join(write(total), top, total);
  }
}

template <uint32_t FMT, int DIM>
hipError_t launch_blocks(uint32_t tile_rows, const AttendArgs &a, hipStream_t stream) {
  const dim3 grid(a.workgroups), block(kThreads);
  if (tile_rows == 16) hipLaunchKernelGGL((attend_rows_kernel<FMT, DIM, 1>), grid, block, 0, stream, a);
  else if (tile_rows == 32) hipLaunchKernelGGL((attend_rows_kernel<FMT, DIM, 2>), grid, block, 0, stream, a);
  else if constexpr (DIM <= 128) hipLaunchKernelGGL((attend_rows_kernel<FMT, DIM, 4>), grid, block, 0, stream, a);
  return hipGetLastError();
}
template <uint32_t FMT>
hipError_t launch_dim(uint32_t tile_rows, const AttendArgs &a, hipStream_t stream) {
  if (a.kv.head_dim <= 64) return launch_blocks<FMT, 64>(tile_rows, a, stream);
  if (a.kv.head_dim <= 128) return launch_blocks<FMT, 128>(tile_rows, a, stream);
  return launch_blocks<FMT, 256>(tile_rows, a, stream);
}

}  // namespace

uint64_t attend_partials(uint32_t tile_rows, uint32_t head_dim, uint32_t workgroups) {
  // Two parts a workgroup (attend.hpp), each a tile's accumulators and its rows' maxima and sums.
  const uint64_t dim = head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256;
  return 2 * uint64_t{workgroups} * tile_rows * (dim + 2);
}
uint64_t attend_counters(uint32_t workgroups) { return workgroups; }

hipError_t launch_attend_rows(uint32_t tile_rows, const AttendArgs &a, hipStream_t stream) {
  if (a.kv.format == SQ_KV_BF16) return launch_dim<SQ_KV_BF16>(tile_rows, a, stream);
  if (a.kv.format == SQ_KV_INT8) return launch_dim<SQ_KV_INT8>(tile_rows, a, stream);
  return launch_dim<SQ_KV_E4M3>(tile_rows, a, stream);
}

}  // namespace sq::kern
