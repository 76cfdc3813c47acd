// Rotary positions and the paged key/value cache: rows rotated, rows written into their pages in 16 or 8 bits, and read
// back. All three are bound by the bytes they move (a value in, a value out). A head row (head_dim values) is a group of
// 8, 16 or 32 lanes of 8 values, so that its largest magnitude is a few lane exchanges away and each lane's access is one
// 16-byte vector (8 bytes of codes). Of few rows each has a workgroup, of many a wave, four heads' loads in flight: a
// workgroup a row of a 30000-key int8 prefix reads back in 68 us, most of it launches, a wave a row in 45 us (4.1 of the
// 4.9 TB/s that a large copy reaches). Both are level at some 1500 rows without a rope and 3500 with one, whatever the
// format (written and read back, 8 heads of 128, us, workgroups / waves):
//   rows              256        1024       2048       3000       4096       8192        30000
//   int8              7.0/9.4    9.1/10.3   13.7/12.9  18.1/16.1  21.8/19.5  36.9/28.7   118/86
//   bf16              6.1/7.3    8.3/8.5    12.2/11.6  15.7/14.7  18.7/17.7  32.1/27.0   126/96
//   int8 with a rope  9.5/16.5   14.5/20.6  22.1/24.5  29.1/30.1  36.4/34.4  74.3/68.0   260/206
// One launch of a few rows takes 3 to 6 us, its loads' round trips.
//
// A rope on the way rounds the keys to bf16 before they are quantised, as sq_rope_add and a write of its output would: the
// cache then holds the same bits whichever way they came, a half step of bf16 (2^-8) against the codes' own (2^-8 of the
// row's largest for int8, 2^-4 of the value for e4m3).
//
// The angles: p f / 2 pi turns in fp64, the whole turns dropped there (p f reaches 10^6 radians, where fp32 has a 16th
// of a radian left), then sine and cosine of the fraction in fp32. A row's pairs are worked out once, by as many
// threads, and serve all of its heads from LDS.
#include "batch.hpp"
#include "device.hpp"

namespace sq::kern {
namespace {

constexpr uint32_t kMaxPairs = 128;   // head_dim is at most 256

struct CosSin {
  float c, s;
};

// The threads of a row: its workgroup's, or its wave's. t: this one's number among them.
template <int THREADS>
__device__ __forceinline__ void row_barrier() {
  if constexpr (THREADS == 256) {
    __syncthreads();
  } else {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
}
// The most rows that have a workgroup each (above).
constexpr uint32_t kFewRows = 2048;

// cs[i] of every pair for a position, by the row's threads.
template <int THREADS>
__device__ __forceinline__ void angles(CosSin *cs, const RopeArgs &rope, double position, uint32_t t) {
  for (uint32_t i = t; i < rope.pairs; i += THREADS) {
    const double turns = position * rope.frequencies[i] * 0.15915494309189533577;
    float s, c;
    sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
    cs[i] = {c * rope.magnitude, s * rope.magnitude};
  }
  row_barrier<THREADS>();
}

__device__ __forceinline__ void widen8(u32x4 w, float (&x)[8]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[2 * e] = bf16_to_f32(w[e] & 0xFFFFu);
    x[2 * e + 1] = bf16_to_f32(w[e] >> 16);
  }
}
__device__ __forceinline__ u32x4 narrow8(const float (&x)[8]) {
  u32x4 w;
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = (uint32_t)f32_to_bf16(x[2 * e]) | ((uint32_t)f32_to_bf16(x[2 * e + 1]) << 16);
  return w;
}

// Values d .. d + 7 of a head, rotated. In the half layout a value's partner lies pairs values away: another lane's,
// read here a second time (from the cache line the wave has just read). Every lane of a head reads before any of them
// writes (a head lies within one wave), so a head may be rotated in place.
__device__ __forceinline__ u32x4 rotated8(const uint16_t *head, uint32_t d, const CosSin *cs, const RopeArgs &rope) {
  const u32x4 own = *(const u32x4 *)(head + d);
  const uint32_t n = rope.pairs;
  if (d >= 2 * n) return own;
  float x[8], y[8];
  widen8(own, x);
  if (rope.interleaved) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      if (d + e < 2 * n) {
        const CosSin t = cs[(d + e) / 2];
        y[e] = x[e] * t.c - x[e + 1] * t.s;
        y[e + 1] = x[e + 1] * t.c + x[e] * t.s;
      } else {
        y[e] = x[e];
        y[e + 1] = x[e + 1];
      }
    }
  } else {
    float z[8];
    if (n % 8 == 0) {
      widen8(*(const u32x4 *)(head + (d < n ? d + n : d - n)), z);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t v = d + e;
        z[e] = v < 2 * n ? bf16_to_f32(head[v < n ? v + n : v - n]) : 0.0f;
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t v = d + e;
      const CosSin t = cs[v < n ? v : v < 2 * n ? v - n : 0];
      y[e] = v >= 2 * n ? x[e] : v < n ? x[e] * t.c - z[e] * t.s : x[e] * t.c + z[e] * t.s;
    }
  }
  return narrow8(y);
}

// LPH: the lanes of a head row, 8 values each (8, 16 or 32 of them hold head_dim).
template <int LPH>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs rope, const uint32_t *positions, uint32_t head_dim,
                                                   HeadRows input, HeadRows output) {
  __shared__ CosSin cs[kMaxPairs];
  const uint32_t row = blockIdx.x, d = 8 * (threadIdx.x % LPH);
  angles<256>(cs, rope, (double)positions[row], threadIdx.x);
  if (d >= head_dim) return;
  const uint16_t *in = input.rows + (size_t)row * input.stride;
  uint16_t *out = output.rows + (size_t)row * output.stride;
  for (uint32_t h = threadIdx.x / LPH; h < input.heads; h += 256 / LPH)
    *(u32x4 *)(out + h * head_dim + d) = rotated8(in + h * head_dim, d, cs, rope);
}

// A head row's eight values (of this lane; lanes past head_dim pass zeros) as codes, with the row's scale. The code is
// x top / m in fp32, rounded to the format: x top is exact (8 bits times 3 or 7), and the quotient of two such numbers
// lies on a tie of the format or further from it (2^-18 of it) than the fp32 quotient is off. That is q + r / m of a first
// quotient q = (x top) (1 / m), off by 2^-23, and its remainder r = x top - q m, which one fma gives exactly: off by 2^-46
// before its rounding, so a tie, which has few bits, comes out exact. The codes are those of the exact quotient, for three
// instructions a value where a division takes ten. Both sides go by 2^-30 in rows past 2^100, where x top would be
// infinite, and by 2^60 below 2^-60, where 1 / m and the remainder would leave the normal range.
struct Codes {
  u32x2 words;
  float scale;
};
template <uint32_t FMT, int LPH>
__device__ __forceinline__ Codes codes8(u32x4 w) {
  uint32_t largest = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) largest = max(largest, max(w[e] & 0x7FFFu, (w[e] >> 16) & 0x7FFFu));
#pragma unroll
  for (int m = LPH / 2; m; m >>= 1) largest = max(largest, (uint32_t)__shfl_xor((int)largest, m));
  if (largest >= 0x7F80u) return {{0u, 0u}, __uint_as_float(0x7FC00000u)};
  if (!largest) return {{0u, 0u}, 0.0f};
  constexpr float kTop = FMT == SQ_KV_INT8 ? 127.0f : 448.0f;
  const float m = bf16_to_f32(largest), shift = m > 0x1p100f ? 0x1p-30f : m < 0x1p-60f ? 0x1p60f : 1.0f;
  const float by = m * shift, over = 1.0f / by;
  float x[8], q[8];
  widen8(w, x);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float top = x[e] * (kTop * shift), first = top * over;
    q[e] = fmaf(fmaf(-first, by, top), over, first);
  }
  Codes out{{0u, 0u}, m / kTop};
  if constexpr (FMT == SQ_KV_INT8) {
#pragma unroll
    for (int e = 0; e < 8; ++e) out.words[e / 4] |= ((uint32_t)(int)rintf(q[e]) & 0xFFu) << (8 * (e % 4));
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      int v = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * i], q[4 * i + 1], 0, false);
      out.words[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[4 * i + 2], q[4 * i + 3], v, true);
    }
  }
  return out;
}

// Heads whose loads a thread has in flight.
constexpr int kAtOnce = 4;

template <uint32_t FMT, int LPH, int THREADS>
__global__ __launch_bounds__(256) void kv_write_kernel(KvArgs kv, HeadRows keys, HeadRows values, RopeArgs rope,
                                                       HeadRows queries, HeadRows rotated) {
  constexpr uint32_t kHeads = THREADS / LPH;   // head rows of the row's threads at a time
  __shared__ CosSin all[256 / THREADS][kMaxPairs];
  CosSin *cs = all[threadIdx.x / THREADS];
  const uint32_t t = threadIdx.x % THREADS, d = 8 * (t % LPH), dim = kv.head_dim;
  const uint32_t row = blockIdx.x * (256 / THREADS) + threadIdx.x / THREADS;
  if (row >= kv.rows) return;
  const bool live = d < dim;
  u32x4 w[kAtOnce];
  const auto load = [&](uint32_t first) {
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const uint32_t u = first + i * kHeads;
      const bool key = u < kv.kv_heads;
      const uint32_t h = key ? u : u - kv.kv_heads;
      const HeadRows &from = key ? keys : values;
      w[i] = u32x4{0u, 0u, 0u, 0u};
      if (!live || u >= 2 * kv.kv_heads) continue;
      const uint16_t *head = from.rows + (size_t)row * from.stride + h * dim;
      w[i] = key && rope.pairs ? rotated8(head, d, cs, rope) : *(const u32x4 *)(head + d);
    }
  };
  // Without a rope the first loads are on their way before the row's place is known.
  if (!rope.pairs) load(t / LPH);
  const RowPlace place = place_of(kv, row);
  if (place.sequence == ~0u) return;
  const uint32_t page = place.position >= 0 ? page_of(kv, place.sequence, place.position) : ~0u;
  const uint32_t slot = (uint32_t)place.position & ((1u << kv.page_shift) - 1);
  if (rope.pairs) angles<THREADS>(cs, rope, (double)place.position, t);
  for (uint32_t first = t / LPH; first < 2 * kv.kv_heads; first += kAtOnce * kHeads) {
    if (rope.pairs || first != t / LPH) load(first);
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const uint32_t u = first + i * kHeads;
      if (u >= 2 * kv.kv_heads) continue;
      const bool key = u < kv.kv_heads;
      const uint32_t h = key ? u : u - kv.kv_heads;
      const size_t at = ((((size_t)page * kv.kv_heads + h) << kv.page_shift) + slot);
      if constexpr (FMT == SQ_KV_BF16) {
        if (page != ~0u && live) *(u32x4 *)((key ? kv.keys : kv.values) + (at * dim + d) * 2) = w[i];
      } else {
        const Codes c = codes8<FMT, LPH>(w[i]);
        if (page == ~0u) continue;
        if (live) *(u32x2 *)((key ? kv.keys : kv.values) + at * dim + d) = c.words;
        if (d == 0) (key ? kv.key_scales : kv.value_scales)[at] = c.scale;
      }
    }
  }
  if (!queries.rows || !live) return;
  for (uint32_t h = t / LPH; h < queries.heads; h += kHeads)
    *(u32x4 *)(rotated.rows + (size_t)row * rotated.stride + h * dim + d) =
        rotated8(queries.rows + (size_t)row * queries.stride + h * dim, d, cs, rope);
}

template <uint32_t FMT, int LPH, int THREADS>
__global__ __launch_bounds__(256) void kv_read_kernel(KvArgs kv, HeadRows keys, HeadRows values) {
  constexpr uint32_t kHeads = THREADS / LPH;
  const uint32_t t = threadIdx.x % THREADS, d = 8 * (t % LPH), dim = kv.head_dim;
  const uint32_t row = blockIdx.x * (256 / THREADS) + threadIdx.x / THREADS;
  if (row >= kv.rows) return;
  const RowPlace place = place_of(kv, row);
  if (place.sequence == ~0u || d >= dim) return;
  const uint32_t page = place.position >= 0 ? page_of(kv, place.sequence, place.position) : ~0u;
  const uint32_t slot = (uint32_t)place.position & ((1u << kv.page_shift) - 1);
  for (uint32_t first = t / LPH; first < 2 * kv.kv_heads; first += kAtOnce * kHeads) {
    u32x4 w[kAtOnce];
    float scale[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const uint32_t u = first + i * kHeads;
      const bool key = u < kv.kv_heads;
      const uint32_t h = key ? u : u - kv.kv_heads;
      w[i] = u32x4{0u, 0u, 0u, 0u};
      scale[i] = 0.0f;
      if (u >= 2 * kv.kv_heads || page == ~0u || !(key ? keys : values).rows) continue;
      const size_t at = ((((size_t)page * kv.kv_heads + h) << kv.page_shift) + slot);
      const uint8_t *from = key ? kv.keys : kv.values;
      if constexpr (FMT == SQ_KV_BF16) {
        w[i] = *(const u32x4 *)(from + (at * dim + d) * 2);
      } else {
        const u32x2 c = *(const u32x2 *)(from + at * dim + d);
        w[i][0] = c[0];
        w[i][1] = c[1];
        scale[i] = (key ? kv.key_scales : kv.value_scales)[at];
      }
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const uint32_t u = first + i * kHeads;
      const bool key = u < kv.kv_heads;
      const uint32_t h = key ? u : u - kv.kv_heads;
      const HeadRows &to = key ? keys : values;
      if (u >= 2 * kv.kv_heads || !to.rows) continue;
      if constexpr (FMT != SQ_KV_BF16) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t c = w[i][j];
          if constexpr (FMT == SQ_KV_INT8) {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 * j + e] = (float)(int8_t)(c >> (8 * e)) * scale[i];
          } else {
            x[4 * j] = __builtin_amdgcn_cvt_f32_fp8((int)c, 0) * scale[i];
            x[4 * j + 1] = __builtin_amdgcn_cvt_f32_fp8((int)c, 1) * scale[i];
            x[4 * j + 2] = __builtin_amdgcn_cvt_f32_fp8((int)c, 2) * scale[i];
            x[4 * j + 3] = __builtin_amdgcn_cvt_f32_fp8((int)c, 3) * scale[i];
          }
        }
        w[i] = narrow8(x);
      }
      *(u32x4 *)(to.rows + (size_t)row * to.stride + h * dim + d) = w[i];
    }
  }
}

template <typename F>
void with_lanes(uint32_t head_dim, F &&f) {
  if (head_dim <= 64) f(std::integral_constant<int, 8>{});
  else if (head_dim <= 128) f(std::integral_constant<int, 16>{});
  else f(std::integral_constant<int, 32>{});
}
template <typename F>
void with_kv_format(uint32_t format, F &&f) {
  if (format == SQ_KV_BF16) f(std::integral_constant<uint32_t, SQ_KV_BF16>{});
  else if (format == SQ_KV_INT8) f(std::integral_constant<uint32_t, SQ_KV_INT8>{});
  else f(std::integral_constant<uint32_t, SQ_KV_E4M3>{});
}

}  // namespace

hipError_t launch_rope(const RopeArgs &rope, const uint32_t *positions, uint32_t rows, uint32_t head_dim,
                       const HeadRows &input, const HeadRows &output, hipStream_t stream) {
  with_lanes(head_dim, [&](auto lanes) {
    hipLaunchKernelGGL((rope_kernel<lanes.value>), dim3(rows), dim3(256), 0, stream, rope, positions, head_dim, input,
                       output);
  });
  return hipGetLastError();
}

hipError_t launch_kv_write(const KvArgs &kv, const HeadRows &keys, const HeadRows &values, const RopeArgs &rope,
                           const HeadRows &queries, const HeadRows &rotated, hipStream_t stream) {
  with_kv_format(kv.format, [&](auto format) {
    with_lanes(kv.head_dim, [&](auto lanes) {
      if (kv.rows <= kFewRows)
        hipLaunchKernelGGL((kv_write_kernel<format.value, lanes.value, 256>), dim3(kv.rows), dim3(256), 0, stream, kv,
                           keys, values, rope, queries, rotated);
      else
        hipLaunchKernelGGL((kv_write_kernel<format.value, lanes.value, 64>), dim3((kv.rows + 3) / 4), dim3(256), 0,
                           stream, kv, keys, values, rope, queries, rotated);
    });
  });
  return hipGetLastError();
}

hipError_t launch_kv_read(const KvArgs &kv, const HeadRows &keys, const HeadRows &values, hipStream_t stream) {
  with_kv_format(kv.format, [&](auto format) {
    with_lanes(kv.head_dim, [&](auto lanes) {
      if (kv.rows <= kFewRows)
        hipLaunchKernelGGL((kv_read_kernel<format.value, lanes.value, 256>), dim3(kv.rows), dim3(256), 0, stream, kv,
                           keys, values);
      else
        hipLaunchKernelGGL((kv_read_kernel<format.value, lanes.value, 64>), dim3((kv.rows + 3) / 4), dim3(256), 0,
                           stream, kv, keys, values);
    });
  });
  return hipGetLastError();
}

}  // namespace sq::kern
