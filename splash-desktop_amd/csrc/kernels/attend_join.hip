// The join of units whose keys several workgroups shared: output = sum_j e^(m_j - m) O_j / sum_j e^(m_j - m) l_j over a
// unit's parts in key order, m their largest maximum. A launch of its own after the attention's: a workgroup of that one
// would find out that it is the last of its unit's only after its stores and an atomic have gone past the XCDs' caches
// (3 us a part), and then join all of the unit's rows alone (one token over 131072 int8 keys, 31 parts a unit: 8 us in
// all), where here the vectors of every unit go over all waves, with many parts' loads in flight: 5.5 us.
#include "attend.hpp"

namespace sq::kern {
namespace {

// Parts of a unit joined: for a lane's row the maximum and sum over them, and VECTORS of its vectors (attend.hpp: the
// layout of a part).
template <int VECTORS>
struct Joined {
  float m = -INFINITY, l = 0.0f;
  f32x4 sum[VECTORS] = {};

  // N more, whose loads were in flight together.
  template <int N>
  __device__ __forceinline__ void add(const float (&pm)[N], const float (&pl)[N], const f32x4 (&got)[N][VECTORS]) {
    float next = m;
#pragma unroll
    for (int d = 0; d < N; ++d) next = pl[d] == 0.0f ? next : fmaxf(next, pm[d]);
    // A part that saw nothing adds nothing, even to a row whose maximum is infinite.
    const float keep = l == 0.0f ? 0.0f : exp2_fast(m - finite_max(next));
    m = next;
    l *= keep;
#pragma unroll
    for (int v = 0; v < VECTORS; ++v) sum[v] *= keep;
#pragma unroll
    for (int d = 0; d < N; ++d) {
      const float by = pl[d] == 0.0f ? 0.0f : exp2_fast(pm[d] - finite_max(next));
      l += pl[d] * by;
#pragma unroll
      for (int v = 0; v < VECTORS; ++v) sum[v] += got[d][v] * by;
    }
  }
};

template <bool WIDE>
__device__ __forceinline__ bool has_row(const UnitNote &note, uint32_t block) {
  constexpr uint32_t kRows = WIDE ? 32 : 16;
  return block * kRows + (threadIdx.x & 63) % kRows < note.live;
}

// Of a block's vectors first .. first + VECTORS - 1, the parts begin .. begin + AT_ONCE - 1 of every `step`.
template <bool WIDE, int VECTORS, int AT_ONCE>
__device__ __forceinline__ Joined<VECTORS> gather(const AttendArgs &a, const UnitNote &note, uint32_t piece, uint32_t dim,
                                                  uint32_t block, uint32_t first, uint32_t begin, uint32_t step) {
  const uint32_t rows = WIDE ? 32 : 16, lane = threadIdx.x & 63, block_floats = rows * (dim + 2);
  const bool on = has_row<WIDE>(note, block);
  Joined<VECTORS> out;
  for (uint32_t j = begin; j < note.parts; j += step) {
    float pm[AT_ONCE], pl[AT_ONCE];
    f32x4 got[AT_ONCE][VECTORS];
#pragma unroll
    for (int d = 0; d < AT_ONCE; ++d) {
      // Past the last part the resource is empty: zeros, and nothing read.
      const bool there = j + d < note.parts;
      const float *from = a.partials + part_block(a, piece, there ? j + d : 0, block) * block_floats;
      const __amdgpu_buffer_rsrc_t r = buffer_rsrc(from, there ? block_floats * 4 : 0);
      const u32x2 two = buffer_b64<0>(r, on ? (rows * dim + 2 * (lane % rows)) * 4 : kNowhere, 0);
      pm[d] = __uint_as_float(two[0]);
      pl[d] = __uint_as_float(two[1]);
#pragma unroll
      for (int v = 0; v < VECTORS; ++v)
        got[d][v] = __builtin_bit_cast(f32x4, buffer_b128<0>(r, on ? ((first + v) * 64 + lane) * 16 : kNowhere, 0));
    }
    out.add(pm, pl, got);
  }
  return out;
}

template <bool WIDE, int VECTORS>
__device__ __forceinline__ void write(const AttendArgs &a, const UnitNote &note, uint32_t dim, uint32_t block,
                                      uint32_t first, const Joined<VECTORS> &all) {
  if (!has_row<WIDE>(note, block)) return;
  const uint32_t rows = WIDE ? 32 : 16, lane = threadIdx.x & 63, p = block * rows + lane % rows;
  const float by = all.l == 0.0f ? 0.0f : 1.0f / all.l;
  const uint32_t i = (uint32_t)row_of((int)p, 1.0f / (float)a.group), g = p - i * a.group;
  uint16_t *out = a.output + (size_t)(note.row + i) * a.output_stride + (note.head * a.group + g) * a.kv.head_dim;
#pragma unroll
  for (int v = 0; v < VECTORS; ++v) {
    const uint32_t value = WIDE ? wide_value(first + v, lane) : few_value(first + v, lane, dim / 16);
    const f32x4 sum = all.sum[v] * by;
    if (value < a.kv.head_dim) *(u32x2 *)(out + value) = u32x2{bf16_pair(sum[0], sum[1]), bf16_pair(sum[2], sum[3])};
  }
}

// The unit's items: VECTORS vectors of a block each.
template <bool WIDE>
__device__ __forceinline__ uint32_t items_of(const UnitNote &note, uint32_t each, uint32_t tile_rows) {
  constexpr uint32_t kRows = WIDE ? 32 : 16;
  return min(tile_rows / kRows, (note.live + kRows - 1) / kRows) * each;
}

// Many units: a workgroup a piece, for the shared unit that it began if any, each wave items of its own. Units of a line
// mostly have two parts, which go eight vectors at a time (rows of the wide tile have as many).
template <bool WIDE, int VECTORS, int AT_ONCE>
__device__ __forceinline__ void join_unit(const AttendArgs &a, const UnitNote &note, uint32_t dim, uint32_t tile_rows) {
  const uint32_t each = dim / (WIDE ? 8 : 16) / VECTORS, items = items_of<WIDE>(note, each, tile_rows);
  for (uint32_t i = uniform(threadIdx.x >> 6); i < items; i += 4) {
    const uint32_t block = i / each, first = VECTORS * (i % each);
    write<WIDE>(a, note, dim, block, first,
                gather<WIDE, VECTORS, AT_ONCE>(a, note, blockIdx.x, dim, block, first, 0, AT_ONCE));
  }
}
template <bool WIDE>
__global__ __launch_bounds__(256) void join_many_kernel(AttendArgs a, uint32_t dim, uint32_t tile_rows) {
  const UnitNote *notes = unit_notes(a);
  const uint32_t pieces = notes[a.workgroups].parts;
  const UnitNote note = notes[blockIdx.x];   // read beside the number of pieces, of which it may be past
  if (blockIdx.x >= pieces || note.parts < 2) return;
  if (WIDE && note.parts == 2) join_unit<WIDE, 8, 2>(a, note, dim, tile_rows);
  else join_unit<WIDE, 2, 16>(a, note, dim, tile_rows);
}

// Few units, of many parts each: every wave looks through the notes, one a lane, and the workgroups take the units'
// blocks and vectors in turn, each wave a quarter of the parts: 8 verify rows over up to 20000 keys of 2 heads of 256,
// 60 parts a unit, join in 9 us, where a wave for a vector's every part, 32 at a time, takes 13.
constexpr uint32_t kFewGroups = 256, kFewAtOnce = 16;
template <bool WIDE>
__global__ __launch_bounds__(256) void join_few_kernel(AttendArgs a, uint32_t dim, uint32_t tile_rows) {
  __shared__ float maxima[4][64], sums[4][64];
  __shared__ f32x4 vectors[4][64];
  const UnitNote *notes = unit_notes(a);
  const uint32_t lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), each = dim / (WIDE ? 8 : 16);
  const uint32_t pieces = min(notes[a.workgroups].parts, a.workgroups);
  uint32_t next = blockIdx.x;
  for (uint32_t from = 0; from < pieces; from += 64) {
    const UnitNote mine = from + lane < pieces ? notes[from + lane] : UnitNote{};
    for (uint64_t shared = __ballot(mine.parts >= 2); shared; shared &= shared - 1) {
      const uint32_t at = (uint32_t)__ffsll((unsigned long long)shared) - 1;
      const UnitNote note{from_lane(mine.parts, at), from_lane(mine.live, at), from_lane(mine.row, at),
                          from_lane(mine.head, at)};
      const uint32_t items = items_of<WIDE>(note, each, tile_rows);
      for (; next < items; next += kFewGroups) {
        const uint32_t block = next / each, first = next % each;
        const Joined<1> some = gather<WIDE, 1, kFewAtOnce>(a, note, from + at, dim, block, first, kFewAtOnce * wave,
                                                           4 * kFewAtOnce);
        __syncthreads();   // the last item's have been read
        maxima[wave][lane] = some.m;
        sums[wave][lane] = some.l;
        vectors[wave][lane] = some.sum[0];
        __syncthreads();
        if (wave) continue;
        float pm[4], pl[4];
        f32x4 got[4][1];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          pm[w] = maxima[w][lane];
          pl[w] = sums[w][lane];
          got[w][0] = vectors[w][lane];
        }
        Joined<1> all;
        all.add(pm, pl, got);
        write<WIDE>(a, note, dim, block, first, all);
      }
      next -= items;
    }
  }
}

uint32_t computed(uint32_t head_dim) { return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256; }

}  // namespace

uint64_t attend_partials(uint32_t tile_rows, uint32_t head_dim, uint32_t workgroups) {
  // Two parts a workgroup, and a note of the unit it began with one more for how many there are.
  return (2 * uint64_t{workgroups} * tile_rows * (computed(head_dim) + 2)) * sizeof(float) +
         (uint64_t{workgroups} + 1) * sizeof(UnitNote);
}

hipError_t launch_attend_join(uint32_t tile_rows, bool few, const AttendArgs &a, hipStream_t stream) {
  const uint32_t dim = computed(a.kv.head_dim);
  const bool wide = tile_rows == kAttendWideRows;
  const auto launch = [&](auto kernel, uint32_t groups) {
    hipLaunchKernelGGL(kernel, dim3(groups), dim3(256), 0, stream, a, dim, tile_rows);
  };
  if (few && wide) launch(join_few_kernel<true>, kFewGroups);
  else if (few) launch(join_few_kernel<false>, kFewGroups);
  else if (wide) launch(join_many_kernel<true>, a.workgroups);
  else launch(join_many_kernel<false>, a.workgroups);
  return hipGetLastError();
}

}  // namespace sq::kern
