// The join of units whose keys several workgroups shared: output = sum_j e^(m_j - m) O_j / sum_j e^(m_j - m) l_j over a
// unit's parts in key order, m their largest maximum. A launch of its own after the attention's: a workgroup of that one
// would find out that it is the last of its unit's only after its stores and an atomic have gone past the XCDs' caches
// (3 us a part), and then join all of the unit's rows alone (one token over 131072 int8 keys, 31 parts a unit: 8 us in
// all), where here the vectors of every unit go over all waves, with many parts' loads in flight.
#include "attend.hpp"

namespace sq::kern {
namespace {

// VECTORS of a unit's vectors (attend.hpp: the layout of a part) by a wave, AT_ONCE parts' loads in flight.
template <bool WIDE, int VECTORS, int AT_ONCE>
__device__ __forceinline__ void join(const AttendArgs &a, const UnitNote &note, uint32_t piece, uint32_t dim_computed,
                                     uint32_t tile_rows, uint32_t block, uint32_t first) {
  const uint32_t rows = WIDE ? 32 : 16, lane = threadIdx.x & 63;
  const uint32_t p = block * rows + lane % rows;
  const bool on = p < note.live;
  const uint32_t part_floats = tile_rows * (dim_computed + 2), block_floats = rows * (dim_computed + 2);
  float m = -INFINITY, l = 0.0f;
  f32x4 sum[VECTORS] = {};
  for (uint32_t j = 0; j < note.parts; j += AT_ONCE) {
    float pm[AT_ONCE], pl[AT_ONCE];
    f32x4 got[AT_ONCE][VECTORS];
#pragma unroll
    for (int d = 0; d < AT_ONCE; ++d) {
      // Past the last part the resource is empty: zeros, and nothing read.
      const bool there = j + d < note.parts;
      const float *from = a.partials + (size_t)part_slot(piece, there ? j + d : 0) * part_floats +
                          (size_t)block * block_floats;
      const __amdgpu_buffer_rsrc_t r = buffer_rsrc(from, there ? block_floats * 4 : 0);
      const u32x2 two = buffer_b64<0>(r, on ? (rows * dim_computed + 2 * (lane % rows)) * 4 : kNowhere, 0);
      pm[d] = __uint_as_float(two[0]);
      pl[d] = __uint_as_float(two[1]);
#pragma unroll
      for (int v = 0; v < VECTORS; ++v)
        got[d][v] = __builtin_bit_cast(f32x4, buffer_b128<0>(r, on ? ((first + v) * 64 + lane) * 16 : kNowhere, 0));
    }
    float next = m;
#pragma unroll
    for (int d = 0; d < AT_ONCE; ++d) next = pl[d] == 0.0f ? next : fmaxf(next, pm[d]);
    // A part that saw nothing adds nothing, even to a row whose maximum is infinite.
    const float keep = l == 0.0f ? 0.0f : exp2_fast(m - finite_max(next));
    m = next;
    l *= keep;
#pragma unroll
    for (int v = 0; v < VECTORS; ++v) sum[v] *= keep;
#pragma unroll
    for (int d = 0; d < AT_ONCE; ++d) {
      const float by = pl[d] == 0.0f ? 0.0f : exp2_fast(pm[d] - finite_max(next));
      l += pl[d] * by;
#pragma unroll
      for (int v = 0; v < VECTORS; ++v) sum[v] += got[d][v] * by;
    }
  }
  if (!on) return;
  const float by = l == 0.0f ? 0.0f : 1.0f / l;
  const uint32_t i = (uint32_t)row_of((int)p, 1.0f / (float)a.group), g = p - i * a.group;
  uint16_t *out = a.output + (size_t)(note.row + i) * a.output_stride + (note.head * a.group + g) * a.kv.head_dim;
#pragma unroll
  for (int v = 0; v < VECTORS; ++v) {
    const uint32_t value = WIDE ? wide_value(first + v, lane) : few_value(first + v, lane, dim_computed / 16);
    if (value < a.kv.head_dim)
      *(u32x2 *)(out + value) = u32x2{bf16_pair(sum[v][0] * by, sum[v][1] * by), bf16_pair(sum[v][2] * by, sum[v][3] * by)};
  }
}

// The blocks and vectors of a unit, from item `next` on every `stride`-th; next becomes that of the unit after. dim is the
// head's values as computed.
template <bool WIDE, int VECTORS, int AT_ONCE>
__device__ __forceinline__ void join_items(const AttendArgs &a, const UnitNote &note, uint32_t piece, uint32_t dim,
                                           uint32_t tile_rows, uint32_t &next, uint32_t stride) {
  const uint32_t rows = WIDE ? 32 : 16, each = dim / (WIDE ? 8 : 16) / VECTORS;
  const uint32_t items = min(tile_rows / rows, (note.live + rows - 1) / rows) * each;
  for (; next < items; next += stride)
    join<WIDE, VECTORS, AT_ONCE>(a, note, piece, dim, tile_rows, next / each, VECTORS * (next % each));
  next -= items;
}

// Many units: a workgroup a piece, for the shared unit that it began if any. Those of a line mostly have two parts, which
// go eight vectors at a time (rows of the wide tile have as many).
template <bool WIDE>
__global__ __launch_bounds__(256) void join_many_kernel(AttendArgs a, uint32_t dim, uint32_t tile_rows) {
  const UnitNote *notes = unit_notes(a);
  const uint32_t pieces = notes[a.workgroups].parts;
  const UnitNote note = notes[blockIdx.x];   // read beside the number of pieces, of which it may be past
  if (blockIdx.x >= pieces || note.parts < 2) return;
  uint32_t next = uniform(threadIdx.x >> 6);
  if (WIDE && note.parts == 2) join_items<WIDE, 8, 2>(a, note, blockIdx.x, dim, tile_rows, next, 4);
  else join_items<WIDE, 2, 16>(a, note, blockIdx.x, dim, tile_rows, next, 4);
}

// Few units, of many parts each: every wave looks through the notes, one a lane, and the waves of all workgroups take the
// units' blocks and vectors in turn.
constexpr uint32_t kFewGroups = 256;
template <bool WIDE>
__global__ __launch_bounds__(256) void join_few_kernel(AttendArgs a, uint32_t dim, uint32_t tile_rows) {
  const UnitNote *notes = unit_notes(a);
  const uint32_t lane = threadIdx.x & 63, pieces = min(notes[a.workgroups].parts, a.workgroups);
  uint32_t next = uniform(4 * blockIdx.x + (threadIdx.x >> 6));
  for (uint32_t first = 0; first < pieces; first += 64) {
    const UnitNote mine = first + lane < pieces ? notes[first + lane] : UnitNote{};
    for (uint64_t shared = __ballot(mine.parts >= 2); shared; shared &= shared - 1) {
      const uint32_t from = (uint32_t)__ffsll((unsigned long long)shared) - 1;
      join_items<WIDE, 1, 32>(a,
                              {from_lane(mine.parts, from), from_lane(mine.live, from), from_lane(mine.row, from),
                               from_lane(mine.head, from)},
                              first + from, dim, tile_rows, next, 4 * kFewGroups);
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
