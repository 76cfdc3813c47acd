// The schedule both attention tiles run on, worked out by each workgroup from the batch on the device, and the join of
// rows whose keys several workgroups share.
//
// A unit is `fit` consecutive rows of one sequence (tile_rows / group of them, with the query heads of one key head)
// against every key that they see, in tiles of 64 keys. Lengths live on the device and differ by orders of magnitude
// within a batch, so no grid over (sequence, head, split) is even: instead the units lie end to end on a line, each as
// long as its keys, and workgroup w takes the w-th of equal pieces of that line. A piece may end inside a unit; the unit
// then has parts, which the workgroup that finishes last joins.
//
// Unit m of a sequence ends at key e_m = position of its last row + 1 (or the sequence's end), starts at key s_m (its
// first row's window), and is e_m - s_m + 126 long: at least 64 for each of its tiles, ceil(e_m / 64) - floor(s_m / 64)
// of them, and a little for its fixed cost. The lengths are linear in m up to the clamps at both ends, so their prefix
// sums have a closed form, and a workgroup finds its place by a search over the sequences' sums (in LDS) and one over m,
// in the few hundred instructions that a walk over the units would spend on a handful of them. Offset o of a unit's line
// lies before tile ceil(o / 64), or past its last tile.
#pragma once
#include "batch.hpp"

namespace sq::kern {

constexpr int kKeyTile = 64;
constexpr int kUnitSlack = 2 * (kKeyTile - 1);
constexpr uint32_t kMaxSequences = SQ_KV_MAX_SEQUENCES;

// sum over i < m of max(lo, a + r i).
__device__ __forceinline__ int64_t clamped_sum(int lo, int a, int r, int m) {
  const int below = a > lo ? 0 : min(m, (lo - a) / r + 1);
  return (int64_t)lo * below + (int64_t)a * (m - below) +
         (int64_t)r * ((int64_t)m * (m - 1) - (int64_t)below * (below - 1)) / 2;
}

// A value that every lane of the wave holds, in scalar registers.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return (uint32_t)uniform((int)v); }
__device__ __forceinline__ int64_t uniform(int64_t v) {
  return (int64_t)(((uint64_t)uniform((uint32_t)((uint64_t)v >> 32)) << 32) | uniform((uint32_t)v));
}

// One sequence's units.
struct Units {
  int rows, keys, base, fit, count, window;   // base: the first row's position; window 0: none
  bool causal;
  __device__ __forceinline__ int end(int m) const {
    return causal ? max(1, base + min(rows, fit * (m + 1))) : max(1, keys);
  }
  __device__ __forceinline__ int start(int m) const {
    return window ? max(0, base + fit * m - window + 1) : 0;
  }
  __device__ __forceinline__ int first_tile(int m) const { return start(m) / kKeyTile; }
  __device__ __forceinline__ int tiles(int m) const { return (end(m) + kKeyTile - 1) / kKeyTile - first_tile(m); }
  __device__ __forceinline__ int length(int m) const { return end(m) - start(m) + kUnitSlack; }
  // The length of units 0 .. m - 1, m < count (the last unit may have fewer rows).
  __device__ __forceinline__ int64_t before(int m) const {
    if (!causal) return (int64_t)m * length(0);
    const int64_t starts = window ? clamped_sum(0, base - window + 1, fit, m) : 0;
    return clamped_sum(1, base + fit, fit, m) - starts + (int64_t)kUnitSlack * m;
  }
  __device__ __forceinline__ int64_t total() const { return count ? before(count - 1) + length(count - 1) : 0; }
};
__device__ __forceinline__ Units units_of(const AttendArgs &a, const Sequence &q, int fit) {
  // A window as long as the keys hides none of them; clamped, it keeps the sums in range.
  const int window = a.window && a.window < (uint32_t)q.keys ? (int)a.window : 0;
  return {(int)q.rows, q.keys, q.keys - (int)q.rows, fit, ((int)q.rows + fit - 1) / fit, window, a.causal != 0};
}

// The line: prefix[s] is where sequence s starts, prefix[sequences] its end; share is a workgroup's piece of it.
struct Line {
  const int64_t *prefix;
  int64_t total;
  int64_t share;
  uint32_t active;   // workgroups with a piece
};

// Every thread of the workgroup takes part. `prefix` is LDS for sequences + 1 values, `part` for a value a wave. least:
// the shortest piece worth a workgroup (at least a tile).
template <int THREADS>
__device__ __forceinline__ Line make_line(const AttendArgs &a, int fit, int least, int64_t *prefix, int64_t *part) {
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t carry = 0;
  for (uint32_t s0 = 0; s0 < a.kv.sequences; s0 += THREADS) {
    const uint32_t s = s0 + threadIdx.x;
    int64_t v = s < a.kv.sequences ? units_of(a, sequence_of(a.kv, s), fit).total() * a.kv.kv_heads : 0;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int64_t u = __shfl_up(v, d);
      if (lane >= (uint32_t)d) v += u;
    }
    if (lane == 63) part[wave] = v;
    __syncthreads();
    int64_t all = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
      if ((uint32_t)w < wave) v += part[w];
      all += part[w];
    }
    if (s < a.kv.sequences) prefix[s + 1] = carry + v;
    carry += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) prefix[0] = 0;
  __syncthreads();
  carry = uniform(carry);
  const int64_t even = (carry + a.workgroups - 1) / a.workgroups, share = even > least ? even : least;
  return {prefix, carry, share, (uint32_t)((carry + share - 1) / share)};
}

// The piece of workgroup `block`. Pieces next to each other on the line share keys (units of one key head), so they go
// to workgroups of one XCD (consecutive workgroups go round the eight), whose L2 then holds them once. Past the last:
// a number past line.active.
__device__ __forceinline__ uint32_t piece_of(const Line &line, uint32_t block) {
  return block % 8 * ((line.active + 7) / 8) + block / 8;
}

// A unit's part that one workgroup runs: tiles [t0, t1) of the unit's, `parts` parts in all of which this is `part`.
struct Part {
  Units units;
  uint32_t sequence, head, first_row;   // first_row: of the sequence, in the batch
  int m, t0, t1;
  uint32_t part, parts, first_piece;    // first_piece: the workgroup piece that holds part 0
};
// The part at x < end on the line (wave-uniform), and x moved past it.
__device__ __forceinline__ Part next_part(const AttendArgs &a, const Line &line, int fit, int64_t &x, int64_t end,
                                          uint32_t piece) {
  uint32_t lo = 0, hi = a.kv.sequences;   // the last sequence that starts at or before x
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if (uniform(line.prefix[mid]) <= x) lo = mid;
    else hi = mid;
  }
  Part p;
  p.sequence = lo;
  const Sequence q = sequence_of(a.kv, p.sequence);
  p.units = units_of(a, q, fit);
  p.first_row = q.first;
  const int64_t one = p.units.total();
  int64_t rest = x - uniform(line.prefix[p.sequence]);
  p.head = (uint32_t)(rest / one);
  rest -= one * p.head;
  int mlo = 0, mhi = p.units.count;
  while (mhi - mlo > 1) {
    const int mid = (mlo + mhi) / 2;
    if (p.units.before(mid) <= rest) mlo = mid;
    else mhi = mid;
  }
  p.m = mlo;
  const int64_t from = rest - p.units.before(mlo), length = p.units.length(mlo);
  const int64_t to = length < from + (end - x) ? length : from + (end - x);
  const int tiles = p.units.tiles(mlo);
  const auto tile_at = [&](int64_t o) {
    const int64_t t = (o + kKeyTile - 1) / kKeyTile;
    return t < tiles ? (int)t : tiles;
  };
  p.t0 = tile_at(from);
  p.t1 = tile_at(to);
  // The parts of a unit are those that start at or before its last tile: a piece is at least a tile long, so each of
  // them has one.
  const int64_t unit = x - from;
  p.first_piece = (uint32_t)(unit / line.share);
  p.parts = (uint32_t)((unit + (int64_t)kKeyTile * (tiles - 1)) / line.share) - p.first_piece + 1;
  p.part = piece - p.first_piece;
  x += to - from;
  return p;
}

// A part's place in the workspace. A piece holds at most two parts of shared units: one that an earlier piece began, and
// one that it begins itself, of which there can be one only, so that the piece's counter counts that unit's parts.
__device__ __forceinline__ uint32_t part_slot(uint32_t first_piece, uint32_t part) {
  return 2 * (first_piece + part) + (part == 0 ? 1 : 0);
}

// Announces this workgroup's part, whose stores (agent-scope, so they lie past the XCD's own L2) come before; true in
// the workgroup that arrives last, which then sees every part through agent-scope loads. As in split_reduce: each wave
// waits for its own stores before the barrier, and the counter returns to zero.
__device__ __forceinline__ bool last_part(uint32_t *counter, uint32_t parts, uint32_t *arrival) {
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (threadIdx.x == 0) {
    const uint32_t n = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (n == parts - 1) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *arrival = n;
  }
  __syncthreads();
  return *arrival == parts - 1;
}
__device__ __forceinline__ void store_pair(float *at, float a, float b) {
  const uint64_t v = (uint64_t)__float_as_uint(a) | ((uint64_t)__float_as_uint(b) << 32);
  __hip_atomic_store((uint64_t *)at, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void load_pair(const float *at, float &a, float &b) {
  const uint64_t v = __hip_atomic_load((const uint64_t *)at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  a = __uint_as_float((uint32_t)v);
  b = __uint_as_float((uint32_t)(v >> 32));
}

// 2^x by the hardware instruction (an ulp; results below the normal range flush to zero, far below any weight that
// counts).
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
// The maximum to subtract: scores of -inf (nothing seen yet) must give weights of zero, not of NaN.
__device__ __forceinline__ float finite_max(float m) { return m == -INFINITY ? 0.0f : m; }

}  // namespace sq::kern
