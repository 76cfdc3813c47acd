// The schedule both attention tiles run on, worked out by each workgroup from the batch on the device, and the join of
// rows whose keys several workgroups share.
//
// A unit is `fit` consecutive rows of one sequence (tile_rows / group of them, with the query heads of one key head)
// against every key that they see, in tiles of 64 keys. Unit m of a sequence ends at key e_m = position of its last row +
// 1 (or the sequence's end), starts at key s_m (its first row's window), and is e_m - s_m + slack long, slack at least
// 126: 64 or more for each of its tiles, ceil(e_m / 64) - floor(s_m / 64) of them, and what a unit costs besides.
// Lengths live on the device and differ by orders of magnitude within a batch, so no grid over (sequence, head, split) is
// even. Two ways of sharing the units out:
//
//  - Few units (a quarter of the workgroups or fewer, all of them about as long, or short): each is cut into equal
//    parts, as many as give no part more than the share, and a workgroup takes one part. The share is the work over the
//    workgroups that cutting leaves whole, so there are enough of them. One token over 700 keys of 8 key heads: 14 us,
//    where a line (below) cuts units at odd places and gives most workgroups two parts, one after the other: 22 us.
//  - Otherwise the units lie end to end on a line, and workgroup w takes the w-th of equal pieces of it. A piece may end
//    inside a unit, which then has parts. The lengths are linear in m up to the clamps at both ends, so their prefix sums
//    have a closed form, and a workgroup finds its place by a search over the sequences' sums (in LDS) and one over m.
//    Offset o of a unit lies before its tile ceil(o / 64), or past its last tile.
//
// Parts go to the workspace, and a second launch (attend_join.hip) joins them.
#pragma once
#include "batch.hpp"
#include "device.hpp"

namespace sq::kern {

constexpr int kKeyTile = 64;
// The least that a unit is longer than its keys, which makes it 64 for each of its tiles; a tile adds what a unit costs
// it besides keys.
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
__device__ __forceinline__ float uniform(float v) { return __int_as_float(uniform(__float_as_int(v))); }
__device__ __forceinline__ int64_t uniform(int64_t v) {
  return (int64_t)(((uint64_t)uniform((uint32_t)((uint64_t)v >> 32)) << 32) | uniform((uint32_t)v));
}

// a / b for a >= 0, b > 0 and a quotient below 2^50: the doubles' quotient is within one of it, and two multiplications
// settle which (a 64-bit integer division is a hundred instructions in a row).
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  int64_t q = (int64_t)((double)a / (double)b);
  if (q * b > a) --q;
  if ((q + 1) * b <= a) ++q;
  return q;
}
__device__ __forceinline__ int64_t quotient_up(int64_t a, int64_t b) { return quotient(a + b - 1, b); }

// One sequence's units.
struct Units {
  int rows, keys, base, fit, slack, count, window;   // base: the first row's position; window 0: none
  bool causal;
  __device__ __forceinline__ int end(int m) const {
    return causal ? max(1, base + min(rows, fit * (m + 1))) : max(1, keys);
  }
  __device__ __forceinline__ int start(int m) const {
    return window ? max(0, base + fit * m - window + 1) : 0;
  }
  __device__ __forceinline__ int first_tile(int m) const { return start(m) / kKeyTile; }
  __device__ __forceinline__ int tiles(int m) const { return (end(m) + kKeyTile - 1) / kKeyTile - first_tile(m); }
  __device__ __forceinline__ int length(int m) const { return end(m) - start(m) + slack; }
  // The length of units 0 .. m - 1, m < count (the last unit may have fewer rows).
  __device__ __forceinline__ int64_t before(int m) const {
    if (!causal) return (int64_t)m * length(0);
    const int64_t starts = window ? clamped_sum(0, base - window + 1, fit, m) : 0;
    return clamped_sum(1, base + fit, fit, m) - starts + (int64_t)slack * m;
  }
  __device__ __forceinline__ int64_t total() const { return count ? before(count - 1) + length(count - 1) : 0; }
};
// How a tile cuts: the rows of a unit, the shortest piece or part worth a workgroup (four tiles at least), a unit's slack.
struct Cut {
  int fit, least, slack;
};
__device__ __forceinline__ Units units_of(const AttendArgs &a, const Sequence &q, const Cut &cut) {
  // A window as long as the keys hides none of them; clamped, it keeps the sums in range.
  const int window = a.window && a.window < (uint32_t)q.keys ? (int)a.window : 0;
  return {(int)q.rows, q.keys, q.keys - (int)q.rows, cut.fit, cut.slack, ((int)q.rows + cut.fit - 1) / cut.fit, window,
          a.causal != 0};
}

// A unit's part that one workgroup runs: tiles [t0, t1) of the unit's, `parts` parts in all of which this is `part`.
struct Part {
  Units units;
  uint32_t sequence, head, first_row;   // first_row: of the sequence, in the batch
  int m, t0, t1;
  uint32_t part, parts, first_piece;    // first_piece: the workgroup's number that holds part 0
};

// p in scalar registers, whichever way it came.
__device__ __forceinline__ Part settled(const AttendArgs &a, const Cut &cut, const Part &p) {
  const Sequence q{uniform(p.first_row), (uint32_t)uniform(p.units.rows), uniform(p.units.keys)};
  return {units_of(a, q, cut), uniform(p.sequence), uniform(p.head), q.first, uniform(p.m), uniform(p.t0), uniform(p.t1),
          uniform(p.part), uniform(p.parts), uniform(p.first_piece)};
}

// A part's place in the workspace. A piece holds at most two parts of shared units: one that an earlier piece began, and
// one that it begins itself, of which there can be one only. (An even part may be empty, where a unit has fewer tiles
// than parts: it is stored all the same.) A part's blocks of 16 rows (32 in the wide tile) are each the accumulators as
// vectors of four, [vector][lane], then each row's maximum and sum; the same block of consecutive parts lies side by
// side, so that a join's loads of a unit of few rows stay within few pages of memory. The block's number in the workspace:
__device__ __forceinline__ size_t part_block(const AttendArgs &a, uint32_t first_piece, uint32_t part, uint32_t block) {
  return (size_t)(2 * block + (part == 0 ? 1 : 0)) * a.workgroups + first_piece + part;
}
// The first of the four values that a lane's accumulators of vector v are: in a block of 16 rows, where lane (kq, r) holds
// accumulator t = run j + d as value d of run 4 kq + j; and in one of 32 rows, where lane (h, r) holds 4 j + i of block b
// as value 32 b + 8 j + 4 h + i.
__device__ __forceinline__ uint32_t few_value(uint32_t v, uint32_t lane, uint32_t run) {
  return run * (4 * (lane >> 4) + 4 * v / run) + 4 * v % run;
}
__device__ __forceinline__ uint32_t wide_value(uint32_t v, uint32_t lane) {
  return 32 * (v / 4) + 8 * (v % 4) + 4 * (lane >> 5);
}
// What the join wants to know of the shared unit that a piece began: parts below 2 where it began none. Behind the parts
// in the workspace, and behind the pieces' notes one whose `parts` is the number of pieces.
struct UnitNote {
  uint32_t parts, live, row, head;   // live: its rows times query heads; row: its first, in the batch
};
__device__ __forceinline__ UnitNote *unit_notes(const AttendArgs &a) { return (UnitNote *)a.notes; }

constexpr uint32_t kNowhere = 0x7FFFFFF0u;   // past every resource's range: loads zeros, and stores nothing

typedef __attribute__((__vector_size__(2 * sizeof(__bf16)))) __bf16 bf16x2;
__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
  return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)a, (__bf16)b});
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
  return v;
}
__device__ __forceinline__ int64_t wave_sum(int64_t v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
  return v;
}
__device__ __forceinline__ int from_lane(int v, uint32_t lane) { return __builtin_amdgcn_readlane(v, (int)lane); }
__device__ __forceinline__ uint32_t from_lane(uint32_t v, uint32_t lane) { return (uint32_t)from_lane((int)v, lane); }

// The workgroup's number among `active` ones with work (`active` or more: none). Numbers next to each other share keys
// (units of one key head), so they go to workgroups of one XCD (consecutive workgroups go round the eight), whose L2 then
// holds them once.
__device__ __forceinline__ uint32_t piece_of(uint32_t active, uint32_t block) {
  const uint32_t each = (active + 7) / 8;
  return block / 8 < each ? block % 8 * each + block / 8 : active;
}

// LDS for the line.
constexpr uint32_t kCached = 256;   // sequences whose rows and keys stay in LDS
// Where a workgroup stands in its piece of the line between one part and the next.
struct Place {
  int64_t x;
  uint32_t sequence, head;
  int m;
};
template <int THREADS>
struct LineShared {
  int64_t prefix[kMaxSequences + 1];   // where each sequence starts
  int64_t waves[THREADS / 64];
  Sequence sequence[kCached];
  int64_t share;
  Place place[2];
};

// A workgroup's work: one even part, or the piece of the line whose state lies in LDS between its parts (a place that every
// wave reads and one thread writes into the other of two, so that the scalar registers are the tiles').
template <int THREADS>
struct Work {
  bool even;
  uint32_t turn;     // even: 0 until the part is run; else of the place to read, + 2 before the first part
  uint32_t piece;
  uint32_t active;   // workgroups with work

  // The next part of the line, or false; an even part comes from make_work. A barrier of the workgroup's lies between one
  // call and the next.
  __device__ __forceinline__ bool next(const AttendArgs &a, const Cut &cut, LineShared<THREADS> &shared, Part &p) {
    if (even) return turn++ == 0;
    const int64_t share = uniform(shared.share), total = uniform(shared.prefix[a.kv.sequences]);
    const int64_t begin = share * piece, end = begin + share < total ? begin + share : total;
    Place at{};
    if (turn >= 2) {
      at.x = begin;
    } else {
      const Place &last = shared.place[turn];
      at = {uniform(last.x), uniform(last.sequence), uniform(last.head), uniform(last.m)};
    }
    do {
      if (at.x >= end) return false;
      int64_t from = 0;
      if (turn >= 2) from = enter(a, cut, shared, at, p);
      else advance(a, cut, shared, at, p);
      turn &= 1;
      cut_at(from, share, end, at, p);
    } while (p.t1 <= p.t0);
    turn ^= 1;
    if (threadIdx.x == 0) shared.place[turn] = at;
    return true;
  }
  // The notes that the join reads, once all of the workgroup's parts are stored: of the unit it began (began.parts 0:
  // none), and one workgroup's of how many there are.
  __device__ __forceinline__ void leave(const AttendArgs &a, const UnitNote &began) const {
    if (threadIdx.x) return;
    if (piece < active) unit_notes(a)[piece] = began;
    if (blockIdx.x == 0) unit_notes(a)[a.workgroups].parts = active;
  }

 private:
  static __device__ __forceinline__ void take(const AttendArgs &a, const Cut &cut, const LineShared<THREADS> &shared,
                                              const Place &at, Part &p) {
    const Sequence q = at.sequence < kCached ? shared.sequence[at.sequence] : sequence_of(a.kv, at.sequence);
    const Sequence s{uniform(q.first), uniform(q.rows), uniform(q.keys)};
    p.units = units_of(a, s, cut);
    p.first_row = s.first;
    p.sequence = at.sequence;
  }
  // The tiles from offset `from` of unit at.m on, up to its end or the piece's, and at.x moved past them. The parts of a
  // unit are those that start at or before its last tile: a piece is at least a tile long, so each of them has one.
  __device__ __forceinline__ void cut_at(int64_t from, int64_t share, int64_t end, Place &at, Part &p) const {
    const int64_t length = p.units.length(at.m);
    const int64_t to = length < from + (end - at.x) ? length : from + (end - at.x);
    const int tiles = p.units.tiles(at.m);
    const auto tile_at = [&](int64_t o) {
      const int64_t t = (o + kKeyTile - 1) / kKeyTile;
      return t < tiles ? (int)t : tiles;
    };
    p.head = at.head;
    p.m = at.m;
    p.t0 = tile_at(from);
    p.t1 = tile_at(to);
    const int64_t unit = at.x - from;
    p.first_piece = from ? (uint32_t)uniform(quotient(unit, share)) : piece;
    p.parts = from == 0 && to == length
                  ? 1
                  : (uint32_t)uniform(quotient(unit + (int64_t)kKeyTile * (tiles - 1), share)) - p.first_piece + 1;
    p.part = piece - p.first_piece;
    at.x += to - from;
  }
  // The first part: the unit at at.x on the line, and the offset in it.
  static __device__ __forceinline__ int64_t enter(const AttendArgs &a, const Cut &cut, const LineShared<THREADS> &shared,
                                                  Place &at, Part &p) {
    uint32_t lo = 0, hi = a.kv.sequences;   // the last sequence that starts at or before x
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) / 2;
      if (uniform(shared.prefix[mid]) <= at.x) lo = mid;
      else hi = mid;
    }
    at.sequence = lo;
    take(a, cut, shared, at, p);
    const Units &u = p.units;
    const int64_t one = u.total();
    int64_t rest = at.x - uniform(shared.prefix[lo]);
    at.head = (uint32_t)uniform(quotient(rest, one));
    rest -= one * at.head;
    int mlo = 0, mhi = u.count;
    while (mhi - mlo > 1) {
      const int mid = (mlo + mhi) / 2;
      if (u.before(mid) <= rest) mlo = mid;
      else mhi = mid;
    }
    at.m = mlo;
    return rest - u.before(mlo);
  }
  // The part after the last one: the next unit, from its start.
  static __device__ __forceinline__ void advance(const AttendArgs &a, const Cut &cut, const LineShared<THREADS> &shared,
                                                 Place &at, Part &p) {
    take(a, cut, shared, at, p);
    if (++at.m < p.units.count) return;
    at.m = 0;
    if (++at.head < a.kv.kv_heads) return;
    at.head = 0;
    do {   // there is one with units: x lies before the line's end
      ++at.sequence;
      take(a, cut, shared, at, p);
    } while (!p.units.count);
  }
};

// Every thread of the workgroup takes part.
template <int THREADS>
__device__ __forceinline__ Work<THREADS> make_work(const AttendArgs &a, const Cut &cut, LineShared<THREADS> &shared,
                                                   Part &p) {
  constexpr int kWaves = THREADS / 64;
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, count = a.kv.sequences;
  Work<THREADS> w{};
  if (count <= 64) {
    // Each wave for itself, a sequence a lane, in registers.
    const Sequence q = lane < count ? sequence_of(a.kv, lane) : Sequence{0u, 0u, 0};
    const Units u = units_of(a, q, cut);
    const float heads = (float)a.kv.kv_heads, units = (float)u.count, last = u.count ? (float)u.length(u.count - 1) : 0.0f,
                first = u.count ? (float)u.length(0) : 0.0f;
    const float number = uniform(heads * wave_sum(units)), most = uniform(heads * wave_sum(units * last)),
                work = uniform(heads * wave_sum(units * 0.5f * (first + last)));
    if (number * 4 <= (float)a.workgroups && (most <= work * 1.25f || most <= number * (float)cut.least)) {
      // The share that leaves every unit's last part room: units ceil(length / share) <= workgroups. The sums are off by
      // 2^-18 at most, the share made larger by as much.
      const int share = max(cut.least, (int)(most * (1 + 0x1p-18f) / ((float)a.workgroups - number)) + 1);
      const uint32_t parts = u.count ? (uint32_t)(u.length(u.count - 1) + share - 1) / (uint32_t)share : 0u;
      const uint32_t mine = parts * (uint32_t)u.count * a.kv.kv_heads;
      uint32_t upto = mine;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const uint32_t below = (uint32_t)__shfl_up((int)upto, d);
        if (lane >= (uint32_t)d) upto += below;
      }
      w.even = true;
      w.active = from_lane(upto, 63);
      w.piece = piece_of(w.active, blockIdx.x);
      if (w.piece >= w.active) {
        w.turn = 1;
        return w;
      }
      // The last sequence that starts at or before the piece: one with units, as the next starts past it.
      const uint32_t before = upto - mine;
      const uint32_t s = (uint32_t)__popcll(__ballot(before <= w.piece)) - 1;
      p.sequence = s;
      p.units = units_of(a, Sequence{from_lane(q.first, s), from_lane(q.rows, s), from_lane(q.keys, s)}, cut);
      p.first_row = from_lane(q.first, s);
      p.parts = from_lane(parts, s);
      const uint32_t rest = w.piece - from_lane(before, s), unit = rest / p.parts;
      p.part = rest - unit * p.parts;
      p.head = unit / (uint32_t)p.units.count;
      p.m = (int)(unit - p.head * (uint32_t)p.units.count);
      // The unit's tiles over its parts, the first ones taking what is left over. (A unit much shorter than its
      // sequence's last may leave parts empty: they count all the same.)
      const uint32_t tiles = (uint32_t)p.units.tiles(p.m), each = tiles / p.parts, over = tiles - each * p.parts;
      p.t0 = (int)(each * p.part + min(p.part, over));
      p.t1 = p.t0 + (int)(each + (p.part < over ? 1 : 0));
      p.first_piece = w.piece - p.part;
      return w;
    }
  }
  int64_t carry = 0;
  for (uint32_t s0 = 0; s0 < count; s0 += THREADS) {
    const uint32_t s = s0 + threadIdx.x;
    int64_t v = 0;
    if (s < count) {
      const Sequence q = sequence_of(a.kv, s);
      if (s < kCached) shared.sequence[s] = q;
      v = units_of(a, q, cut).total() * a.kv.kv_heads;
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int64_t below = __shfl_up(v, d);
      if (lane >= (uint32_t)d) v += below;
    }
    if (s0) __syncthreads();   // the last turn's sums have been read
    if (lane == 63) shared.waves[wave] = v;
    __syncthreads();
    int64_t all = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      if ((uint32_t)i < wave) v += shared.waves[i];
      all += shared.waves[i];
    }
    if (s < count) shared.prefix[s + 1] = carry + v;
    carry += all;
  }
  if (threadIdx.x == 0) shared.prefix[0] = 0;
  const int64_t total = uniform(carry), even_share = uniform(quotient_up(total, a.workgroups));
  const int64_t share = even_share > cut.least ? even_share : cut.least;
  if (threadIdx.x == 0) shared.share = share;
  w.active = (uint32_t)uniform(quotient_up(total, share));
  w.piece = piece_of(w.active, blockIdx.x);
  w.turn = 2;
  __syncthreads();
  return w;
}

// Two of a key's values for each of two keys, regrouped: two keys of each of two values.
__device__ __forceinline__ uint32_t low_halves(uint32_t k0, uint32_t k1) {
  return __builtin_amdgcn_perm(k1, k0, 0x05040100u);
}
__device__ __forceinline__ uint32_t high_halves(uint32_t k0, uint32_t k1) {
  return __builtin_amdgcn_perm(k1, k0, 0x07060302u);
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

// The sign bits of a word's e4m3 codes that are NaN (all seven bits below the sign's set), in their places.
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) { return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u; }

// A running maximum is raised when a score exceeds it by more than this.
constexpr float kRaise = 8.0f;

// p / group for a packed row p < 128 and a group of at most 64: the fp32 quotient of p + 1/2 is a 128th or more from a
// whole number, its error far less.
__device__ __forceinline__ int row_of(int p, float by_group) { return (int)(((float)p + 0.5f) * by_group); }

// 2^x by the hardware instruction (an ulp; results below the normal range flush to zero, far below any weight that
// counts).
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
// The maximum to subtract: scores of -inf (nothing seen yet) must give weights of zero, not of NaN.
__device__ __forceinline__ float finite_max(float m) { return m == -INFINITY ? 0.0f : m; }

}  // namespace sq::kern
