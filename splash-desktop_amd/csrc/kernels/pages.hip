// A cache's pages shared out, released, moved and copied, from books that only the device holds (include/splash_q4.h). What
// moves is whole pages, or the rows with keys of a sequence's last one: twice their bytes of HBM, at a large copy's rate if
// enough is under way. So a copy is cut into chunks of 4 KiB, each a wave's, four vectors a lane in flight, the chunks of all
// pages end to end over the card's waves. The rest is latency: a launch each for what has to be known before the next part,
// two for a grow or a fork (which pages are free; then entries and copies), three to compact (how many pages of each 4096 are
// in use; which goes where; then entries and copies), one for the others.
//
// What it reaches: 1012 pages of 68 KiB copied in 32 us, 4.3 TB/s read and written of a large copy's 4.9 to 5.1; a
// pool with 251 MB to move compacted in 53 us, 4.7 TB/s, after 5 + 5; 11 sequences released and forked in 4.7 and 5.9 + 4.6, of
// which a launch that does nothing takes 1.6 and each round trip 1 to 2.
//
// A grow or a fork looks for free pages with one workgroup, from the first page on until it has enough, 16384 references a step of
// 2.4 us. Where the free ones are the last, the release and fork of 11 sequences take 17 us in a pool of 1024 pages, 20 of
// 16384, 27 of 65536, 50 of 262144 and 174 of 2^20.
//
// No order of atomics shows: counts go up and down by whole numbers, and new pages are given out by prefix sums, the lowest
// free one first.
#include "pages.hpp"

#include <algorithm>

#include "device.hpp"

namespace sq::kern {
namespace {

constexpr uint32_t kHole = ~0u;
constexpr uint32_t kRequests = SQ_KV_MAX_SEQUENCES;
constexpr int kPlanThreads = 1024, kPagesAThread = 16;
constexpr uint32_t kBlockPages = 256 * kPagesAThread;   // of a workgroup that counts
constexpr uint32_t kSlab = 4096;                        // entries of a table row that a workgroup takes at a time

// The workspace: a head of 16 words, items, and lists of words.
struct Head {
  uint32_t moves, live;   // compact: pages to move, and in use
};
constexpr uint32_t kHeadWords = 16;
static_assert(sizeof(Head) <= 4 * kHeadWords);
struct Item {
  uint32_t row, offset, first, fresh;   // first: the entry of the first of `fresh` new pages; offset: theirs in the free list
  uint32_t length, from, rows, parent;  // from, rows: the page to copy (rows 0: none) into the first of them
};
struct Workspace {
  Head *head;
  Item *items;         // take: a request's; row ~0u where it is not carried out
  uint32_t *free;      // take: pages; compact: the free places below the number in use
  uint32_t *used;      // compact: the pages in use past it, last first
  uint32_t *rank;      // compact: such a page's number among them
  uint32_t *counts;    // compact: pages in use of each kBlockPages
};
__device__ __forceinline__ Workspace workspace_of(const PoolArgs &p) {
  uint32_t *w = p.workspace;
  uint32_t *lists = w + kHeadWords + kRequests * sizeof(Item) / 4;
  return {(Head *)w, (Item *)(w + kHeadWords), lists, lists + p.pages, lists + 2 * (size_t)p.pages, lists + 3 * (size_t)p.pages};
}

// The sum over the threads before this one, and over all of them; THREADS / 64 words of LDS. A barrier before the next call.
template <int THREADS, typename T>
__device__ __forceinline__ T block_sums(T v, T *waves, T &all) {
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  T upto = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const T below = __shfl_up(upto, d);
    if (lane >= (uint32_t)d) upto += below;
  }
  if (lane == 63) waves[wave] = upto;
  __syncthreads();
  T before = upto - v;
  all = 0;
#pragma unroll
  for (int i = 0; i < THREADS / 64; ++i) {
    if ((uint32_t)i < wave) before += waves[i];
    all += waves[i];
  }
  return before;
}

// One bit a page, set where it is free, of the pages from `first` on; pages past the last are not free. (Buffer loads: the
// references are 4-byte aligned.)
__device__ __forceinline__ uint32_t free_bits(const PoolArgs &p, uint32_t first) {
  const __amdgpu_buffer_rsrc_t r = buffer_rsrc(p.references, p.pages * 4);
  u32x4 v[kPagesAThread / 4];
#pragma unroll
  for (int i = 0; i < kPagesAThread / 4; ++i) v[i] = buffer_b128<0>(r, first < p.pages ? (first + 4 * i) * 4 : 0, 0);
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < kPagesAThread; ++i) bits |= (uint32_t)(first + i < p.pages && v[i / 4][i % 4] == 0) << i;
  return bits;
}

// One entry fewer names the page. (A count that is zero stays so, whatever books that contradict themselves say.)
__device__ __forceinline__ void drop(uint32_t *references, uint32_t page) {
  uint32_t was = __hip_atomic_load(&references[page], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  while (was) {
    const uint32_t got = atomicCAS(&references[page], was, was - 1);
    if (got == was) return;
    was = got;
  }
}

// The wave's chunk `chunk` of page `from` copied to page `to`: the rows below `rows` of each key head.
__device__ __forceinline__ void copy_chunk(const PageRuns &p, uint32_t from, uint32_t to, uint32_t rows, uint32_t chunk) {
  uint32_t run = 0;
#pragma unroll
  for (uint32_t i = 1; i < 4; ++i)
    if (i < p.runs && chunk >= p.first_chunk[i]) run = i;
  const uint32_t bytes = p.bytes[run], at = (chunk - p.first_chunk[run]) * kPageChunk + 16 * (threadIdx.x & 63);
  const uint8_t *source = p.from[run] + (size_t)from * bytes;
  uint8_t *target = p.to[run] + (size_t)to * bytes;
  u32x4 v[4];
  uint32_t live[4];   // bytes of the vector
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t o = at + 1024 * i;
    live[i] = o < bytes ? 16 : 0;
    if (rows < p.page_rows && live[i]) {
      // A vector lies in one key head (pages have a multiple of 16 rows), and holds a part of a row or several of them.
      const uint32_t row = o / p.row_bytes[run] % p.page_rows;
      live[i] = row >= rows ? 0 : min(16u, max(16u, p.row_bytes[run]) == 16u ? (rows - row) * p.row_bytes[run] : 16u);
    }
    if (live[i]) v[i] = *(const u32x4 *)(source + o);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint8_t *out = target + at + 1024 * i;
    if (live[i] == 16) {
      *(u32x4 *)out = v[i];
    } else if (live[i]) {   // the last scales: an even number of bytes, one row's at least 2
#pragma unroll
      for (uint32_t b = 0; b < 16; b += 2)
        if (b < live[i]) *(uint16_t *)(out + b) = (uint16_t)(v[i][b / 4] >> (8 * (b % 4)));
    }
  }
}

__global__ __launch_bounds__(256) void release_kernel(PoolArgs p, const uint32_t *rows, const uint32_t *keeps,
                                                      uint32_t requests, uint32_t slabs) {
  if (blockIdx.x == 0) {
    __shared__ uint32_t waves[4];
    uint32_t missing = 0, all;
    for (uint32_t i = threadIdx.x; i < requests; i += 256) missing += rows[i] >= p.sequences;
    (void)block_sums<256>(missing, waves, all);
    if (threadIdx.x == 0) {
      p.report[0] = all;
      p.report[1] = 0;
    }
  }
  for (uint32_t task = blockIdx.x; task < requests * slabs; task += gridDim.x) {
    const uint32_t slab = task % slabs, row = rows[task / slabs], keep = keeps[task / slabs];
    if (row >= p.sequences) continue;
    if (slab == 0 && threadIdx.x == 0) atomicMin(&p.lengths[row], keep);
    const uint32_t first = keep / p.page_rows + (keep % p.page_rows != 0);
    const uint32_t end = min(p.pages_per_sequence, kSlab * (slab + 1));
    uint32_t *entries = p.table + (size_t)row * p.pages_per_sequence;
    for (uint32_t e = max(first, kSlab * slab) + threadIdx.x; e < end; e += 256) {
      // Exchanged, so that of two requests that name the sequence one alone drops the entry.
      if (entries[e] == kHole) continue;
      const uint32_t page = atomicExch(&entries[e], kHole);
      if (page < p.pages) drop(p.references, page);
    }
  }
}

// Which requests are carried out, and with which pages. One workgroup, a thread a request.
__global__ __launch_bounds__(kPlanThreads) void take_plan_kernel(PoolArgs p, const uint32_t *rows, const uint32_t *more,
                                                                 const uint32_t *parents, uint32_t requests) {
  __shared__ uint32_t named[kRequests], from[kRequests], waves[kPlanThreads / 64], lost, copied;
  __shared__ uint64_t wide[kPlanThreads / 64];
  const Workspace w = workspace_of(p);
  const uint32_t i = threadIdx.x;
  const bool fork = parents != nullptr;
  const uint64_t most = (uint64_t)p.pages_per_sequence * p.page_rows;
  if (i == 0) lost = copied = 0;
  uint32_t bits = free_bits(p, i * kPagesAThread);   // the first pages' while the requests are looked at
  Item item{kHole, 0, 0, 0, 0, 0, 0, 0};
  uint32_t row = kHole, parent = kHole;
  if (i < requests) {
    row = rows[i];
    parent = fork ? parents[i] : row;
  }
  named[i] = row;
  from[i] = parent;
  __syncthreads();
  bool valid = row < p.sequences && parent < p.sequences;
  for (uint32_t j = 0; j < requests; ++j) valid = valid && !(j < i && named[j] == row) && !(fork && from[j] == row);
  if (valid) {
    const uint64_t keys = min((uint64_t)p.lengths[parent], most), grown = fork ? keys : keys + more[i];
    valid = grown <= most;
    if (valid) {
      const uint32_t part = (uint32_t)(keys % p.page_rows), full = (uint32_t)(keys / p.page_rows);
      const uint32_t page = part ? p.table[(size_t)parent * p.pages_per_sequence + full] : kHole;
      const bool copy = page < p.pages && (fork || (grown > keys && p.references[page] > 1));
      item.row = row;
      item.parent = parent;
      item.length = (uint32_t)grown;
      item.first = fork || copy ? full : full + (part != 0);
      item.fresh = fork ? copy : (uint32_t)((grown + p.page_rows - 1) / p.page_rows) - full - (part != 0) + copy;
      item.from = page;
      item.rows = copy ? part : 0;
    }
  }
  uint64_t wanted;
  const uint64_t before = block_sums<kPlanThreads>((uint64_t)item.fresh, wide, wanted);
  item.offset = (uint32_t)min(before, (uint64_t)p.pages);
  // The free pages in order, as many as are wanted.
  uint32_t found = 0;
  for (uint32_t first = 0; first < p.pages && found < wanted;) {
    const uint32_t next = first + kPlanThreads * kPagesAThread;
    const uint32_t ahead = next < p.pages && next > first ? free_bits(p, next + i * kPagesAThread) : 0u;
    uint32_t all;
    uint32_t at = found + block_sums<kPlanThreads>((uint32_t)__popc(bits), waves, all);
    for (uint32_t rest = bits; rest && at < wanted; rest &= rest - 1)
      w.free[at++] = first + i * kPagesAThread + (uint32_t)__ffs(rest) - 1;
    found += all;
    bits = ahead;
    __syncthreads();
    if (next <= first) break;
    first = next;
  }
  if (i < requests) {
    if (valid && item.fresh && before + item.fresh > found) valid = false;
    if (!valid) {
      item = Item{kHole, 0, 0, 0, 0, 0, 0, 0};
      atomicAdd(&lost, 1u);
    } else if (item.rows) {
      atomicAdd(&copied, 1u);
    }
    w.items[i] = item;
  }
  __syncthreads();
  if (i == 0) {
    p.report[0] = lost;
    p.report[1] = copied;
  }
}

__global__ __launch_bounds__(256) void take_apply_kernel(PoolArgs p, uint32_t requests, uint32_t slabs, uint32_t fork) {
  const Workspace w = workspace_of(p);
  for (uint32_t task = blockIdx.x; task < requests * slabs; task += gridDim.x) {
    const Item item = w.items[task / slabs];
    const uint32_t slab = task % slabs;
    if (item.row == kHole) continue;
    uint32_t *entries = p.table + (size_t)item.row * p.pages_per_sequence;
    const uint32_t *theirs = p.table + (size_t)item.parent * p.pages_per_sequence;
    if (slab == 0 && threadIdx.x == 0) p.lengths[item.row] = item.length;
    const uint32_t end = min(p.pages_per_sequence, kSlab * (slab + 1));
    const uint32_t shared = fork ? item.length / p.page_rows : 0;   // a fork's whole pages
    for (uint32_t e = kSlab * slab + threadIdx.x; e < end; e += 256) {
      if (e - item.first < item.fresh) {
        const uint32_t page = w.free[item.offset + e - item.first];
        if (!fork && e == item.first && item.rows) drop(p.references, item.from);
        p.references[page] = 1;
        entries[e] = page;
      } else if (fork) {
        const uint32_t page = e < shared ? theirs[e] : kHole;
        if (page < p.pages) atomicAdd(&p.references[page], 1u);
        entries[e] = page < p.pages ? page : kHole;
      }
    }
  }
  const uint32_t chunks = p.runs.first_chunk[p.runs.runs], waves = gridDim.x * 4;
  for (uint32_t task = blockIdx.x * 4 + (uint32_t)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6); task < requests * chunks;
       task += waves) {
    const Item item = w.items[task / chunks];
    if (item.rows) copy_chunk(p.runs, item.from, w.free[item.offset], item.rows, task % chunks);
  }
}

__global__ __launch_bounds__(256) void compact_count_kernel(PoolArgs p) {
  __shared__ uint32_t waves[4];
  const uint32_t first = blockIdx.x * kBlockPages + threadIdx.x * kPagesAThread;
  const uint32_t here = first < p.pages ? min((uint32_t)kPagesAThread, p.pages - first) : 0u;
  uint32_t all;
  (void)block_sums<256>(here - (uint32_t)__popc(free_bits(p, first)), waves, all);
  if (threadIdx.x == 0) workspace_of(p).counts[blockIdx.x] = all;
}

__global__ __launch_bounds__(256) void compact_plan_kernel(PoolArgs p) {
  __shared__ uint32_t waves[3][4];
  const Workspace w = workspace_of(p);
  const uint32_t first = blockIdx.x * kBlockPages + threadIdx.x * kPagesAThread;
  const uint32_t bits = free_bits(p, first);
  uint32_t mine = 0, sum = 0, live, earlier, all;
  for (uint32_t b = threadIdx.x; b < gridDim.x; b += 256) {
    const uint32_t n = w.counts[b];
    sum += n;
    if (b < blockIdx.x) mine += n;
  }
  (void)block_sums<256>(sum, waves[0], live);
  (void)block_sums<256>(mine, waves[1], earlier);
  const uint32_t here = first < p.pages ? min((uint32_t)kPagesAThread, p.pages - first) : 0u;
  uint32_t before = earlier + block_sums<256>(here - (uint32_t)__popc(bits), waves[2], all);   // pages in use before this one
  for (uint32_t i = 0; i < here; ++i) {
    const uint32_t page = first + i;
    const bool free = bits >> i & 1;
    if (page == live) {
      w.head->moves = live - before;   // as many in use from here on as places free before
      p.report[1] = live - before;
    }
    if (free && page < live) w.free[page - before] = page;
    if (!free && page >= live) {
      w.used[live - 1 - before] = page;
      w.rank[page] = live - 1 - before;
    }
    before += !free;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    p.report[0] = 0;
    p.report[2] = live;
    w.head->live = live;
    if (live == p.pages) {
      w.head->moves = 0;
      p.report[1] = 0;
    }
  }
}

__global__ __launch_bounds__(256) void compact_apply_kernel(PoolArgs p) {
  const Workspace w = workspace_of(p);
  const uint32_t moves = min(w.head->moves, p.pages), live = w.head->live;
  const uint32_t chunks = p.runs.first_chunk[p.runs.runs], waves = gridDim.x * 4;
  const uint32_t threads = gridDim.x * 256, thread = blockIdx.x * 256 + threadIdx.x;
  for (uint64_t task = blockIdx.x * 4 + (uint32_t)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
       task < (uint64_t)moves * chunks; task += waves) {
    const uint32_t move = (uint32_t)(task / chunks);
    copy_chunk(p.runs, w.used[move], w.free[move], p.page_rows, (uint32_t)(task % chunks));
  }
  for (uint32_t e = thread; e < p.sequences * p.pages_per_sequence; e += threads) {
    const uint32_t page = p.table[e];
    if (page < live || page >= p.pages) continue;
    const uint32_t rank = w.rank[page];   // of a page that no reference counts, anything
    if (rank < moves) p.table[e] = w.free[rank];
  }
  for (uint32_t i = thread; i < moves; i += threads) {
    p.references[w.free[i]] = p.references[w.used[i]];
    p.references[w.used[i]] = 0;
  }
}

__global__ __launch_bounds__(256) void page_copy_kernel(PageRuns p, const uint32_t *pairs, uint32_t count) {
  const uint32_t chunks = p.first_chunk[p.runs], waves = gridDim.x * 4;
  for (uint64_t task = blockIdx.x * 4 + (uint32_t)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
       task < (uint64_t)count * chunks; task += waves) {
    const uint32_t pair = (uint32_t)(task / chunks);
    const uint32_t from = pairs[2 * (size_t)pair], to = pairs[2 * (size_t)pair + 1];
    if (from < p.from_pages && to < p.to_pages) copy_chunk(p, from, to, p.page_rows, (uint32_t)(task % chunks));
  }
}

// Workgroups of copies: eight a compute unit, or fewer where there is less to copy.
constexpr uint64_t kCopyGroups = 2048;
uint32_t groups_for(uint64_t waves) { return (uint32_t)std::min(std::max<uint64_t>((waves + 3) / 4, 1), kCopyGroups); }
uint32_t slabs_of(const PoolArgs &p) { return (p.pages_per_sequence + kSlab - 1) / kSlab; }

}  // namespace

uint64_t pool_workspace_words(uint32_t pages) {
  return kHeadWords + kRequests * sizeof(Item) / 4 + 3 * uint64_t{pages} + (uint64_t{pages} + kBlockPages - 1) / kBlockPages;
}

hipError_t launch_pool_release(const PoolArgs &p, const uint32_t *rows, const uint32_t *keeps, uint32_t requests,
                               hipStream_t stream) {
  const uint32_t slabs = slabs_of(p);
  const uint32_t groups = (uint32_t)std::min<uint64_t>(uint64_t{requests} * slabs, kCopyGroups);
  hipLaunchKernelGGL(release_kernel, dim3(groups), dim3(256), 0, stream, p, rows, keeps, requests, slabs);
  return hipGetLastError();
}

hipError_t launch_pool_take(const PoolArgs &p, const uint32_t *rows, const uint32_t *more, const uint32_t *parents,
                            uint32_t requests, hipStream_t stream) {
  hipLaunchKernelGGL(take_plan_kernel, dim3(1), dim3(kPlanThreads), 0, stream, p, rows, more, parents, requests);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const uint32_t slabs = slabs_of(p);
  const uint64_t copies = uint64_t{requests} * p.runs.first_chunk[p.runs.runs];
  const uint32_t groups = std::max(groups_for(copies), (uint32_t)std::min<uint64_t>(uint64_t{requests} * slabs, kCopyGroups));
  hipLaunchKernelGGL(take_apply_kernel, dim3(groups), dim3(256), 0, stream, p, requests, slabs, parents ? 1u : 0u);
  return hipGetLastError();
}

hipError_t launch_pool_compact(const PoolArgs &p, hipStream_t stream) {
  const uint32_t blocks = (p.pages + kBlockPages - 1) / kBlockPages;
  hipLaunchKernelGGL(compact_count_kernel, dim3(blocks), dim3(256), 0, stream, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(compact_plan_kernel, dim3(blocks), dim3(256), 0, stream, p);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  // At most half of the pages move.
  const uint32_t groups = groups_for(uint64_t{p.pages} / 2 * p.runs.first_chunk[p.runs.runs] +
                                     uint64_t{p.sequences} * p.pages_per_sequence / 64);
  hipLaunchKernelGGL(compact_apply_kernel, dim3(groups), dim3(256), 0, stream, p);
  return hipGetLastError();
}

hipError_t launch_page_copy(const PageRuns &runs, const uint32_t *pairs, uint32_t count, hipStream_t stream) {
  hipLaunchKernelGGL(page_copy_kernel, dim3(groups_for(uint64_t{count} * runs.first_chunk[runs.runs])), dim3(256), 0, stream,
                     runs, pairs, count);
  return hipGetLastError();
}

}  // namespace sq::kern
