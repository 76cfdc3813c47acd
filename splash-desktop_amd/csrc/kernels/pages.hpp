// The pages of a cache (pages.hip): what the host hands over. It has checked the views' sizes; the kernels check what the
// requests, references, table and lengths hold.
#pragma once
#include "kernels.hpp"

namespace sq::kern {

// A page as up to four runs of memory (keys, values, their scales): run r of page p is the bytes [r] bytes from from[r] + p *
// bytes[r] on, of kv_heads times page_rows rows of row_bytes[r] each.
struct PageRuns {
  const uint8_t *from[4];
  uint8_t *to[4];
  uint32_t bytes[4], row_bytes[4];
  uint32_t runs, page_rows, from_pages, to_pages;
  uint32_t first_chunk[5];   // of each run, in chunks of kPageChunk bytes; the last: all of a page's
};
constexpr uint32_t kPageChunk = 4096;   // what a wave copies at a time: four vectors a lane

// A pool's books. The workspace's parts: see pages.hip.
struct PoolArgs {
  PageRuns runs;
  uint32_t *references, *table, *lengths, *report;
  uint32_t pages, sequences, pages_per_sequence, page_rows;
  uint32_t *workspace;
};
// Words of workspace that a pool of `pages` pages takes.
uint64_t pool_workspace_words(uint32_t pages);

hipError_t launch_pool_release(const PoolArgs &pool, const uint32_t *rows, const uint32_t *keeps, uint32_t requests,
                               hipStream_t stream);
// more: the keys that each sequence grows by; null: a fork, rows the children and parents theirs.
hipError_t launch_pool_take(const PoolArgs &pool, const uint32_t *rows, const uint32_t *more, const uint32_t *parents,
                            uint32_t requests, hipStream_t stream);
hipError_t launch_pool_compact(const PoolArgs &pool, hipStream_t stream);
hipError_t launch_page_copy(const PageRuns &runs, const uint32_t *pairs, uint32_t count, hipStream_t stream);

}  // namespace sq::kern
