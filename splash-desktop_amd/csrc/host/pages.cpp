#include "pages.hpp"

#include "../kernels/pages.hpp"
#include "stream.hpp"

namespace sq::ops {
namespace {

constexpr uint32_t kMaxPages = 1u << 28, kMaxEntries = 1u << 28, kMaxTableRows = 1u << 20;

void requireWords(Buffer b, uint64_t words, const char *what) {
  requireBytes(b, words * 4, what);
  if (!aligned(b, 4)) throw std::invalid_argument(std::string(what) + " are 4-byte aligned");
}

kern::PageRuns runsOf(const KvCache &from, const KvCache &to) {
  const KvShape &s = from.shape;
  const KvSize page = s.bytes(1);
  const uint64_t heads = uint64_t{s.kvHeads} * s.pageRows, bytes[4] = {page.keys, page.values, page.keyScales, page.valueScales};
  const Buffer source[4] = {from.keys, from.values, from.keyScales, from.valueScales},
               target[4] = {to.keys, to.values, to.keyScales, to.valueScales};
  kern::PageRuns out{};
  for (uint32_t i = 0; i < 4 && bytes[i]; ++i) {
    out.from[i] = source[i].as<const uint8_t>();
    out.to[i] = target[i].as<uint8_t>();
    out.bytes[i] = uint32_t(bytes[i]);
    out.row_bytes[i] = uint32_t(bytes[i] / heads);
    out.first_chunk[i + 1] = out.first_chunk[i] + uint32_t((bytes[i] + kern::kPageChunk - 1) / kern::kPageChunk);
    out.runs = i + 1;
  }
  out.page_rows = s.pageRows;
  out.from_pages = from.pages;
  out.to_pages = to.pages;
  return out;
}

kern::PoolArgs poolArgs(const KvPool &pool, Buffer workspace) {
  return {runsOf(pool.cache, pool.cache), pool.references.as<uint32_t>(), pool.pageTable.as<uint32_t>(),
          pool.lengths.as<uint32_t>(),    pool.report.as<uint32_t>(),     pool.cache.pages,
          pool.sequences,                 pool.pagesPerSequence,          pool.cache.shape.pageRows,
          workspace.as<uint32_t>()};
}

void requireRequests(Buffer a, const char *first, Buffer b, const char *second, uint32_t requests) {
  if (requests > SQ_KV_MAX_SEQUENCES) throw std::invalid_argument("a call takes at most 1024 requests");
  requireWords(a, requests, first);
  requireWords(b, requests, second);
}

void requireWorkspace(const KvPool &pool, Buffer workspace) {
  requireBytes(workspace, pool.workspaceBytes(), "pool workspace");
  if (!aligned(workspace, 16)) throw std::invalid_argument("a pool's workspace is 16-byte aligned");
}

}  // namespace

void KvPool::require() const {
  cache.require();
  if (cache.pages > kMaxPages) throw std::invalid_argument("a pool has at most 2^28 pages");
  if (!sequences || sequences > kMaxTableRows) throw std::invalid_argument("a pool has 1 to 2^20 sequences");
  if (!pagesPerSequence || uint64_t{sequences} * pagesPerSequence > kMaxEntries)
    throw std::invalid_argument("a pool's table has entries, at most 2^28");
  if (uint64_t{pagesPerSequence} * cache.shape.pageRows > kMaxKeys)
    throw std::invalid_argument("a pool's sequences have pages for at most 2^30 keys");
  requireWords(references, cache.pages, "page references");
  requireWords(pageTable, uint64_t{sequences} * pagesPerSequence, "page table entries");
  requireWords(lengths, sequences, "sequence lengths");
  requireWords(report, 4, "pool report words");
}

uint64_t KvPool::workspaceBytes() const { return kern::pool_workspace_words(cache.pages) * 4; }

void KvPool::addRelease(hipStream_t graph, const KvPool &pool, Buffer rows, Buffer keeps, uint32_t requests) {
  pool.require();
  requireRequests(rows, "rows to release", keeps, "keys to keep", requests);
  if (!requests) return;
  const OnStreamDevice on(graph);
  launched(kern::launch_pool_release(poolArgs(pool, {}), rows.as<const uint32_t>(), keeps.as<const uint32_t>(), requests,
                                     graph),
           "pool release");
}

void KvPool::addGrow(hipStream_t graph, const KvPool &pool, Buffer rows, Buffer more, uint32_t requests, Buffer workspace) {
  pool.require();
  requireRequests(rows, "rows to grow", more, "keys to grow by", requests);
  requireWorkspace(pool, workspace);
  if (!requests) return;
  const OnStreamDevice on(graph);
  launched(kern::launch_pool_take(poolArgs(pool, workspace), rows.as<const uint32_t>(), more.as<const uint32_t>(), nullptr,
                                  requests, graph),
           "pool grow");
}

void KvPool::addFork(hipStream_t graph, const KvPool &pool, Buffer parents, Buffer children, uint32_t requests,
                     Buffer workspace) {
  pool.require();
  requireRequests(parents, "parents", children, "children", requests);
  requireWorkspace(pool, workspace);
  if (!requests) return;
  const OnStreamDevice on(graph);
  launched(kern::launch_pool_take(poolArgs(pool, workspace), children.as<const uint32_t>(), nullptr,
                                  parents.as<const uint32_t>(), requests, graph),
           "pool fork");
}

void KvPool::addCompact(hipStream_t graph, const KvPool &pool, Buffer workspace) {
  pool.require();
  requireWorkspace(pool, workspace);
  const OnStreamDevice on(graph);
  launched(kern::launch_pool_compact(poolArgs(pool, workspace), graph), "pool compact");
}

void KvPool::addCopy(hipStream_t graph, const KvCache &from, const KvCache &to, Buffer pairs, uint32_t count) {
  from.require();
  to.require();
  if (!(from.shape == to.shape)) throw std::invalid_argument("pages are copied between caches of one shape");
  if (count > kMaxPages) throw std::invalid_argument("a call copies at most 2^28 pages");
  if (!count) return;
  requireBytes(pairs, uint64_t{count} * 8, "page pairs");
  if (!aligned(pairs, 8)) throw std::invalid_argument("page pairs are 8-byte aligned");
  const OnStreamDevice on(graph);
  launched(kern::launch_page_copy(runsOf(from, to), pairs.as<const uint32_t>(), count, graph), "page copy");
}

}  // namespace sq::ops
