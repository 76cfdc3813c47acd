// The pages of a cache, shared out, released, moved and copied (include/splash_q4.h).
#pragma once
#include "attention.hpp"

namespace sq::ops {

struct KvPool {
  KvCache cache;
  uint32_t sequences = 0, pagesPerSequence = 0;
  Buffer references, pageTable, lengths, report;
  void require() const;
  [[nodiscard]] uint64_t workspaceBytes() const;
  static void addRelease(hipStream_t graph, const KvPool &pool, Buffer rows, Buffer keeps, uint32_t requests);
  static void addGrow(hipStream_t graph, const KvPool &pool, Buffer rows, Buffer more, uint32_t requests, Buffer workspace);
  static void addFork(hipStream_t graph, const KvPool &pool, Buffer parents, Buffer children, uint32_t requests,
                      Buffer workspace);
  static void addCompact(hipStream_t graph, const KvPool &pool, Buffer workspace);
  // Pages from[pairs[2 i]] to to[pairs[2 i + 1]].
  static void addCopy(hipStream_t graph, const KvCache &from, const KvCache &to, Buffer pairs, uint32_t count);
};

}  // namespace sq::ops
