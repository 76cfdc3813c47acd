// Host-only use of the C++ face's page pool, 4-bit cache and scored attention (include/splash_q4.hpp): sizes and exceptions.
// Nothing here touches a GPU. Built and run by tests/test_pages_cpu.py.
#include <cstdio>
#include <stdexcept>

#include "splash_q4.hpp"

using namespace splash_q4::ops;

template <typename F>
static bool refused(F &&f) {
  try {
    f();
  } catch (const std::invalid_argument &e) {
    std::printf("invalid_argument: %s\n", e.what());
    return true;
  }
  return false;
}

int main() {
  const KvShape shape{2, 64, 16, SQ_KV_E2M1};
  const KvSize size = KvCache::size(shape, 10);
  char *const at = reinterpret_cast<char *>(1 << 20);   // never read
  const KvCache cache(shape, 10, {at, size.keys}, {at, size.values}, {at, size.key_scales}, {at, size.value_scales});
  const KvPool pool(cache, 3, 4, {at, 40}, {at, 48}, {at, 12}, {at, 16});
  std::printf("workspace %llu keys %llu\n", (unsigned long long)pool.workspace(), (unsigned long long)size.keys);
  const AttentionPlan plan = Attention({256}).plan({8, shape, 1, 0, 0.125f}, 4, 4, 1);
  const KvBatch batch{1, 1, 1, {}, {}, {}};
  const HeadRows rows{{}, 8, 512};
  const AttentionScores scores{-1.0f, {}, {}, {}};
  const bool all = refused([&] { pool.addRelease(nullptr, {}, {}, 1); }) &&
                   refused([&] { pool.addGrow(nullptr, {}, {}, 1, {}); }) &&
                   refused([&] { pool.addFork(nullptr, {}, {}, 1, {}); }) && refused([&] { pool.addCompact(nullptr, {}); }) &&
                   refused([&] { KvPool::addCopy(nullptr, cache, cache, {}, 1); }) &&
                   refused([&] { Attention::add(nullptr, {rows, rows, {}}, cache, batch, plan, scores); }) &&
                   refused([&] { KvCache::size({2, 80, 16, SQ_KV_E2M1}, 1); });
  return all ? 0 : 1;
}
