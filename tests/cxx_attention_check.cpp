// Host-only use of the C++ face's rope, cache and attention (include/splash_q4.hpp): sizes, plans and exceptions. Nothing
// here touches a GPU. Built and run by tests/test_attention_cpu.py.
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
  double frequencies[32];
  const float magnitude = Rope::frequencies({64, SQ_ROPE_HALF, SQ_ROPE_SCALING_NONE, 0, 1e4, 0, 0, 0}, frequencies);
  const KvShape shape{2, 64, 16, SQ_KV_INT8};
  const KvSize size = KvCache::size(shape, 10);
  const AttentionPlan plan = Attention({256}).plan({8, shape, 1, 0, 0.125f}, 4, 4, 1);
  std::printf("magnitude %g first %g; keys %llu scales %llu; tile %u waves %u workgroups %u\n", magnitude, frequencies[0],
              (unsigned long long)size.keys, (unsigned long long)size.key_scales, plan.tile_rows, plan.waves,
              plan.workgroups);
  const Rope rope(64, SQ_ROPE_HALF, magnitude, {});
  const KvCache cache(shape, 10, {}, {});
  const KvBatch batch{1, 1, 1, {}, {}, {}};
  const HeadRows rows{{}, 2, 128};
  const bool all = refused([&] { rope.add(nullptr, {}, 1, 64, rows, rows); }) &&
                   refused([&] { cache.addWrite(nullptr, batch, rows, rows, &rope); }) &&
                   refused([&] { cache.addRead(nullptr, batch, &rows, nullptr); }) &&
                   refused([&] { Attention::add(nullptr, {rows, rows, {}}, cache, batch, plan); });
  return all ? 0 : 1;
}
