// Rotary positions, the paged key/value cache and attention over it, over HIP: the part of a layer between its q|k|v and
// output projections. As everywhere here, an add validates what the host can see and throws std::invalid_argument
// before anything is launched, then launches in order on the stream.
#pragma once
#include "ops.hpp"

namespace sq::ops {

// bf16 rows of attention heads: row r's head h from element r * rowStride + h * headDim on.
struct HeadRowsView {
  Buffer buffer;
  uint32_t heads = 0, rowStride = 0;
};

enum class RopeLayout : uint32_t { Half = SQ_ROPE_HALF, Interleaved = SQ_ROPE_INTERLEAVED };
enum class RopeScaling : uint32_t {
  None = SQ_ROPE_SCALING_NONE,
  Linear = SQ_ROPE_SCALING_LINEAR,
  Ntk = SQ_ROPE_SCALING_NTK,
  Yarn = SQ_ROPE_SCALING_YARN,
  Wavelength = SQ_ROPE_SCALING_WAVELENGTH,
};
struct RopeConfig {
  uint32_t rotaryDim = 0;
  RopeLayout layout = RopeLayout::Half;
  RopeScaling scaling = RopeScaling::None;
  uint32_t originalPositions = 0;
  double base = 0, factor = 1, low = 0, high = 0;
};
struct Rope {
  uint32_t rotaryDim = 0;
  RopeLayout layout = RopeLayout::Half;
  float magnitude = 1;
  Buffer frequencies;
  // Fills rotaryDim / 2 radians a position and returns the magnitude.
  static float frequenciesOf(const RopeConfig &config, double *frequencies);
  static void add(hipStream_t graph, const Rope &rope, Buffer positions, uint32_t rows, uint32_t headDim,
                  const HeadRowsView &input, const HeadRowsView &output);
};

// The most keys that a sequence's pages hold: a position, and a length that grows, stay inside 32 bits.
constexpr uint32_t kMaxKeys = 1u << 30;
enum class KvFormat : uint32_t { BFloat16 = SQ_KV_BF16, Int8 = SQ_KV_INT8, E4m3 = SQ_KV_E4M3, E2m1 = SQ_KV_E2M1 };
struct KvSize {
  uint64_t keys = 0, values = 0, keyScales = 0, valueScales = 0;
};
struct KvShape {
  uint32_t kvHeads = 0, headDim = 0, pageRows = 0;
  KvFormat format = KvFormat::BFloat16;
  void require() const;
  [[nodiscard]] KvSize bytes(uint32_t pages) const;
  [[nodiscard]] bool operator==(const KvShape &) const = default;
};
struct KvBatch {
  uint32_t sequences = 0, rows = 0, pagesPerSequence = 0;
  Buffer rowStarts, lengths, pageTable;
};
struct KvCache {
  KvShape shape;
  uint32_t pages = 0;
  Buffer keys, values, keyScales, valueScales;
  void require() const;
  void require(const KvBatch &batch) const;
  static void addWrite(hipStream_t graph, const KvCache &cache, const KvBatch &batch, const HeadRowsView &keys,
                       const HeadRowsView &values, const Rope *rope, const HeadRowsView *queries,
                       const HeadRowsView *rotated);
  static void addRead(hipStream_t graph, const KvCache &cache, const KvBatch &batch, const HeadRowsView *keys,
                      const HeadRowsView *values);
};

struct AttentionShape {
  uint32_t heads = 0;
  KvShape kv;
  bool causal = true;
  uint32_t window = 0;
  float scale = 1;
  void require() const;
  [[nodiscard]] uint32_t group() const noexcept { return heads / kv.kvHeads; }
  [[nodiscard]] float exponentScale() const;   // the scale's magnitude as the kernels' powers of two take it
};
struct AttentionPlan {
  AttentionShape shape;
  uint32_t sequences = 0, rows = 0, chunkRows = 0, tileRows = 0, waves = 0, workgroups = 0;
  uint64_t partials = 0;   // bytes of workspace
};
// What a scored call does to scores, and which keys it hides or shows (splash_q4.h); none of it: absent.
struct AttentionScores {
  float cap = 0;
  Buffer slopes, begins, prefixes;
  [[nodiscard]] bool none() const noexcept { return cap == 0 && !slopes.ptr && !begins.ptr && !prefixes.ptr; }
};
struct Attention {
  static AttentionPlan plan(const DeviceCapabilities &device, const AttentionShape &shape, uint32_t sequences,
                            uint32_t rows, uint32_t chunkRows);
  static void add(hipStream_t graph, const HeadRowsView &query, const HeadRowsView &output, Buffer partials,
                  const KvCache &cache, const KvBatch &batch, const AttentionPlan &plan,
                  const AttentionScores &scores = {});
};

}  // namespace sq::ops
