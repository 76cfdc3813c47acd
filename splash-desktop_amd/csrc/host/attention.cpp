#include "attention.hpp"

#include <cmath>
#include <numbers>

#include "../kernels/kernels.hpp"
#include "stream.hpp"

namespace sq::ops {
namespace {

// The most rows of a batch: with kMaxKeys, sums of lengths over every unit of a batch stay far inside 64 bits.
constexpr uint32_t kMaxRows = 1u << 20, kMaxHeads = 1024, kMaxUnits = 65536;

void requireHeadDim(uint32_t dim) {
  if (!dim || dim > 256 || dim % 16)
    throw std::invalid_argument("attention heads have a multiple of 16 values, at most 256");
}

kern::HeadRows headRows(const HeadRowsView &v, uint32_t rows, uint32_t dim, const char *what) {
  const std::string name(what);
  if (!v.heads || v.heads > kMaxHeads * kern::kAttendMaxGroup)
    throw std::invalid_argument(name + " have heads, at most 65536");
  if (v.rowStride < uint64_t{v.heads} * dim || v.rowStride % 8)
    throw std::invalid_argument(name + "' row stride holds their heads and is a multiple of 8");
  if (!v.buffer) throw std::invalid_argument(name + " are null");
  requireBytes(v.buffer, rowBytes(rows, v.rowStride, uint64_t{v.heads} * dim, 2), what);
  if (!aligned(v.buffer, 16)) throw std::invalid_argument(name + " are 16-byte aligned");
  return {v.buffer.as<uint16_t>(), v.heads, v.rowStride};
}

kern::RopeArgs ropeArgs(const Rope &rope, uint32_t headDim) {
  if (!rope.rotaryDim || rope.rotaryDim % 2 || rope.rotaryDim > headDim)
    throw std::invalid_argument("a rope rotates an even number of a head's values");
  if (rope.layout != RopeLayout::Half && rope.layout != RopeLayout::Interleaved)
    throw std::invalid_argument("unknown rope layout");
  if (!std::isfinite(rope.magnitude)) throw std::invalid_argument("a rope's magnitude is finite");
  requireBytes(rope.frequencies, uint64_t{rope.rotaryDim / 2} * 8, "rope frequencies");
  if (!aligned(rope.frequencies, 8)) throw std::invalid_argument("rope frequencies are 8-byte aligned");
  return {rope.frequencies.as<const double>(), rope.rotaryDim / 2, rope.layout == RopeLayout::Interleaved,
          rope.magnitude};
}

// Rotating in place is one tensor under one stride.
void requireInPlace(const HeadRowsView &input, const HeadRowsView &output, const char *what) {
  if (input.buffer.ptr == output.buffer.ptr && input.rowStride != output.rowStride)
    throw std::invalid_argument(std::string(what) + " in place keeps its row stride");
}

kern::KvArgs kvArgs(const KvCache &cache, const KvBatch &batch) {
  cache.require(batch);
  uint32_t shift = 0;
  while (1u << shift < cache.shape.pageRows) ++shift;
  return {cache.keys.as<uint8_t>(),
          cache.values.as<uint8_t>(),
          cache.keyScales.as<float>(),
          cache.valueScales.as<float>(),
          batch.rowStarts.as<const uint32_t>(),
          batch.lengths.as<const uint32_t>(),
          batch.pageTable.as<const uint32_t>(),
          batch.sequences,
          batch.rows,
          batch.pagesPerSequence,
          cache.pages,
          shift,
          cache.shape.kvHeads,
          cache.shape.headDim,
          uint32_t(cache.shape.format)};
}

}  // namespace

float Rope::frequenciesOf(const RopeConfig &c, double *frequencies) {
  if (!c.rotaryDim || c.rotaryDim % 2 || c.rotaryDim > 256)
    throw std::invalid_argument("a rope rotates an even number of values, at most 256");
  if (c.layout != RopeLayout::Half && c.layout != RopeLayout::Interleaved)
    throw std::invalid_argument("unknown rope layout");
  if (!std::isfinite(c.base) || c.base <= 1) throw std::invalid_argument("a rope's base is a number above 1");
  const bool scaled = c.scaling != RopeScaling::None;
  if (scaled && (!std::isfinite(c.factor) || c.factor < 1))
    throw std::invalid_argument("a rope's scaling factor is a number of at least 1");
  const double d = c.rotaryDim, pi = std::numbers::pi, original = c.originalPositions;
  double base = c.base, low = c.low, high = c.high;
  switch (c.scaling) {
    case RopeScaling::None:
    case RopeScaling::Linear: break;
    case RopeScaling::Ntk:
      if (c.rotaryDim == 2) throw std::invalid_argument("a rope of one pair has no base to scale");
      base *= std::pow(c.factor, d / (d - 2));
      break;
    case RopeScaling::Yarn:
    case RopeScaling::Wavelength:
      if (!c.originalPositions) throw std::invalid_argument("this rope scaling takes the original positions");
      if (high == 0) high = c.scaling == RopeScaling::Yarn ? 32 : 4;
      if (low == 0) low = 1;
      if (!std::isfinite(low) || !std::isfinite(high) || low <= 0 || high <= low)
        throw std::invalid_argument("a rope's high bound is above its low one, and both above 0");
      break;
    default: throw std::invalid_argument("unknown rope scaling");
  }
  // The pair that turns `turns` times over the original positions, as a real number.
  const auto turning = [&](double turns) { return d * std::log(original / (turns * 2 * pi)) / (2 * std::log(base)); };
  double from = 0, to = 1;
  if (c.scaling == RopeScaling::Yarn) {
    from = std::max(std::floor(turning(high)), 0.0);
    to = std::min(std::ceil(turning(low)), d - 1);
  }
  for (uint32_t i = 0; i < c.rotaryDim / 2; ++i) {
    const double f = std::pow(base, -2.0 * i / d);
    if (c.scaling == RopeScaling::Linear) {
      frequencies[i] = f / c.factor;
    } else if (c.scaling == RopeScaling::Yarn) {
      const double ramp = std::clamp((i - from) / std::max(to - from, 0.001), 0.0, 1.0);
      frequencies[i] = f * (1 - ramp) + f / c.factor * ramp;
    } else if (c.scaling == RopeScaling::Wavelength) {
      const double turns = original * f / (2 * pi), t = std::clamp((turns - low) / (high - low), 0.0, 1.0);
      frequencies[i] = (1 - t) * f / c.factor + t * f;
    } else {
      frequencies[i] = f;
    }
  }
  return c.scaling == RopeScaling::Yarn ? float(0.1 * std::log(c.factor) + 1) : 1.0f;
}

void Rope::add(hipStream_t graph, const Rope &rope, Buffer positions, uint32_t rows, uint32_t headDim,
               const HeadRowsView &input, const HeadRowsView &output) {
  requireHeadDim(headDim);
  const kern::RopeArgs args = ropeArgs(rope, headDim);
  if (rows > kMaxRows) throw std::invalid_argument("a batch has at most 2^20 rows");
  if (!rows) return;
  requireBytes(positions, uint64_t{rows} * 4, "rope positions");
  if (!aligned(positions, 4)) throw std::invalid_argument("rope positions are 4-byte aligned");
  if (input.heads != output.heads) throw std::invalid_argument("a rope's input and output have the same heads");
  const kern::HeadRows in = headRows(input, rows, headDim, "rope input"), out = headRows(output, rows, headDim, "rope output");
  requireInPlace(input, output, "a rope");
  const OnStreamDevice on(graph);
  launched(kern::launch_rope(args, positions.as<const uint32_t>(), rows, headDim, in, out, graph), "rope");
}

void KvShape::require() const {
  requireHeadDim(headDim);
  if (!kvHeads || kvHeads > kMaxHeads) throw std::invalid_argument("a cache has 1 to 1024 key heads");
  if (pageRows < 16 || pageRows > 1024 || (pageRows & (pageRows - 1)))
    throw std::invalid_argument("a cache's pages have a power of two of rows, 16 to 1024");
  if (format != KvFormat::BFloat16 && format != KvFormat::Int8 && format != KvFormat::E4m3 && format != KvFormat::E2m1)
    throw std::invalid_argument("unknown cache format");
  if (format == KvFormat::E2m1 && headDim % 32)
    throw std::invalid_argument("heads of a 4-bit cache have a multiple of 32 values");
}

KvSize KvShape::bytes(uint32_t pages) const {
  require();
  if (!pages || pages == ~0u) throw std::invalid_argument("a cache has pages");
  const uint64_t rows = uint64_t{pages} * kvHeads * pageRows;
  if (format == KvFormat::BFloat16) return {rows * headDim * 2, rows * headDim * 2, 0, 0};
  if (format == KvFormat::E2m1) {
    const uint64_t scales = rows * (headDim <= 64 ? 2 : headDim <= 128 ? 4 : 8);
    return {rows * headDim / 2, rows * headDim / 2, scales, scales};
  }
  return {rows * headDim, rows * headDim, rows * 4, rows * 4};
}

void KvCache::require() const {
  const KvSize size = shape.bytes(pages);
  requireBytes(keys, size.keys, "cache keys");
  requireBytes(values, size.values, "cache values");
  requireBytes(keyScales, size.keyScales, "cache key scales");
  requireBytes(valueScales, size.valueScales, "cache value scales");
  if (!aligned(keys, 16) || !aligned(values, 16) || !aligned(keyScales, 16) || !aligned(valueScales, 16))
    throw std::invalid_argument("a cache's buffers are 16-byte aligned");
}

void KvCache::require(const KvBatch &batch) const {
  require();
  if (!batch.sequences || batch.sequences > SQ_KV_MAX_SEQUENCES)
    throw std::invalid_argument("a batch has 1 to 1024 sequences");
  if (batch.rows > kMaxRows) throw std::invalid_argument("a batch has at most 2^20 rows");
  if (!batch.pagesPerSequence || uint64_t{batch.pagesPerSequence} * shape.pageRows > kMaxKeys)
    throw std::invalid_argument("a sequence has pages, for at most 2^30 keys");
  requireBytes(batch.rowStarts, (uint64_t{batch.sequences} + 1) * 4, "row starts");
  requireBytes(batch.lengths, uint64_t{batch.sequences} * 4, "sequence lengths");
  requireBytes(batch.pageTable, uint64_t{batch.sequences} * batch.pagesPerSequence * 4, "page table");
  if (!aligned(batch.rowStarts, 4) || !aligned(batch.lengths, 4) || !aligned(batch.pageTable, 4))
    throw std::invalid_argument("row starts, lengths and page table are 4-byte aligned");
}

void KvCache::addWrite(hipStream_t graph, const KvCache &cache, const KvBatch &batch, const HeadRowsView &keys,
                       const HeadRowsView &values, const Rope *rope, const HeadRowsView *queries,
                       const HeadRowsView *rotated) {
  const kern::KvArgs args = kvArgs(cache, batch);
  const uint32_t dim = cache.shape.headDim;
  if (!queries != !rotated || (queries && !rope))
    throw std::invalid_argument("queries are rotated with a rope, into rows of their own or in place");
  kern::RopeArgs turn{};
  if (rope) turn = ropeArgs(*rope, dim);
  if (!batch.rows) return;
  if (keys.heads != cache.shape.kvHeads || values.heads != cache.shape.kvHeads)
    throw std::invalid_argument("the cache's key heads are the rows'");
  const kern::HeadRows k = headRows(keys, batch.rows, dim, "key rows"), v = headRows(values, batch.rows, dim, "value rows");
  kern::HeadRows q{}, r{};
  if (queries) {
    if (queries->heads != rotated->heads) throw std::invalid_argument("queries and rotated queries have the same heads");
    q = headRows(*queries, batch.rows, dim, "query rows");
    r = headRows(*rotated, batch.rows, dim, "rotated query rows");
    requireInPlace(*queries, *rotated, "a rope");
  }
  const OnStreamDevice on(graph);
  launched(kern::launch_kv_write(args, k, v, turn, q, r, graph), "cache write");
}

void KvCache::addRead(hipStream_t graph, const KvCache &cache, const KvBatch &batch, const HeadRowsView *keys,
                      const HeadRowsView *values) {
  const kern::KvArgs args = kvArgs(cache, batch);
  if (!batch.rows || (!keys && !values)) return;
  kern::HeadRows k{}, v{};
  for (const HeadRowsView *rows : {keys, values})
    if (rows && rows->heads != cache.shape.kvHeads) throw std::invalid_argument("the cache's key heads are the rows'");
  if (keys) k = headRows(*keys, batch.rows, cache.shape.headDim, "key rows");
  if (values) v = headRows(*values, batch.rows, cache.shape.headDim, "value rows");
  const OnStreamDevice on(graph);
  launched(kern::launch_kv_read(args, k, v, graph), "cache read");
}

float AttentionShape::exponentScale() const { return float(std::fabs(double(scale)) * std::numbers::log2e); }

void AttentionShape::require() const {
  kv.require();
  if (!heads || heads % kv.kvHeads || heads / kv.kvHeads > kern::kAttendMaxGroup)
    throw std::invalid_argument("attention heads are a multiple of the key heads, at most 64 times as many");
  if (window && !causal) throw std::invalid_argument("a window takes causal attention");
  if (!std::isfinite(scale)) throw std::invalid_argument("an attention scale is finite");
  if (!std::isfinite(exponentScale())) throw std::invalid_argument("an attention scale is finite times log2 e too");
}

AttentionPlan Attention::plan(const DeviceCapabilities &device, const AttentionShape &shape, uint32_t sequences,
                              uint32_t rows, uint32_t chunkRows) {
  shape.require();
  if (!sequences || sequences > SQ_KV_MAX_SEQUENCES)
    throw std::invalid_argument("a batch has 1 to 1024 sequences");
  if (!rows || rows > kMaxRows) throw std::invalid_argument("an attention plan takes 1 to 2^20 rows");
  if (!chunkRows || chunkRows > rows) throw std::invalid_argument("a sequence's new rows are 1 to the plan's rows");
  if (device.computeUnits > kMaxUnits) throw std::invalid_argument("an attention plan takes at most 65536 compute units");
  AttentionPlan out{shape, sequences, rows, chunkRows};
  // The smallest tile of few rows that holds a sequence's new rows with their query heads, so that their keys are read
  // once; past the largest of those, the wide tile.
  const uint64_t packed = uint64_t{chunkRows} * shape.group();
  out.tileRows = kern::kAttendWideRows;
  for (uint32_t few = kern::attend_few_rows(shape.kv.headDim); few >= 16 && few >= packed; few /= 2) out.tileRows = few;
  const uint32_t format = uint32_t(shape.kv.format);
  const uint32_t units = ((device.computeUnits ? device.computeUnits : 256) + 7) / 8 * 8;
  // Few sequences: workgroups of twice the waves, one a compute unit, halve a unit's parts and its waves' turns.
  const bool few = out.tileRows != kern::kAttendWideRows &&
                   kern::attend_rows_resident(out.tileRows, shape.kv.headDim, format) > 1 &&
                   uint64_t{sequences} * shape.kv.kvHeads * 2 <= units;
  out.waves = few ? 8 : 4;
  out.workgroups = units * kern::attend_resident(out.tileRows, out.waves, shape.kv.headDim, format);
  out.partials = kern::attend_partials(out.tileRows, shape.kv.headDim, out.workgroups);
  return out;
}

void Attention::add(hipStream_t graph, const HeadRowsView &query, const HeadRowsView &output, Buffer partials,
                    const KvCache &cache, const KvBatch &batch, const AttentionPlan &plan, const AttentionScores &scores) {
  const kern::KvArgs kv = kvArgs(cache, batch);
  const AttentionShape &shape = plan.shape;
  if (!(cache.shape == shape.kv)) throw std::invalid_argument("the attention plan is another cache's");
  if (batch.sequences > plan.sequences || batch.rows > plan.rows)
    throw std::invalid_argument("the batch is larger than its attention plan");
  // The lengths of every sequence's units end to end (attend.hpp), row starts that overlap included, are counted in 52 bits.
  const uint64_t keys = uint64_t{batch.pagesPerSequence} * cache.shape.pageRows;
  if (double(batch.sequences) * (batch.rows + 1.0) * (double(keys) + 4096) * shape.kv.kvHeads > 0x1p52)
    throw std::invalid_argument("an attention batch's sequences, rows, keys and key heads multiply to less than 2^52");
  if (!batch.rows) return;
  if (query.heads != shape.heads || output.heads != shape.heads)
    throw std::invalid_argument("query and output rows have the attention's heads");
  const kern::HeadRows q = headRows(query, batch.rows, shape.kv.headDim, "query rows"),
                       o = headRows(output, batch.rows, shape.kv.headDim, "output rows");
  requireInPlace(query, output, "attention");
  requireBytes(partials, plan.partials, "attention partials");
  if (!aligned(partials, 16)) throw std::invalid_argument("attention partials are 16-byte aligned");
  if (!std::isfinite(scores.cap) || scores.cap < 0) throw std::invalid_argument("a score cap is finite, and not negative");
  const float exponent = shape.scale == 0 ? 1.0f : shape.exponentScale();
  const double log2e = std::numbers::log2e, cap = scores.cap;
  if (scores.cap != 0 && (!std::isfinite(float(2 * exponent / cap)) || !std::isfinite(float(2 / cap)) ||
                          !std::isfinite(float(cap * log2e)) || float(cap) < 0x1p-100f))
    throw std::invalid_argument("an attention scale over its score cap, and the cap times log2 e, are finite");
  const auto optional = [&](Buffer b, uint64_t words, const char *what) {
    if (!b.ptr) return;
    requireBytes(b, words * 4, what);
    if (!aligned(b, 4)) throw std::invalid_argument(std::string(what) + " are 4-byte aligned");
  };
  optional(scores.slopes, shape.heads, "attention slopes");
  optional(scores.begins, batch.sequences, "sequence begins");
  optional(scores.prefixes, batch.sequences, "sequence prefixes");
  if (scores.prefixes.ptr && !shape.causal) throw std::invalid_argument("prefixes take causal attention");
  const kern::AttendArgs args{kv,
                              q.rows,
                              o.rows,
                              q.stride,
                              o.stride,
                              shape.group(),
                              shape.causal,
                              shape.window,
                              exponent,
                              shape.scale == 0 ? 0u : ~0u,
                              shape.scale < 0 ? 0x80008000u : 0u,
                              partials.as<float>(),
                              partials.as<uint8_t>() + plan.partials - (plan.workgroups + 1) * kern::kAttendNoteBytes,
                              plan.workgroups};
  // A batch of few units, none longer than a workgroup takes at least, is cut nowhere (attend.hpp), and leaves no parts.
  const uint64_t units = (batch.rows / (plan.tileRows / shape.group()) + batch.sequences) * uint64_t{shape.kv.kvHeads};
  const bool whole = plan.tileRows != kern::kAttendWideRows && batch.sequences <= 64 && units * 4 <= plan.workgroups &&
                     keys + 384 <= kern::attend_least(shape.kv.headDim, args.kv.format, !scores.none());
  const OnStreamDevice on(graph);
  const bool wide = plan.tileRows == kern::kAttendWideRows;
  if (scores.none()) {
    launched(wide ? kern::launch_attend_tile(args, graph)
                  : kern::launch_attend_rows(plan.tileRows, plan.waves, args, graph),
             "attention");
  } else {
    const kern::ScoredArgs scored{args,
                                  scores.slopes.as<const float>(),
                                  scores.begins.as<const uint32_t>(),
                                  scores.prefixes.as<const uint32_t>(),
                                  float(cap * log2e),
                                  cap != 0 ? float(2 / cap) : 0.0f,
                                  cap != 0 ? float(1 / (cap * log2e)) : 0.0f,
                                  cap > kern::kCapWithScores};
    // Powers up to the seventh of the score's share of the cap are normal numbers.
    const double share = exponent / (cap * log2e);
    const bool capped = cap != 0 && cap <= kern::kCapWithScores && !scores.slopes.ptr && share > 0x1p-15 && share < 0x1p15;
    launched(!wide ? kern::launch_attend_rows_scored(plan.tileRows, plan.waves, scored, graph)
             : capped ? kern::launch_attend_tile_capped({scored}, graph)
                      : kern::launch_attend_tile_scored(scored, graph),
             "scored attention");
  }
  if (!whole) launched(kern::launch_attend_join(plan.tileRows, units * 4 <= plan.workgroups, args, graph), "attention join");
}

}  // namespace sq::ops
