/*
 * splash_q4 — MI355X (gfx950) quantized matmul path: bf16 activations x 4-bit group-quantized weights (and the
 * adjacent 5-, 6- and 8-bit formats), fp32 accumulation. C ABI over the reference's splash::ops::Linear /
 * splash::ops::MoE call surface.
 *
 * Conventions
 *  - Buffers are device-pointer views {ptr, bytes} (the reference's MetalBuffer views). The caller owns every
 *    buffer; nothing here allocates device memory.
 *  - A "graph" is a hipStream_t passed as void*: an add call validates everything, then launches in order on it.
 *    NULL is the default stream.
 *  - Every function returns SQ_OK or an error code; nothing is launched when it fails. sq_last_error() holds the
 *    thread's message for the last failure (the text of the reference's std::invalid_argument where it has one).
 *  - Format ids, plane layouts and parameter blocks are the reference's (runtime/metal/abi/QuantFormat.h, Gguf.h,
 *    MoE.h): Q4_K (0), Q5_K (3), Q6_K (4), Q8_0 (6), MLX affine 4-bit in groups of 32, 64 and 128 (25, 26, 27)
 *    and MLX affine 8-bit in groups of 64 (35), in every entry point.
 *  - Split scratch (partials, counters) is reused serially on one stream: counters are zero at allocation and every
 *    split or stream dispatch returns them to zero; two streams never share one scratch.
 * Reference interfaces each entry point replaces are named in its comment (paths under the reference checkout).
 */
#ifndef SPLASH_Q4_H
#define SPLASH_Q4_H
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define SQ_OK 0
#define SQ_INVALID_ARGUMENT 1 /* the reference throws std::invalid_argument */
#define SQ_RUNTIME_ERROR 2    /* a HIP launch or runtime failure */

#define SQ_FMT_Q4K 0u
#define SQ_FMT_Q5K 3u
#define SQ_FMT_Q6K 4u
#define SQ_FMT_Q80 6u
#define SQ_FMT_AF4G32 25u
#define SQ_FMT_AF4G64 26u
#define SQ_FMT_AF4G128 27u
#define SQ_FMT_AF8G64 35u
/* Float rows (QuantizedSegment::rows, Weights.hpp:67-81): F32 rows carry the format id kFloat32, BF16 rows
 * GGUF_FMT_BF16; the float projection multiplies them unrounded in fp32. */
#define SQ_FMT_BF16 41u
#define SQ_FLOAT32_ROWS 0xFFFFFFFFu

/* enum values match the reference's enum class order (Linear.hpp:67-80, Weights.hpp:62) */
#define SQ_PHASE_PREFILL 0u
#define SQ_PHASE_DECODE 1u
#define SQ_EPILOGUE_NONE 0u
#define SQ_EPILOGUE_RESIDUAL 1u
#define SQ_EPILOGUE_GATE_UP 2u
#define SQ_EPILOGUE_UP_WITH_GATE 3u
#define SQ_TILE_STAGED 0u   /* LinearTile::GgufStaged: the decode tile */
#define SQ_TILE_PREFILL 1u  /* LinearTile::GgufPrefill */
#define SQ_TILE_REGISTER 2u /* LinearTile::GgufRegister: refused (Apple9 only) */
#define SQ_OUTPUT_BF16 0u
#define SQ_OUTPUT_F32 1u
#define SQ_MAX_SEGMENTS 3u

typedef struct sq_buffer {
  void *ptr;
  uint64_t bytes;
} sq_buffer;

/* QuantizedSegment, planes layout (runtime/ops/Weights.hpp:79-121). */
typedef struct sq_segment {
  sq_buffer plane0, plane1, meta;
  uint32_t output_size, input_size, column_offset, format_id;
} sq_segment;

/* Projection (runtime/ops/Weights.hpp:131-188): segments tile the leading output columns in order. */
typedef struct sq_projection {
  uint32_t output_size, input_size;
  uint32_t segment_count;
  uint32_t destination; /* SQ_OUTPUT_* */
  sq_segment segments[SQ_MAX_SEGMENTS];
} sq_projection;

/* LinearWorkload / LinearConfig / LinearPlan (runtime/ops/Linear.hpp:93-214). */
typedef struct sq_linear_workload {
  uint32_t output_size, input_size, rows, phase, epilogue;
} sq_linear_workload;
typedef struct sq_linear_config {
  uint32_t tile, splits, spread, one_gate_up_pass, sixteen_rows;
} sq_linear_config;
typedef struct sq_linear_plan {
  sq_linear_workload workload;
  sq_linear_config config;
  uint32_t destination;
  uint32_t storage_rows;
} sq_linear_plan;

/* LinearScratch / LinearScratchSize / LinearBuffers (runtime/ops/Linear.hpp:125-162,216-226). A decode plan's
 * partials hold its K splits' fp32 sums; a prefill plan's, where its tiles' K is halved (projections of 64 to 128
 * tiles of 256 rows by 256 columns, K a multiple of 512; reserved there also where the narrow tile runs instead and
 * leaves them untouched), the two halves' fp32 sums [2][rows][N], and where its
 * tiles number more than one round over the 256 compute units (K a multiple of 256), the fp32 sums of the last
 * round's stream pieces (128 MiB: two 256 x 256 tiles of sums for each of 256 workgroups) with a 4-byte counter
 * a stream tile. */
typedef struct sq_linear_scratch_size {
  uint64_t input, sums, partials, counters, rotated;
} sq_linear_scratch_size;
typedef struct sq_linear_scratch {
  sq_buffer input, sums, partials, counters, rotated;
} sq_linear_scratch;
/* LinearInput (Linear.hpp:166-169): the activation layout a plan reads. TABLE16 is the reference's Apple9 register
 * tile table, which no plan here reads (a producer asked for it is refused); HALF_ROWS is this build's prefill
 * table: the rows in fp16, scaled by a power of two per row and stored group by group in the prefill tile's read
 * order, in scratch.input, with the powers (fp32) in scratch.sums. */
#define SQ_LINEAR_INPUT_PLAIN 0u
#define SQ_LINEAR_INPUT_TABLE16 1u
#define SQ_LINEAR_INPUT_HALF_ROWS 2u
/* PreparedInput (Linear.hpp:184-190): the scratch table currently holds `source` in `layout`. */
typedef struct sq_prepared_input {
  sq_buffer source;
  uint32_t layout;
} sq_prepared_input;
typedef struct sq_linear_buffers {
  sq_buffer input, output, residual, gate_scratch;
  sq_linear_scratch scratch;
  /* What the scratch table holds (LinearBuffers::prepared, Linear.hpp:216-226): a plan that reads a table prepares
   * one unless this describes its input (same pointer and bytes). All zero: nothing. */
  sq_prepared_input prepared;
} sq_linear_buffers;

/* DeviceCapabilities, as far as the MI355X policy reads it (the decode split law, and the column tile's 16-column
 * workgroups for dispatches of few tiles, which compute the same bits as 64-column ones); compute_units 0 takes 256.
 * The prefill tile's schedule is a function of the shape alone, for the MI355X's 256 compute units. */
typedef struct sq_device {
  uint32_t compute_units;
} sq_device;

const char *sq_last_error(void);
/* Library version string. */
const char *sq_version(void);

/* ---- planning (host only; no GPU needed) ---- */

/* Linear::plan(LinearWorkload) and Linear::plan(workload, projection, gate) (Linear.cpp:151-164).
 * projection and gate may be NULL. */
int sq_linear_plan_for(const sq_device *device, const sq_linear_workload *workload, const sq_projection *projection,
                       const sq_projection *gate, sq_linear_plan *out);
/* static Linear::plan(workload, config, destination) (Linear.cpp:155-157). */
int sq_linear_plan_config(const sq_linear_workload *workload, const sq_linear_config *config, uint32_t destination,
                          sq_linear_plan *out);
/* Linear::decodePlan (Linear.cpp:166-169): rows = lanes * 8. */
int sq_linear_decode_plan(const sq_device *device, const sq_projection *projection, uint32_t lanes, uint32_t epilogue,
                          const sq_projection *gate, sq_linear_plan *out);
/* Linear::prefillPlan (Linear.cpp:170-172). */
int sq_linear_prefill_plan(const sq_device *device, const sq_projection *projection, uint32_t rows, uint32_t epilogue,
                           sq_linear_plan *out);
/* LinearPlan::scratchSize and gateScratchBytes (LinearGguf.cpp:432-453, Linear.cpp:123-129). */
int sq_linear_plan_scratch(const sq_linear_plan *plan, sq_linear_scratch_size *out, uint64_t *gate_scratch_bytes);
/* Linear::decodeScratchSize / prefillScratchSize (Linear.cpp:174-196). */
int sq_linear_decode_scratch_size(const sq_device *device, uint32_t output_size, uint32_t input_size,
                                  sq_linear_scratch_size *out);
int sq_linear_prefill_scratch_size(const sq_device *device, uint32_t output_size, uint32_t input_size,
                                   sq_linear_scratch_size *out);
/* Linear::decodeStorageRows (Linear.hpp:254-257; Linear.cpp:145-149): the rows of storage a decode step of `rows`
 * rows (1..32) binds for a projection of output_size x input_size, the storage_rows of its decode plans, which every
 * epilogue shares. The engine sizes its decode activation and output buffers with it (QwenTarget.cpp:125,
 * DFlashDraft.cpp:239). */
int sq_linear_decode_storage_rows(const sq_device *device, uint32_t rows, uint32_t output_size, uint32_t input_size,
                                  uint32_t *storage_rows);
/* Linear::ggufFloatTile (Linear.hpp:273-276; LinearGguf.cpp:837-844): the SQ_FLOAT_TILE_* a float projection of `rows`
 * rows into output_size columns of rows in format_id takes on this device. MI355X's policy: the matrix-core tile
 * from 64 rows on, the lane chains below. ExecutionPlans picks the MoE router's tile with it (ExecutionPlans.cpp:62),
 * as sq_moe_config_for does. */
int sq_linear_float_tile(const sq_device *device, uint32_t rows, uint32_t output_size, uint32_t format_id,
                         uint32_t *tile);
/* requireSegmentPlanes (LinearGguf.cpp:905-923): SQ_OK when the planes hold every tile of the segment. */
int sq_require_segment_planes(const sq_segment *segment, const char *what, uint32_t plane_inputs);

/* ---- dispatch ---- */

/* Linear::add (Linear.cpp:203-232; LinearGguf.cpp:579-802): the plan's projection of buffers->input. A decode of a
 * projection of up to SQ_MAX_SEGMENTS segments runs them in one dispatch whatever their formats (gguf_decode_fused);
 * a prefill runs one dispatch per format. A prefill plan's input, output, residual, gate scratch, scratch table and
 * partials are 16-byte aligned and its row scales (scratch sums) 4-byte aligned. Whether a prefill halves its tiles'
 * K, or runs its narrow tile (K in eight slices), depends on the chunk's rows as well as the shape (a 4096-input,
 * 14336-output projection runs narrow up to 256 rows and halves from 257 to 512), so a row's output bits may differ
 * between chunks of different row counts; each lies within the row's fp64 interval. The same holds for the tiles past
 * a prefill's whole rounds over the compute units, whose K runs in pieces on several workgroups (their sums add in K
 * order whatever order the pieces finish in, so a chunk's bits repeat from run to run). A decode row's bits depend only
 * on the shape, the segments' formats and the tile kind its rows run (1..4 rows, 5..16, 17..32). */
int sq_linear_add(void *graph, const sq_linear_buffers *buffers, const sq_projection *projection,
                  const sq_linear_plan *plan, const sq_projection *gate);
/* Linear::add with its result: *prepared (may be NULL) receives what the scratch table describes after the
 * dispatch (the PreparedInput Linear::add returns, Linear.cpp:222-231). */
int sq_linear_add_prepared(void *graph, const sq_linear_buffers *buffers, const sq_projection *projection,
                           const sq_linear_plan *plan, const sq_projection *gate, sq_prepared_input *prepared);
/* No counterpart in the reference: Linear::add for callers that cannot allocate device memory (code under HIP graph
 * capture, tight serving loops, harnesses that forbid allocation). The same plans and kernels as sq_linear_add, but
 * the split partials and counters, the prefill table and its row scales and a two-pass gate/up pair's gate scratch
 * come from a static array of SQ_STATIC_SCRATCH_BYTES per GPU inside the library (held from its first use on that GPU
 * to the end of the process); buffers->scratch is ignored and buffers->prepared must be empty. buffers->gate_scratch
 * is read only by an UP_WITH_GATE plan, as the gate operand its epilogue multiplies in (the caller's gate projection
 * output, checked to hold the plan's rows as sq_linear_add checks it), and ignored by every other plan. A plan whose
 * scratch exceeds the array is refused (SQ_INVALID_ARGUMENT). Nothing is allocated: it launches a counter-clearing
 * kernel, then the plan's dispatches. Every call on one GPU shares that GPU's array, so calls that overlap on one GPU
 * (two streams, two threads) race; calls in one stream's order do not. */
#define SQ_STATIC_SCRATCH_BYTES (16u << 20)
int sq_linear_add_static(void *graph, const sq_linear_buffers *buffers, const sq_projection *projection,
                         const sq_linear_plan *plan, const sq_projection *gate);
/* LinearPlan::input (Linear.hpp:199-202): the layout the producer of the plan's input may write (SQ_LINEAR_INPUT_*):
 * HALF_ROWS for a prefill plan, PLAIN otherwise. */
int sq_linear_plan_input(const sq_linear_plan *plan, uint32_t *layout);

/* ---- producers either side of the path ---- */

/* NormWeights (Normalization.hpp:14-23): the per-channel multipliers of an RMS norm, bf16 (float32 0) or F32. */
typedef struct sq_norm_weights {
  sq_buffer buffer;
  uint32_t float32;
} sq_norm_weights;
/* Normalization::addRms (Normalization.hpp:35-39; Normalization.cpp:16-38): output = bf16((x rsqrt(sum x^2 / width +
 * 1e-6)) w) for `rows` rows of `width` bf16 inputs. With layout SQ_LINEAR_INPUT_HALF_ROWS it also writes the prefill
 * table of `output` into *scratch (input: rows * width * 2 bytes, sums: rows * 4), the bits the prefill's own
 * preparation would write; *prepared (may be NULL) receives what the scratch then describes. scratch may be NULL
 * for PLAIN. width % 64 == 0; input, output, weights and the table 16-byte aligned. */
int sq_norm_add_rms(void *graph, sq_buffer input, const sq_norm_weights *weight, sq_buffer output, uint32_t width,
                    uint32_t rows, const sq_linear_scratch *scratch, uint32_t layout, sq_prepared_input *prepared);
/* addGgufFloat (Linear.hpp:34-40; LinearGguf.cpp:847-853) for a float segment (format SQ_FLOAT32_ROWS or
 * SQ_FMT_BF16, its rows in plane0): output[r][out_offset + n] = sum_k input[r][k] W[n][k] for r < rows, products and
 * sums in fp32, into an fp32 or bf16 (destination SQ_OUTPUT_*) destination of out_stride columns, on `tile`
 * (SQ_FLOAT_TILE_*, sq_linear_float_tile's choice or the caller's). input_size % 4 == 0; the matrix-core tile takes
 * input_size a multiple of 256 (the reference's neural accelerator tile: 32), else SQ_INVALID_ARGUMENT. Both tiles lie
 * within (input_size / 64 + 8) 2^-24 sum |x w| of the exact sum. */
int sq_float_add(void *graph, sq_buffer input, const sq_segment *weights, sq_buffer output, uint32_t rows,
                 uint32_t out_stride, uint32_t out_offset, uint32_t destination, uint32_t tile);
/* Linear::addPrefill / addPrefillResidual / addPrefillUpWithGate (Linear.cpp:234-256). */
int sq_linear_add_prefill(const sq_device *device, void *graph, sq_buffer input, const sq_projection *projection,
                          sq_buffer output, uint32_t rows, const sq_linear_scratch *scratch);
int sq_linear_add_prefill_residual(const sq_device *device, void *graph, sq_buffer input,
                                   const sq_projection *projection, sq_buffer residual, sq_buffer output,
                                   uint32_t rows, const sq_linear_scratch *scratch);
int sq_linear_add_prefill_up_with_gate(const sq_device *device, void *graph, sq_buffer input, const sq_projection *up,
                                       sq_buffer gate_scratch, sq_buffer output, uint32_t rows,
                                       const sq_linear_scratch *scratch);
/* Linear::addPrefillSwiGlu (Linear.cpp:244-250): output = residual + down(silu(gate x) * up x). */
int sq_linear_add_prefill_swiglu(const sq_device *device, void *graph, const sq_projection *gate,
                                 const sq_projection *up, const sq_projection *down, sq_buffer normalized,
                                 sq_buffer gate_scratch, sq_buffer intermediate, const sq_linear_scratch *scratch,
                                 sq_buffer residual, sq_buffer output, uint32_t rows);

/* ---- weight preparation (load time) ---- */

/* The gguf_repack dispatch (kernels/shared/gguf_repack.metal:232-238; GgufRepack.h:10-18): native rows in src
 * (src_row_bytes apart) into dst: plane0 at 0, meta at dst_meta, and Q5_K's and Q6_K's high bits at dst_plane1
 * (unused by the other formats).
 * params points at the reference's 24-byte GgufRepackParams {rows, input_size, fmt, src_row_bytes, dst_plane1,
 * dst_meta}. */
int sq_gguf_repack(void *graph, sq_buffer src, sq_buffer dst, const void *params);
/* MLX tensors (mlx.core.quantize affine, bits 4 or 8: uint32 codes [rows][K * bits / 32], bf16 scales and biases
 * [rows][K/group]) straight into planes: the loader's native-block build (model/GgufPreparation.cpp:141-193) and
 * the repack in one dispatch. */
int sq_mlx_repack(void *graph, uint32_t format_id, uint32_t rows, uint32_t input_size, sq_buffer weight,
                  sq_buffer scales, sq_buffer biases, sq_buffer plane0, sq_buffer meta);
/* Every weight of a segment dequantised: fp32 fma(q, s, z) (Q6_K s (q - 32), Q8_0 d v) and its fp16 rounding (the
 * staged tiles' weight), [N][K] each; either output may have a NULL ptr (reference test kernel
 * gguf_test_dequant_<fmt>, dev/tests/engine/gguf_dequant_test.metal:5-21). */
int sq_dequant(void *graph, const sq_segment *segment, sq_buffer values_f32, sq_buffer values_f16);

/* ---- measurement ---- */

/* No counterpart in the reference: a read-only stream of src (whole 16-byte vectors) by `workgroups` workgroups of
 * `threads` threads, thread g folding vectors g, g + S, g + 2S, ... (S = workgroups * threads). A workgroup's word of
 * sink is written only when one of its threads' folds equals the marker word 0x9E3779B9 (the thread's index + 1), so
 * no store is timed. The HBM floor the GEMV is measured against (bench.py). */
int sq_diag_stream_read(void *graph, sq_buffer src, sq_buffer sink, uint32_t workgroups, uint32_t threads);

/* No counterpart in the reference: `workgroups` workgroups of four waves (at most waves_per_simd, 1 or 2, resident a
 * SIMD), each wave running `iterations` x 8 independent 16x16x32 f16 MFMAs (16384 flops each) on operands held in
 * registers. The sustained MFMA ceiling the prefill GEMM is measured against (bench.py). */
int sq_diag_mfma_peak(void *graph, sq_buffer sink, uint32_t workgroups, uint32_t waves_per_simd, uint32_t iterations);

/* ---- MoE (runtime/ops/MoE.hpp:387-423) ---- */

/* MoeRouter (MoE.hpp:22-28): Softmax weights the top_k routes by the softmax of their scores, SigmoidNormalized by
 * each one's sigmoid over the sum of theirs. */
#define SQ_MOE_ROUTER_SOFTMAX 0u
#define SQ_MOE_ROUTER_SIGMOID_NORMALIZED 1u

/* MoeShape (MoE.hpp:54-102). The reference compiles two routings, (Softmax, 1 shared slice, gated) and
 * (SigmoidNormalized, 2 shared slices, ungated) (kCompiledMoeRoutings, MoE.hpp:34-46); this build also takes
 * (Softmax, no shared expert). The shared expert is shared_slices experts every row visits after its routed ones,
 * each of the routed experts' intermediate width; gated, slice weights are sigmoid(x . g) of the block's fp32
 * scalar gate g, else 1. */
typedef struct sq_moe_shape {
  uint32_t hidden_size, experts, experts_per_token, expert_intermediate_size;
  uint32_t expert_format; /* the format of most routed expert weights (each projection runs in its own) */
  uint32_t router;        /* SQ_MOE_ROUTER_* */
  uint32_t shared_slices; /* 0, 1 or 2 */
  uint32_t shared_gated;  /* 1: slice weights sigmoid(x . g); 0: 1 */
} sq_moe_shape;
typedef struct sq_moe_workspace {
  uint64_t selected_experts, routing_weights, tile_descriptors, tile_count, grouped_routes, route_rows,
      grouped_input, expert_intermediate, expert_output;
} sq_moe_workspace;
/* MoeExpertTile (MoE.hpp:284): the rows of an expert tile. */
#define SQ_MOE_EXPERT_TILE_M8 8u
#define SQ_MOE_EXPERT_TILE_M32 32u
/* MoeGgufTile (MoE.hpp:297): Staged runs here; Register is the reference's Apple9 tile, which a plan refuses. */
#define SQ_MOE_GGUF_TILE_STAGED 0u
#define SQ_MOE_GGUF_TILE_REGISTER 1u
/* FloatTile (Linear.hpp:29-33): a float projection's tile (the MoE router's among them). On MI355X SIMDGROUP runs
 * the lane chains (a wave of four rows by four columns, K over the lanes) and NEURAL_ACCELERATOR the matrix-core tile
 * (fp32 16x16x4 MFMA, 32 rows by 32 columns a workgroup, K a multiple of 256); their results lie within one fp32
 * bound. */
#define SQ_FLOAT_TILE_SIMDGROUP 0u
#define SQ_FLOAT_TILE_NEURAL_ACCELERATOR 1u
/* MoeConfig (MoE.hpp:333-346): the device's policy for a MoE plan. cpu_bf16_experts opts the reference's streamed
 * CPU experts in; its experts here are never streamed, so the flag selects nothing, as the reference's MoE::add
 * takes the GPU route for weights that are not streamed (MoE.cpp:225-245). */
typedef struct sq_moe_config {
  uint32_t expert_tile; /* SQ_MOE_EXPERT_TILE_* */
  uint32_t gguf_tile;   /* SQ_MOE_GGUF_TILE_* */
  uint32_t router_tile; /* SQ_FLOAT_TILE_* */
  uint32_t cpu_bf16_experts;
} sq_moe_config;
typedef struct sq_moe_plan {
  sq_moe_shape shape;
  uint32_t rows, phase, tile_rows, maximum_tiles;
  sq_moe_config config;
  sq_moe_workspace workspace;
} sq_moe_plan;
/* BlockExpertProjection (MoE.hpp:111-148). routed: `slots` experts' planes in one segment of slots * N rows.
 * shared: the shared slices' planes in their order, slice s's rows s * N on (a shared down of shared_slices * I
 * inputs laid out as shared_slices column windows of I inputs, window s rows s * H on). Each of the six segments
 * has a format of its own (MoE.cpp:27-62): a gate and up of different formats run as a gate pass and an up pass
 * whose epilogue reads the gate's bf16 output from expert_output (MoE.cpp:154-173), the same bits as one pass.
 * shared_scalar_gate: the block's fp32 gate [hidden] for a gated shared expert. The shared views are ignored
 * without shared slices. */
typedef struct sq_moe_weights {
  sq_segment gate, up, down;
  sq_buffer slot_table; /* uint32 per expert: its slot */
  uint32_t slots;
  sq_segment shared_gate, shared_up, shared_down;
  sq_buffer shared_scalar_gate;
  /* BlockMoeWeights::router (MoE.hpp:133): F32 (SQ_FLOAT32_ROWS) or BF16 rows [experts][hidden] in plane0. The
   * routing projects the input onto it into the router scores (MoE::addRoutes, MoE.cpp:527-543). With plane0 NULL
   * the routing reads scores the caller wrote (below). */
  sq_segment router;
} sq_moe_weights;
/* MoeScratch (MoE.hpp:225-245), sized by the plan's workspace. As in the reference, the router's fp32 scores live in
 * grouped_input, a row of the shape's router width (256 expert slots, or 512 past 256 experts:
 * sq_moe_router_width) per row; a block without router rows takes the caller's scores from there. As the reference's
 * gather does, the routed work (sq_moe_add_routed) then overwrites them, with the block's input rows in the expert
 * tiles' read order; the gate/up pass reads those through the grouped routes. Every buffer here, and the block's
 * input, output and residual, is 16-byte aligned. */
typedef struct sq_moe_scratch {
  sq_buffer selected_experts, routing_weights, tile_descriptors, tile_count, grouped_routes, route_rows,
      grouped_input, expert_intermediate, expert_output;
} sq_moe_scratch;
/* MoeBuffers (MoE.hpp:375-385). residual may be a NULL view (zeros). verify_rows: a verify step's live rows per lane
 * of 8 rows, a uint32 per lane (ceil(rows / 8) of them); routed routes of rows past their lane's count are grouped
 * into no tile, their route_rows are ~0u and the combine adds nothing for them, so such a row's output is its
 * residual plus its shared slices' routes (moe_group_routes_verified, moe.metal:164-173,196-236, 496). A NULL view:
 * every row routes. Decode plans only. */
typedef struct sq_moe_buffers {
  sq_buffer input, residual, output;
  sq_moe_scratch scratch;
  sq_buffer verify_rows;
} sq_moe_buffers;

/* The policy a plan takes when its config is NULL (ExecutionPlans::moeConfig, ExecutionPlans.cpp:56-65): Staged tiles,
 * 8-row tiles in decode and, in prefill, 8-row tiles while rows * top_k <= experts, else 32 (moeGgufPrefillTile,
 * MoE.hpp:321-330). phase is SQ_PHASE_*. */
int sq_moe_config_for(const sq_moe_shape *shape, uint32_t rows, uint32_t phase, sq_moe_config *out);
/* MoE::prefillPlan(shape, rows, config) (MoE.cpp:561-565): rows 1..2048. config NULL takes sq_moe_config_for's. */
int sq_moe_prefill_plan(const sq_moe_shape *shape, uint32_t rows, const sq_moe_config *config, sq_moe_plan *out);
/* MoE::decodePlan(shape, lanes, config) (MoE.cpp:567-571): lanes 1..4 of 8 rows each, 8-row tiles. */
int sq_moe_decode_plan(const sq_moe_shape *shape, uint32_t lanes, const sq_moe_config *config, sq_moe_plan *out);
/* No counterpart in the reference: a decode plan of any 1..32 rows (the reference's decode rows are lanes * 8). */
int sq_moe_decode_rows_plan(const sq_moe_shape *shape, uint32_t rows, sq_moe_plan *out);
/* MoeShape::routerWidth (MoE.hpp:94-96): the fp32 scores a row of the router scores holds. */
uint32_t sq_moe_router_width(const sq_moe_shape *shape);
/* MoE::add = addRouting then addRouted (MoE.cpp:225-525). */
int sq_moe_add(void *graph, const sq_moe_buffers *buffers, const sq_moe_weights *weights, const sq_moe_plan *plan);
int sq_moe_add_routing(void *graph, const sq_moe_buffers *buffers, const sq_moe_weights *weights,
                       const sq_moe_plan *plan);
int sq_moe_add_routed(void *graph, const sq_moe_buffers *buffers, const sq_moe_weights *weights,
                      const sq_moe_plan *plan);
/* MoE::addRoutes (MoE.hpp:403-411; MoE.cpp:527-543): the routing of `rows` rows (1..2048) of `input` (bf16
 * [rows][hidden]) with no plan and no grouping, into caller buffers. With router rows (router non-NULL, plane0 set:
 * F32 or BF16 [experts][hidden]) it first projects the input onto them into `scores` on router_tile (SQ_FLOAT_TILE_*);
 * otherwise it reads the fp32 scores the caller wrote there. scores: rows of sq_moe_router_width(shape) fp32 slots;
 * selected (uint32) and routing_weights (fp32): experts_per_token + shared_slices per row, the top-k experts then
 * the shared slices, as sq_moe_add_routing writes them. shared_scalar_gate (fp32 [hidden]) is read only for a gated
 * shared expert. input, scores and shared_scalar_gate are 16-byte aligned. */
int sq_moe_add_routes(void *graph, sq_buffer input, const sq_segment *router, sq_buffer shared_scalar_gate,
                      sq_buffer scores, sq_buffer selected, sq_buffer routing_weights, uint32_t rows,
                      const sq_moe_shape *shape, uint32_t router_tile);
/* MoE::addExpertLoad (MoE.hpp:411-420, MoE.cpp:553-558; kernel moe_expert_load, gguf_repack.metal:239-257): the
 * gate, up and down projections of up to `jobs` streamed experts repacked into their slots of `arena`. Job j's
 * projection z takes its native rows (row_bytes apart) from staging + sources[3 j + z] (bytes) on, and writes them
 * as sq_gguf_repack does into plane i of slot slots[j]: arena + planes[i] + slots[j] * slot_bytes[i] (plane0, plane1,
 * meta). params is the reference's 192-byte MoeExpertLoadParams: three 64-byte MoeExpertLoadProjection
 * {format, rows, columns, row_bytes, planes[3], slot_bytes[3]} (rows 0: no projection). slots: jobs uint32; sources:
 * 3 jobs uint64 (8-byte aligned); grid: three uint32 workgroup counts (x, y, z) that an earlier dispatch may write,
 * the reference's indirect grid. The launch covers (sq_moe_expert_load_groups(params), jobs, 3) workgroups of 256
 * threads, and those past grid's counts do nothing. A job whose rows or slot planes would lie outside staging or
 * arena writes nothing. */
typedef struct sq_moe_expert_load_projection {
  uint32_t format_id, rows, columns, row_bytes;
  uint64_t planes[3];     /* plane0, plane1, meta: byte offsets in the arena */
  uint64_t slot_bytes[3]; /* bytes a slot in each */
} sq_moe_expert_load_projection;
typedef struct sq_moe_expert_load_params {
  sq_moe_expert_load_projection projections[3]; /* gate, up, down */
} sq_moe_expert_load_params;
int sq_moe_expert_load(void *graph, sq_buffer staging, sq_buffer arena, sq_buffer slots, sq_buffer sources,
                       const sq_moe_expert_load_params *params, uint32_t jobs, sq_buffer grid);
/* MoE::expertLoadGroups (MoE.cpp:545-551): the workgroups that repack one job's largest projection (0 without
 * params). */
uint32_t sq_moe_expert_load_groups(const sq_moe_expert_load_params *params);

/* ---- rotary positions, a paged key/value cache, and attention over it ---- */

/* What lies between a layer's q|k|v projection and its output projection. A batch of new rows (one token, a verify
 * lane, a chunk of a prompt; of up to SQ_KV_MAX_SEQUENCES sequences at once) is rotated, its keys and values are
 * written into the cache's pages, and its queries attend to every key of their sequence. Every entry point validates
 * what the host can see, launches on the stream's own device, allocates nothing, and may be captured into a graph.
 * What only the device can see (row starts, lengths, page ids) is bounds-checked in the kernels: nothing outside the
 * views is read or written whatever they hold. */

/* bf16 rows of attention heads: row r's head h is the head_dim values from element r * row_stride + h * head_dim on. A
 * fused projection's query, key and value columns are three of these over one tensor. row_stride is at least heads *
 * head_dim and a multiple of 8; the buffer is 16-byte aligned and holds the last row's heads. */
typedef struct sq_head_rows {
  sq_buffer buffer;
  uint32_t heads, row_stride;
} sq_head_rows;

/* Rotary positions. The first rotary_dim values of a head are pairs, (i, i + rotary_dim / 2) in the HALF layout and
 * (2i, 2i + 1) in the INTERLEAVED one, i < rotary_dim / 2; a row at position p turns pair i by the angle p *
 * frequencies[i] and scales it by magnitude; the values from rotary_dim on are copied. frequencies: doubles, radians a
 * position, on the device, 8-byte aligned. Angles are reduced in 64 bits, so far positions keep their phase. */
#define SQ_ROPE_HALF 0u
#define SQ_ROPE_INTERLEAVED 1u
typedef struct sq_rope {
  uint32_t rotary_dim, layout;
  float magnitude;
  sq_buffer frequencies;
} sq_rope;
/* The frequencies f_i = base^(-2 i / rotary_dim), scaled for contexts past original_positions:
 *  LINEAR      f_i / factor.
 *  NTK         base * factor^(rotary_dim / (rotary_dim - 2)) in the place of base (rotary_dim > 2).
 *  YARN        f_i (1 - r) + (f_i / factor) r, r the ramp 0..1 from the pair that turns `high` times over
 *              original_positions to the one that turns `low` times (rounded outwards); magnitude 0.1 ln(factor) + 1.
 *              high 0 takes 32 and low 0 takes 1.
 *  WAVELENGTH  with w_i = 2 pi / f_i: f_i below original_positions / high, f_i / factor above original_positions /
 *              low, and between them (1 - t) f_i / factor + t f_i, t = (original_positions / w_i - low) / (high - low).
 *              high 0 takes 4 and low 0 takes 1.
 * magnitude is 1 but for YARN. */
#define SQ_ROPE_SCALING_NONE 0u
#define SQ_ROPE_SCALING_LINEAR 1u
#define SQ_ROPE_SCALING_NTK 2u
#define SQ_ROPE_SCALING_YARN 3u
#define SQ_ROPE_SCALING_WAVELENGTH 4u
typedef struct sq_rope_config {
  uint32_t rotary_dim, layout, scaling, original_positions;
  double base, factor, low, high;
} sq_rope_config;
/* Host only: fills frequencies[0 .. rotary_dim / 2) (host memory; the caller uploads them once) and *magnitude. */
int sq_rope_frequencies(const sq_rope_config *config, double *frequencies, float *magnitude);
/* output = input rotated, row r at positions[r] (uint32 [rows], on the device). input and output have the same heads;
 * output may be input itself (same pointer and stride), and otherwise shares no element with it. head_dim is a multiple
 * of 16 up to 256; rotary_dim is even and at most head_dim. rows may be 0. */
int sq_rope_add(void *graph, const sq_rope *rope, sq_buffer positions, uint32_t rows, uint32_t head_dim,
                const sq_head_rows *input, const sq_head_rows *output);

/* The cache: `pages` pages of page_rows tokens (a power of two, 16..1024), keys and values each [pages][kv_heads]
 * [page_rows][head_dim] (head_dim a multiple of 16 up to 256), 16-byte aligned. The 8-bit formats hold a code a value
 * and one fp32 scale a token and head ([pages][kv_heads][page_rows], keys and values apart); a code stands for code *
 * scale. INT8: scale = m / 127, code = x 127 / m rounded to the nearest even, m the head row's largest magnitude. E4M3:
 * scale = m / 448, code = x 448 / m rounded to the nearest value of that type. A head row of zeros has scale 0; one with
 * an infinity or NaN has a NaN scale and zero codes, so all of it reads back as NaN; no code is E4M3's NaN. BF16 pages hold the rows as they
 * are, and have no scales. */
#define SQ_KV_BF16 0u
#define SQ_KV_INT8 1u
#define SQ_KV_E4M3 2u
/* Four bits (no format has the id 3): e2m1 codes, magnitudes 0, 0.5, 1, 1.5, 2, 3, 4 and 6 under a sign, two a byte, the first
 * in its low half, so keys and values are each [pages][kv_heads][page_rows][head_dim / 2] bytes; head_dim is a multiple of 32.
 * A group of 32 values has a scale byte b for 2^(b - 127): the least (2 to 252) under which the group's largest magnitude is
 * at most 7. The code is that of x / scale rounded to the nearest, ties to the even code, 6 above it; a value is code * scale,
 * exactly a bf16. A group with an infinity or NaN has byte 255 and zero codes, so all of it reads back as NaN. No write makes
 * bytes 253 and 254, under which values past bf16's range are infinite. Scales: [pages][kv_heads][page_rows] times 2, 4 or 8
 * bytes (head_dim up to 64, 128, 256) in the order of the groups; bytes past head_dim / 32 are 2 as written and not read. */
#define SQ_KV_E2M1 4u
#define SQ_KV_MAX_SEQUENCES 1024u
typedef struct sq_kv_shape {
  uint32_t kv_heads, head_dim, page_rows, format;
} sq_kv_shape;
typedef struct sq_kv_cache {
  sq_kv_shape shape;
  uint32_t pages;
  sq_buffer keys, values, key_scales, value_scales;
} sq_kv_cache;
typedef struct sq_kv_size {
  uint64_t keys, values, key_scales, value_scales; /* bytes of each buffer; the scales' are 0 for BF16 */
} sq_kv_size;
int sq_kv_cache_size(const sq_kv_shape *shape, uint32_t pages, sq_kv_size *out);
/* The new rows of a batch, packed one sequence after the other: sequence s has rows row_starts[s] .. row_starts[s + 1] -
 * 1 (uint32 [sequences + 1], not decreasing), and lengths[s] keys (uint32) with them, so that its row i of n sits at
 * position lengths[s] - n + i; token t of it is row t % page_rows of page page_table[s * pages_per_sequence + t /
 * page_rows] (uint32). rows is the rows that the head rows hold: rows from row_starts[sequences] on belong to no
 * sequence and are left as they were. A length past pages_per_sequence * page_rows counts as that many. A table entry
 * that names no page of the cache is a hole: nothing is written there, it reads back as zeros, and attention does not
 * see its keys. Rows before position 0 (more rows than keys) are not written and read back as zeros. */
typedef struct sq_kv_batch {
  uint32_t sequences, rows, pages_per_sequence;
  sq_buffer row_starts, lengths, page_table;
} sq_kv_batch;
/* Writes the batch's key and value rows into their pages. With a rope the keys are rotated at their positions (and
 * rounded to bf16, as sq_rope_add rounds them) before they are stored; with queries and rotated as well (both NULL
 * otherwise), the query rows are rotated into `rotated`, which may be the queries themselves, in the same launch. keys,
 * values and queries are left as they are. Two rows of one call must not name one token's place: pages that sequences
 * share are written by neither. */
int sq_kv_add_write(void *graph, const sq_kv_cache *cache, const sq_kv_batch *batch, const sq_head_rows *keys,
                    const sq_head_rows *values, const sq_rope *rope, const sq_head_rows *queries,
                    const sq_head_rows *rotated);
/* The way back: the batch's rows out of their pages as bf16 (code * scale rounded once). keys or values may be NULL. */
int sq_kv_add_read(void *graph, const sq_kv_cache *cache, const sq_kv_batch *batch, const sq_head_rows *keys,
                   const sq_head_rows *values);

/* Attention: for each row of the batch at position p and query head h, over the keys j of its sequence that it sees,
 *   output = sum_j e^(scale q.k_j - max) v_j / sum_j e^(scale q.k_j - max)
 * with key/value head h / (heads / kv_heads). causal: a row sees the keys up to its own position, and with a window
 * (0: none) only the last `window` of them, its own among them; not causal: every key of its sequence. A row that sees
 * no key gets zeros. (Of a row all of whose scores are minus infinity the formula says nothing: zeros, or NaN.) Keys that a
 * row does not see do not touch its output, whatever they hold. scale is finite, and its product with log2 e is. heads is a
 * multiple of kv_heads, at most 64 times as many. Scores, maxima, sums and the output's accumulators are fp32; the weights e^...
 * enter the matrix units as two bf16 each in tiles of 16 or 32 rows, rounded to one in those of 128, 8-bit codes exactly. */
typedef struct sq_attention_shape {
  uint32_t heads;
  sq_kv_shape kv;
  uint32_t causal, window;
  float scale;
} sq_attention_shape;
/* A plan for batches of at most `sequences` sequences and `rows` rows; chunk_rows, the most new rows that one sequence
 * usually has, picks the tile (any batch is computed right whatever it is). One tile serves all of a call's sequences: a
 * chunk of a prompt and single tokens mostly take less time in one call than in two (1024 rows at 4096 keys beside 32 tokens
 * of 3000 to 16000, bf16 heads of 128: 249 us for 111 + 184; of 200 to 2000: 130 for 109 + 54), but more with long contexts
 * in 8 bits (int8: 265 for 126 + 116; 150 for 124 + 41 with the short ones). tile_rows: the rows times query heads of one
 * key head that a tile holds (16, 32 or 128); waves: of a workgroup. partials: the bytes of workspace, which may hold
 * anything before a call; one workspace serves one stream at a time. */
typedef struct sq_attention_plan {
  sq_attention_shape shape;
  uint32_t sequences, rows, chunk_rows, tile_rows, waves, workgroups;
  uint64_t partials;
} sq_attention_plan;
typedef struct sq_attention_buffers {
  sq_head_rows query, output; /* output may be the query itself, and otherwise shares no element with it */
  sq_buffer partials;         /* 16-byte aligned */
} sq_attention_buffers;
int sq_attention_plan_for(const sq_device *device, const sq_attention_shape *shape, uint32_t sequences, uint32_t rows,
                          uint32_t chunk_rows, sq_attention_plan *out);
/* The work (tiles of 64 keys over every sequence, key head and tile of rows) is split evenly over the workgroups
 * whatever the lengths are; a second launch joins the tiles of rows whose keys several workgroups shared, in key order,
 * so a batch repeats its bits from run to run. How the work falls depends on the whole batch, so a row's output
 * bits may differ between batches. A call's sequences, rows, keys (pages_per_sequence * page_rows) and key heads multiply
 * to less than 2^52. */
int sq_attention_add(void *graph, const sq_attention_buffers *buffers, const sq_kv_cache *cache,
                     const sq_kv_batch *batch, const sq_attention_plan *plan);
/* What sq_attention_add_scored does to the scores t = scale q.k of a row at position p and a key at j, and to which keys the
 * row sees; each part may be absent (cap 0, views NULL), and all of it (scores NULL: sq_attention_add).
 *  cap       t becomes cap tanh(t / cap), off by 2^-21 of the cap (of a cap up to 128), or 2^-20 of t (of a larger one).
 *            Finite, 2^-100 or more; the cap and |scale| / cap, each times log2 e, are finite too.
 *  slopes    then t - slopes[h] |p - j|, fp32 [heads] on the device, 4-byte aligned.
 *  begins    uint32 [sequences], 4-byte aligned: rows of sequence s see no key before begins[s]. Packed documents, each for
 *            itself, are sequences of a batch that share a page table row: a document that ends at position e of them has
 *            length e, and begins at its first key.
 *  prefixes  uint32 [sequences], 4-byte aligned: rows of sequence s see its keys before prefixes[s] too, where they lie behind
 *            the row. Causal attention only.
 * A window hides what it hides of the keys seen by these. The plan is sq_attention_plan_for's. */
typedef struct sq_attention_scores {
  float cap;
  sq_buffer slopes, begins, prefixes;
} sq_attention_scores;
int sq_attention_add_scored(void *graph, const sq_attention_buffers *buffers, const sq_kv_cache *cache,
                            const sq_kv_batch *batch, const sq_attention_plan *plan, const sq_attention_scores *scores);

/* ---- the pages of a cache ---- */

/* The books of a cache's pages, on the device: how many entries of the page table name each page (references, uint32 [pages];
 * 0: the page is free), the table (uint32 [sequences][pages_per_sequence]; a kv batch's own, or the rows that batches are made
 * of), and the keys of each sequence (lengths, uint32 [sequences]). A call of the four below takes them from one consistent
 * state to the next, in stream order and with no word from the host; a captured one does so at each replay. New pages are
 * always the free ones of lowest number, in the order of the requests and of their entries, so that results repeat.
 * An empty pool has zero references and lengths and a table of ~0u. Entries of a sequence past its keys are ~0u; an entry that
 * names no page is a hole, shares and releases nothing.
 * report (uint32 [4]) tells what the last call did: [0] requests not carried out, [1] pages copied, [2] (compact alone writes
 * it) pages in use. A release, grow or fork of no requests launches nothing, and leaves the report as it was. Requests are
 * uint32 arrays on the device, at most SQ_KV_MAX_SEQUENCES of them a call. One that names no sequence, or one that an earlier
 * request of the call names, is not carried out; nor is one that needs new pages where too few are free for it and the requests
 * before it. All views are 4-byte aligned; workspace (16-byte aligned, of sq_kv_pool_workspace's bytes) may hold anything
 * before a call and serves one stream at a time. Nothing here reads or writes past the views, whatever they hold.
 * The books are of one cache, and which pages a call moved or copied is not told. A model's caches, one a layer, have books
 * each: the same calls make the same of equal books, and their tables stay equal. */
typedef struct sq_kv_pool {
  sq_kv_cache cache;
  /* sequences at most 2^20, sequences * pages_per_sequence at most 2^28, pages_per_sequence * page_rows at most 2^30 */
  uint32_t sequences, pages_per_sequence;
  sq_buffer references, page_table, lengths, report;
} sq_kv_pool;
int sq_kv_pool_workspace(const sq_kv_pool *pool, uint64_t *bytes);
/* Cuts sequence rows[i] back to keeps[i] keys (0: frees it; as many as it has or more: leaves it): entries past the kept keys'
 * pages become holes, and a page that no entry names any more is free. A sequence may be named twice: the shorter counts. */
int sq_kv_pool_add_release(void *graph, const sq_kv_pool *pool, sq_buffer rows, sq_buffer keeps, uint32_t requests);
/* Makes sequence rows[i] hold more[i] keys more, which a write then fills: entries for them name new pages, and its length
 * grows. If its last page holds keys and other entries name it too, the sequence gets a copy of it (of the rows with keys) in a
 * new page before. A sequence that would outgrow its table row is not grown. */
int sq_kv_pool_add_grow(void *graph, const sq_kv_pool *pool, sq_buffer rows, sq_buffer more, uint32_t requests,
                        sq_buffer workspace);
/* Makes sequence children[i] a fork of sequence parents[i]: the same keys, whole pages shared with it, the last page (if it
 * is not full) a copy, of the rows with keys, in a new page that the child goes on writing. What the child's entries named
 * before is not released. A child that is a parent of the call is not forked. */
int sq_kv_pool_add_fork(void *graph, const sq_kv_pool *pool, sq_buffer parents, sq_buffer children, uint32_t requests,
                        sq_buffer workspace);
/* Moves the pages in use to the front: of n of them, the last one goes to the first free place, the one before it to the second,
 * until all lie in places 0 to n - 1. References and table entries follow; the places left are free and keep their bits. */
int sq_kv_pool_add_compact(void *graph, const sq_kv_pool *pool, sq_buffer workspace);
/* Copies page pairs[2 i] of `from` to page pairs[2 i + 1] of `to` (uint32 [pairs][2] on the device, 8-byte aligned), keys,
 * values and scales. Both caches have one shape, and may be one cache. No page is written twice, or read and written, by one
 * call; a pair that names a page that its cache has not copies nothing. */
int sq_kv_add_copy(void *graph, const sq_kv_cache *from, const sq_kv_cache *to, sq_buffer pairs, uint32_t count);

#ifdef __cplusplus
}
#endif
#endif
