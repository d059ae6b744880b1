/*
 * awqb200.h - C ABI of the B200 (sm_100a) AWQ W4A16 quantized-linear library.
 *
 * Every entry point is plain C: device pointers, sizes, a dtype code and a
 * CUDA stream passed as void* (cudaStream_t). Each returns 0 on success or a
 * non-zero status; awqb_last_error() then holds a message for the calling
 * thread. No entry point allocates device memory or synchronises the device
 * unless its comment says so, so the GEMM paths can be captured in CUDA graphs.
 *
 * Status codes:
 *   0 ok, 1 invalid argument, 2 unsupported shape/config, 3 CUDA error,
 *   4 NCCL error, 5 a bounded device-side wait gave up.
 *
 * Each declaration cites the reference (SGLite) interface it replaces, by path
 * inside python/sglite/.
 */
#ifndef AWQB200_H
#define AWQB200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define AWQB_ABI_VERSION 1

enum { AWQB_DTYPE_F16 = 0, AWQB_DTYPE_BF16 = 1 };

/* Message describing the last failure on this thread ("" if none).
 * Replaces host::PanicError messages, kernels/csrc/include/sglite/utils.h:42-92. */
const char* awqb_last_error(void);
int awqb_abi_version(void);

/* ------------------------------------------------------------------------
 * Weight repack (load time).
 * Replaces awq_marlin_repack + marlin_permute_scales + awq_to_marlin_zero_points
 * called from AWQMarlinLinearMethod.process_weights_after_loading,
 * srt/model_executor/layers/quantization/awq_marlin.py:270-334.
 *
 * AWQ inputs (awq.py:87-124): qweight int32 [batch][K][N/8], qzeros int32
 * [batch][K/G][N/8], scales (fp16 or bf16 bits) [batch][K/G][N]. batch > 1
 * repacks stacked MoE experts ([E, K, N/8], weight_loader.py:134-142).
 * G must be 32, 64 or a multiple of 128, K % G == 0, N % 8 == 0.
 */
int awqb_blob_bytes(int64_t K, int64_t N, int64_t G, int64_t* bytes);
int awqb_repack(const int32_t* qweight, const int32_t* qzeros, const uint16_t* scales,
                int64_t batch, int64_t K, int64_t N, int64_t G, void* blob, void* stream);
/* Exact inverse of awqb_repack (used to prove the repack is lossless). */
int awqb_unrepack(const void* blob, int64_t batch, int64_t K, int64_t N, int64_t G,
                  int32_t* qweight, int32_t* qzeros, uint16_t* scales, void* stream);
/* W[batch][K][N] = (q - z) * s in the activation dtype, with the GEMM's own
 * dequantisation routine; bit-exact with the reference unpack + dequantise,
 * layers/quantization/awq_triton.py:53-62,94-96,119-122. */
int awqb_dequant(const void* blob, int64_t batch, int64_t K, int64_t N, int64_t G, int dtype,
                 void* w, void* stream);

/* ------------------------------------------------------------------------
 * W4A16 GEMM: y[M][N] = x[M][K] * dequant(blob)[K][N] (+ bias[N]).
 * Replaces awq_gemm_triton, layers/quantization/awq_triton.py:144-195 (called by
 * AWQLinearMethod.apply_weights, awq.py:126-147) and gptq_marlin_gemm through
 * apply_awq_marlin_linear, marlin_utils.py:355-415.
 * x, y, bias are in the activation dtype; x 16-byte aligned, rows contiguous.
 * fp32 accumulation. The workspace (size from awqb_gemm_workspace_bytes) must
 * be 256-byte aligned. Its first 8 KiB hold split-tile counters: zero them
 * before the first use; every call leaves them zero again (the rest is scratch
 * for fp32 partial tiles). Calls of any shape may share one workspace as long
 * as it is large enough for each; calls that share it must not overlap in time.
 * At most 1024 CTAs.
 */
int awqb_gemm_workspace_bytes(int64_t M, int64_t K, int64_t N, int64_t G, int64_t* bytes);
int awqb_gemm(const void* x, int64_t M, int64_t K, int64_t N, int64_t G, int dtype,
              const void* blob, const void* bias, void* y, void* workspace,
              int64_t workspace_bytes, void* stream);
/* Same with an explicit token tile (16, 32, 64, 128, 256; 0 = default) and CTA
 * count (0 = one per SM); for tuning and tests. */
int awqb_gemm_workspace_bytes_ex(int64_t M, int64_t K, int64_t N, int64_t G, int ntok,
                                 int64_t ctas, int64_t* bytes);
int awqb_gemm_ex(const void* x, int64_t M, int64_t K, int64_t N, int64_t G, int dtype,
                 const void* blob, const void* bias, void* y, void* workspace,
                 int64_t workspace_bytes, int ntok, int64_t ctas, void* stream);
/* The launch awqb_gemm / awqb_gemm_ex would make for these arguments: token
 * tile, CTA count, and cluster size (0 = the small-batch kernel below, one
 * slice of output features per CTA over all of K; 1 = stream-K with the
 * reduction through the workspace; >= 2 = one tile per cluster of that many
 * CTAs, reduced through distributed shared memory). Diagnostics; no
 * counterpart in the reference. */
int awqb_gemm_plan(int64_t M, int64_t K, int64_t N, int64_t G, int ntok, int64_t ctas, int* ntok_out,
                   int64_t* ctas_out, int* cluster_out);

/* Small-batch (decode) kernel that awqb_gemm takes for small M (see
 * awqb_gemm_plan: cluster 0) when no token tile or CTA count is forced: each
 * CTA computes features_per_cta output features over all of K with `warps`
 * compute warps, the weights dequantised in registers and multiplied on
 * mma.sync with fp32 accumulation. Built pairs (features_per_cta, warps):
 * (16, 16), (32, 16), (32, 8), (64, 8); 0 picks by M, N and the SM count.
 * ring (1..16, 0 = by shared memory) is its depth of load stages (warps
 * k-blocks each). 1 <= M <= 32. Needs no workspace. silu_mul != 0 gives the
 * output of awqb_gemm_silu_mul (interleaved gate/up columns, y [M][N/2]).
 * Exposed for tuning and tests. Replaces, for decode batches,
 * awq_gemm_triton, layers/quantization/awq_triton.py:144-195. */
int awqb_gemv_ex(const void* x, int64_t M, int64_t K, int64_t N, int64_t G, int dtype,
                 const void* blob, const void* bias, void* y, int features_per_cta, int warps, int ring,
                 int silu_mul, void* stream);

/* GEMM for callers that cannot provide or allocate device memory: a host that
 * owns every device byte through its own arena, or code that must never call
 * cudaMalloc (it may run during CUDA graph capture, or on a path that cannot
 * afford an allocation's implicit synchronisation). No counterpart in the
 * reference. Same computation and arguments as awqb_gemm minus the workspace:
 * the split-K scratch is a fixed array inside the library
 * (awqb_gemm_noalloc_scratch_bytes() = 16 MiB, held by every GPU that loads the
 * library until the process exits). Problems that need more scratch are
 * rejected with status 2 and a message; every M <= 64 fits. Nothing is
 * allocated: the array's device address is looked up once per device by the
 * first call made with that device current, so make that first call before
 * any stream capture. All calls share the one array, so calls that can run at
 * the same time on the GPU (different streams) race and must be serialised by
 * the caller. */
int64_t awqb_gemm_noalloc_scratch_bytes(void);
int awqb_gemm_noalloc(const void* x, int64_t M, int64_t K, int64_t N, int64_t G, int dtype,
                      const void* blob, const void* bias, void* y, void* stream);

/* ------------------------------------------------------------------------
 * MoE (Qwen3-MoE experts). The reference runs dense experts through
 * FusedMoe.forward, srt/model_executor/layers/fused_moe/fused.py:205-233;
 * these entry points give the same pipeline over AWQ expert weights.
 */
/* softmax over E router logits (fp32) and top-k; renormalize divides by the
 * top-k sum and then by (sum + 1e-8). Replaces fused_topk, fused.py:11-31. */
int awqb_moe_topk_softmax(const float* logits, int64_t M, int64_t E, int64_t topk,
                          int renormalize, float* topk_weights, int32_t* topk_ids, void* stream);
/* Length of sorted_ids needed by awqb_moe_align. */
int64_t awqb_moe_max_padded(int64_t numel, int64_t num_experts, int64_t block_m);
/* Sort the numel = M*topk (token, k) pairs routed to experts [e_begin, e_end)
 * by expert (stable), pad each expert to block_m with the sentinel numel, write
 * the local expert index of every block and the padded row count.
 * Replaces moe_align_block_size, fused.py:34-61. */
int awqb_moe_align(const int32_t* topk_ids, int64_t numel, int64_t e_begin, int64_t e_end,
                   int64_t block_m, int32_t* sorted_ids, int64_t max_padded,
                   int32_t* block_expert, int32_t* num_post_pad, void* stream);
/* The same result computed by many CTAs (chunk histograms, one scan CTA, one
 * warp per chunk for the stable scatter): for large inputs (thousands of pairs),
 * where one CTA is bound by a single SM. Needs a caller-owned workspace of
 * awqb_moe_align_workspace_bytes(numel, e_end - e_begin) bytes (per-chunk
 * counts; no zeroing needed). Replaces moe_align_block_size, fused.py:34-61. */
int64_t awqb_moe_align_workspace_bytes(int64_t numel, int64_t num_experts);
int awqb_moe_align_ex(const int32_t* topk_ids, int64_t numel, int64_t e_begin, int64_t e_end,
                      int64_t block_m, int32_t* sorted_ids, int64_t max_padded, int32_t* block_expert,
                      int32_t* num_post_pad, void* workspace, int64_t workspace_bytes, void* stream);
/* out[r] = x[sorted_ids[r] / topk] (zero for padding rows), r < *num_post_pad.
 * Stands in for the row gather done by fused_moe_kernel's a_ptrs,
 * kernels/triton/fused_moe.py:241. */
int awqb_moe_gather_rows(const void* x, int64_t K, const int32_t* sorted_ids,
                         const int32_t* num_post_pad, int64_t numel, int64_t topk,
                         int64_t rows_max, void* out, void* stream);
/* Grouped W4A16 GEMM over expert-sorted rows: blobs holds one blob per expert,
 * blob_stride bytes apart (awqb_repack with batch = E). ntok must equal the
 * align block size. Optional row_map / row_scale scatter rows to
 * row_map[r] (< num_valid) and multiply by row_scale[that row].
 * Replaces fused_moe_kernel, kernels/triton/fused_moe.py:155-285. */
int awqb_moe_grouped_workspace_bytes(int64_t rows_max, int64_t K, int64_t N, int64_t G, int ntok,
                                     int64_t* bytes);
int awqb_moe_grouped_gemm(const void* x_sorted, int64_t rows_max, int64_t K, int64_t N, int64_t G,
                          int dtype, const void* blobs, int64_t blob_stride,
                          const int32_t* block_expert, const int32_t* num_post_pad, int ntok,
                          const int32_t* row_map, const float* row_scale, int64_t num_valid,
                          void* y, int64_t ldy, void* workspace, int64_t workspace_bytes,
                          void* stream);
/* The gate_up projection fused with SiLU-and-mul: y[M][N/2] = silu(x W_gate) *
 * (x W_up), computed from the fp32 accumulators (one rounding). The blob must
 * come from AWQ tensors whose columns are interleaved one by one (column 2j =
 * gate j, column 2j + 1 = up j; ops.interleave_gate_up repacks the AWQ
 * tensors). N % 16 == 0; bias (if any) is interleaved the same way. Replaces the gate_up GEMM + SiluAndMul pair of the MLP
 * (layers/activation.py:11-22, blocks.py:53-57) and of the MoE experts
 * (fused.py:160-178). Workspace as for awqb_gemm. */
int awqb_gemm_silu_mul(const void* x, int64_t M, int64_t K, int64_t N, int64_t G, int dtype,
                       const void* blob, const void* bias, void* y, void* workspace,
                       int64_t workspace_bytes, void* stream);
/* The same for the MoE expert gate_up GEMM over expert-sorted rows: y [rows][ldy]
 * with ldy >= N / 2, rows in sorted order (as awqb_moe_grouped_gemm without
 * row_map / row_scale). */
int awqb_moe_grouped_gemm_silu_mul(const void* x_sorted, int64_t rows_max, int64_t K, int64_t N,
                                   int64_t G, int dtype, const void* blobs, int64_t blob_stride,
                                   const int32_t* block_expert, const int32_t* num_post_pad, int ntok,
                                   void* y, int64_t ldy, void* workspace, int64_t workspace_bytes,
                                   void* stream);
/* out[r][j] = silu(in[r][j]) * in[r][I + j] in fp32; rows = min(rows_max,
 * *rows_dev) when rows_dev is given. Replaces silu_and_mul (flashinfer),
 * srt/model_executor/layers/activation.py:11-15. */
int awqb_silu_and_mul(const void* in, int64_t rows_max, const int32_t* rows_dev, int64_t I,
                      int dtype, void* out, void* stream);
/* The same for gate_up outputs in the interleaved layout of awqb_gemm_silu_mul
 * (in[r][2j] = gate j, in[r][2j + 1] = up j). */
int awqb_silu_and_mul_interleaved(const void* in, int64_t rows_max, const int32_t* rows_dev, int64_t I,
                                  int dtype, void* out, void* stream);
/* out[m][h] = sum_k in[m][k][h] (fp32 accumulate), counting only pairs whose
 * expert is in [e_begin, e_end) when topk_ids is given.
 * Replaces moe_sum_reduce_triton, kernels/moe_triton.py:68-102. */
int awqb_moe_topk_sum(const void* in, int64_t M, int64_t topk, int64_t H, const int32_t* topk_ids,
                      int64_t e_begin, int64_t e_end, int dtype, void* out, void* stream);

/* ------------------------------------------------------------------------
 * RMSNorm after a projection. Replace flashinfer.rmsnorm and
 * flashinfer.fused_add_rmsnorm as called by RMSNorm / RMSNormFused,
 * srt/model_executor/layers/norm.py:10-47 (arithmetic of flashinfer 0.6.11,
 * include/flashinfer/norm.cuh): per row, x = input (+ residual) in fp32,
 * out = x * rsqrt(mean(x * x) + eps) * weight, rounded to the dtype.
 * N (features) is a multiple of 8 and at most 16384; row strides ld_* are in
 * elements, multiples of 8; all pointers 16-byte aligned. The kernels are
 * launched with programmatic dependent launch after a GEMM on the same stream.
 * ------------------------------------------------------------------------ */
/* out[m] = RMSNorm(input[m]) * weight (out may equal input). */
int awqb_rmsnorm(const void* input, const void* weight, void* out, int64_t M, int64_t N, int64_t ld_in,
                 int64_t ld_out, float eps, int dtype, void* stream);
/* In place: residual[m] = input[m] + residual[m] (rounded), then
 * input[m] = RMSNorm(fp32 sum) * weight. */
int awqb_fused_add_rmsnorm(void* input, void* residual, const void* weight, int64_t M, int64_t N,
                           int64_t ld_in, int64_t ld_res, float eps, int dtype, void* stream);

/* The entry points of this section that take a structure read it during the call
 * only; it may be reused or freed afterwards. */
/* The norms around a block, fused with its gate and residual scale: the step
 * between one block's projection output x and the next block's input. Per row,
 * in fp32:
 *   b = post_weight ? x * rsqrt(mean(x * x) + eps) * (weight_offset + post_weight) : x
 *   h = residual + scale * act(gate) * b
 *   residual_out = h (rounded to the residual's type)
 *   out = h * rsqrt(mean(h * h) + eps) * (weight_offset + weight)
 * where the second norm is taken over the unrounded h, as in
 * awqb_fused_add_rmsnorm. post_weight, gate and weight (with out) may be null:
 * no norm after the block, a gate of 1, no norm before the next block; one of
 * post_weight and weight must be given. weight_offset is 0, or 1 for models
 * that store their norm weights minus one. x, the weights, gate and out are of
 * `dtype`; residual and residual_out are fp32 if residual_f32 != 0, else of
 * `dtype`. Element (m, n) of the gate is gate[m * gate_row + n * gate_col]
 * with gate_col 0 or 1 (0, 1: per channel; 1, 0: per row). gate_act: 0 none,
 * 1 sigmoid, 2 tanh, 3 SiLU. N is a multiple of 8, at most 16384; row strides
 * ld_* (and gate_row where gate_col is 1) are in elements, multiples of 8;
 * pointers 16-byte aligned. out may equal x and residual_out may equal
 * residual; other overlaps are not allowed. Extends RMSNormFused,
 * srt/model_executor/layers/norm.py:28-47. */
typedef struct {
  const void* x;
  int64_t ld_x;
  const void* residual;
  int64_t ld_res;
  int residual_f32;
  const void* post_weight;
  const void* gate;
  int64_t gate_row;
  int64_t gate_col;
  int gate_act;
  float scale;
  const void* weight;
  float weight_offset;
  void* out;
  int64_t ld_out;
  void* residual_out;
  int64_t ld_res_out;
  int64_t M;
  int64_t N;
  float eps;
  int dtype;
} awqb_gated_norm_args;
int awqb_gated_add_rmsnorm(const awqb_gated_norm_args* args, void* stream);

/* ------------------------------------------------------------------------
 * Rotary positions of q and k between the QKV projection and attention, with
 * the per-head RMSNorm of q and k (if q_weight / k_weight are given) folded in.
 * Head h of token m starts at q + m * q_row + h * q_head (elements), likewise
 * k and the outputs, so q and k may be slices of the merged projection's
 * output. Per head, in fp32 with one rounding at the end:
 *   v = q_weight ? q * rsqrt(mean(q * q) + eps) * q_weight : q
 *   pair j < rot_dim / 2 of v (elements j and j + rot_dim / 2, or 2j and 2j + 1
 *   if interleaved) turns by the angle positions[m] * inv_freq[j]: (a, b) ->
 *   scale * (a cos - b sin, a sin + b cos); elements from rot_dim on stay.
 * inv_freq is fp64. The angle is the position times a 64-bit fraction of a turn,
 * modulo whole turns, so far positions keep their accuracy (2^-24 of a turn at
 * position 2^29); a long-context scaling enters through inv_freq and scale.
 * positions are int32, or int64 if positions_i64 != 0. A token with a negative
 * position is padding: its outputs are left as they were. Outputs may be the
 * inputs (in place); other overlaps are not allowed. head_dim is a multiple of
 * 8, at most 256; rot_dim is even, 2..head_dim; strides are multiples of 8
 * and pointers of q, k, the weights and outputs 16-byte aligned. Hk may be 0
 * (no k). Replaces the rotary call of RopeAttn, models/blocks.py:134-139 and
 * layers/rotary.py. */
typedef struct {
  const void* q;
  int64_t q_row, q_head, Hq;
  const void* k;
  int64_t k_row, k_head, Hk;
  const void* positions;
  int positions_i64;
  const double* inv_freq;
  int64_t rot_dim, head_dim, M;
  int interleaved;
  float scale;
  const void* q_weight;
  const void* k_weight;
  float eps;
  void* q_out;
  int64_t q_out_row, q_out_head;
  void* k_out;
  int64_t k_out_row, k_out_head;
  int dtype;
} awqb_rotary_args;
int awqb_rotary(const awqb_rotary_args* args, void* stream);

/* ------------------------------------------------------------------------
 * Work on rows that belong to groups (experts, adapters).
 * ------------------------------------------------------------------------ */
/* Stable grouping of n ids: order [n] lists the indices whose id is begin, then
 * those whose id is begin + 1, ..., then all others (in no group), each in
 * index order; group g's indices are order[offsets[g] .. offsets[g + 1]),
 * offsets [groups + 1], offsets[0] = 0. groups is 1..1024. The workspace
 * (awqb_group_rows_workspace_bytes; none for small n) needs no zeroing.
 * Replaces the sort of moe_align_block_size, fused.py:34-61, without padding. */
int64_t awqb_group_rows_workspace_bytes(int64_t n, int64_t groups);
int awqb_group_rows(const int32_t* ids, int64_t n, int64_t begin, int64_t groups, int32_t* order,
                    int32_t* offsets, void* workspace, int64_t workspace_bytes, void* stream);
/* Matrix products grouped by expert over 16-bit weights w [E][N][K]:
 *   y[r] = x[r] w[e]^T for offsets[e] <= r < offsets[e + 1]
 * (fp32 accumulation, one rounding), or with silu_mul != 0, w [E][2I][K] holding
 * the gate rows and then the up rows (N = 2I), y[r] = silu(gate) * up (I
 * features). offsets [E + 1] is on the device, does not decrease and stays in
 * 0..rows (values outside are clamped); rows of x outside
 * [offsets[0], offsets[E]) are not computed. With row_map, y[r] goes to row
 * row_map[r] of out (rows that map outside 0..out_rows - 1 are dropped), else
 * to row r; with row_scale (fp32) it is multiplied by row_scale[its out row].
 * No two rows may map to one. Rows of out that nothing maps to are left as they
 * were. K is a multiple of 8,
 * N of 8 (16 with silu_mul); ldx and ldo are in elements, multiples of 8;
 * x, w and out 16-byte aligned. out must not overlap the inputs. E <= 1024.
 * Replaces fused_moe_kernel over dense experts, kernels/triton/fused_moe.py:155-285. */
typedef struct {
  const void* x;
  int64_t rows, ldx;
  const void* w;
  int64_t E, K, N;
  const int32_t* offsets;
  int dtype;
  int silu_mul;
  const int32_t* row_map;
  const float* row_scale;
  void* out;
  int64_t out_rows, ldo;
} awqb_grouped_gemm_args;
int awqb_grouped_gemm(const awqb_grouped_gemm_args* args, void* stream);
/* Low-rank adapters of many requests beside a shared projection:
 *   out[t] = base[t] + scales[a] * (x[t] a[a]^T) b[a]^T
 * for the rows t = order[offsets[a] .. offsets[a + 1]) of adapter a; rows in no
 * adapter (the rest of order) get out = base. A merged projection (QKV,
 * gate_up) has num_slices > 1 slices of its N outputs (slices: their widths,
 * adding up to N), each with its own pair: a
 * [L][num_slices * rank][K] stacks the slices' first factors, b [L][N][rank]
 * their second ones. Sums are fp32; the product of the first factor enters the
 * second one as two 16-bit halves: bf16 loses 2^-16 of each value, fp16 2^-22 or
 * 2^-39 of the row's largest value in the slice. scales [L] fp32 or null (1).
 * order [M] and offsets [L + 1] as awqb_group_rows gives them: order is a
 * permutation of the rows (an entry outside 0..M - 1 is skipped). out may
 * equal base (with the same row stride); other overlaps are not allowed. K is a multiple of 8, the slice widths of 8, rank of 8 and at
 * most 128, num_slices at most 4, L at most 1024; row strides are in elements,
 * multiples of 8; pointers 16-byte aligned. No counterpart in the reference. */
int awqb_lora_workspace_bytes(int64_t M, int64_t K, int64_t N, int64_t L, int64_t rank, int64_t num_slices,
                              int64_t* bytes);
typedef struct {
  const void* x;
  int64_t M, ldx, K;
  const void* a;
  const void* b;
  int64_t L, rank, N;
  int64_t num_slices;
  int64_t slices[4];
  const int32_t* order;
  const int32_t* offsets;
  const float* scales;
  const void* base;
  int64_t ld_base;
  void* out;
  int64_t ld_out;
  int dtype;
  void* workspace;
  int64_t workspace_bytes;
} awqb_lora_args;
int awqb_lora(const awqb_lora_args* args, void* stream);

/* ------------------------------------------------------------------------
 * Tensor-parallel all-reduce. Replaces NCCLWrapper (create_nccl_uid, ctor,
 * all_reduce), kernels/csrc/src/pynccl.cu:75-189, used through
 * PyNCCLDistributedImpl.all_reduce, srt/distributed/communicator.py:62-65.
 * sym_bytes > 0 allocates an ncclMemAlloc buffer registered as a symmetric
 * window (the reference's max_bytes buffer); reductions up to that size are
 * staged through it. awqb_nccl_init allocates (NCCL-owned) memory.
 */
int awqb_nccl_unique_id_bytes(void);
int awqb_nccl_get_unique_id(uint8_t* out);
int awqb_nccl_init(const uint8_t* uid, int rank, int world, int64_t sym_bytes, void** comm);
int awqb_nccl_symmetric_buffer(void* comm, void** ptr, int64_t* bytes);
int awqb_nccl_all_reduce(void* comm, void* buf, int64_t count, int dtype, void* stream);
int awqb_nccl_destroy(void* comm);

/* ------------------------------------------------------------------------
 * Row-parallel GEMM fused with its all-reduce over peer memory (NVLink).
 * Replaces, for small M, the pair RowParallelLinear.forward
 * (layers/linear.py:189-194) = quantised GEMM + PyNCCLCommunicator.all_reduce
 * (kernels/csrc/src/pynccl.cu:96-138): every rank computes its K-slice
 * product and writes each finished value, as one 8-byte {fp32, call tag} word,
 * into every rank's landing buffer; each rank waits for the world words of its
 * values (no fences or flags: the tag travels with the value), sums them in
 * rank order (identical bits on all ranks), adds the bias once and stores
 * y [M][N] in the activation dtype. One kernel, no NCCL call.
 *
 * Set-up, once per rank of the group (collective in spirit: every rank must do
 * it): awqb_tp_exchange_create allocates this rank's exchange buffer
 * (cudaMalloc, (16 * world + 8) * max_rows * max_n bytes + 256) on the current
 * device; exchange the awqb_tp_exchange_handle bytes of all ranks (any host
 * channel), then awqb_tp_exchange_open(ctx, handles of ranks 0..world-1 back to
 * back). Every rank must then issue the same sequence of awqb_gemm_allreduce
 * calls with the same M, K, N, G (a collective); M <= max_rows, N <= max_n.
 * The kernel waits (bounded, 2 s) for its peers' tiles: a rank that does not
 * take part turns into a device error (awqb_device_error), not a hang. The
 * context may be used inside CUDA graphs (no host state changes per call).
 */
int awqb_tp_exchange_handle_bytes(int64_t* bytes);
int awqb_tp_exchange_create(int rank, int world, int64_t max_rows, int64_t max_n, void** ctx);
int awqb_tp_exchange_handle(void* ctx, void* handle_out);
int awqb_tp_exchange_open(void* ctx, const void* handles);
/* Exchange pattern of the fused all-reduce (every rank must set the same):
 * 0 auto (reduce-scatter + all-gather from 4 ranks and 8 rows, on launches
 * that split K over a thread-block cluster; all-to-all otherwise), 1 always
 * all-to-all (each rank sends its partial to every rank; every rank sums),
 * 2 reduce-scatter + all-gather wherever the launch allows it (each rank sends
 * its partial of feature tile t to rank t % world only; that rank sums and
 * sends the rounded result to the others). Results are bit-identical across
 * modes: every sum is taken in rank order. No counterpart in the reference. */
int awqb_tp_exchange_set_mode(void* ctx, int mode);
int awqb_tp_exchange_destroy(void* ctx);
int awqb_gemm_allreduce(const void* x, int64_t M, int64_t K, int64_t N, int64_t G, int dtype,
                        const void* blob, const void* bias, void* y, void* workspace,
                        int64_t workspace_bytes, void* ctx, void* stream);

/* Device-side error word (bits set when a bounded wait inside a kernel gave
 * up). Both calls synchronise the current device. */
int awqb_device_error(uint32_t* out);
int awqb_clear_device_error(void);

#ifdef __cplusplus
}
#endif

#endif /* AWQB200_H */
