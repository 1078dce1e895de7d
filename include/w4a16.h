/*
 * w4a16.h -- C ABI of the MI355X (gfx950) W4A16 linear library (libw4a16.so).
 *
 * Weight format consumed: AutoAWQ "GEMM" version, 4-bit, zero point, group 128:
 *   qweight int32 [K, N/8]   nibble i of word [k, j] holds column 8j + (0,2,4,6,1,3,5,7)[i]
 *   qzeros  int32 [K/128, N/8] same nibble order
 *   scales  bf16  [K/128, N]
 *   W[k, n] = bf16_rne( (q[k, n] - z[k/128, n]) * s[k/128, n] )
 * Activations x bf16 [M, K] row-major, output y bf16 [M, N] row-major.
 *
 * Conventions
 *   - Every tensor pointer is a device pointer owned by the caller; the library never
 *     allocates.  bf16 data is passed as uint16_t bit patterns.
 *   - `stream` is a hipStream_t (NULL = the legacy default stream).  Calls only enqueue
 *     work; nothing synchronises the host.
 *   - Return 0 on success, otherwise a W4A16_ERR_* code; w4a16_last_error() then gives a
 *     thread-local message.  No C++ exception crosses this boundary.
 *
 * Reference interfaces replaced (HGinkgo/LLM-Serve):
 *   pybind module of llmserve/layers/quantization/csrc/awq_w4a16.cu:375-379
 *     (repack_qweight, reorder_qzeros, linear) and its Python wrappers in
 *     llmserve/layers/quantization/awq_cuda.py:17-185, plus the reference backend
 *     functions of llmserve/layers/quantization/awq.py:184-276.
 */
#ifndef W4A16_H_
#define W4A16_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define W4A16_ABI_VERSION 5

enum w4a16_status {
  W4A16_OK = 0,
  W4A16_ERR_ARG = 1,       /* null pointer or non-positive size */
  W4A16_ERR_SHAPE = 2,     /* K / N / group contract violated */
  W4A16_ERR_ALIGN = 3,     /* a pointer is not aligned as the kernel requires */
  W4A16_ERR_WORKSPACE = 4, /* workspace missing or smaller than w4a16_workspace_bytes */
  W4A16_ERR_LAUNCH = 5     /* hipGetLastError() reported a launch failure */
};

/* Kernel families reported by w4a16_regime(). */
/* Element type of a float weight given to w4a16_quantize (its scales get the same type). */
enum w4a16_dtype {
  W4A16_DTYPE_BF16 = 0,
  W4A16_DTYPE_F16 = 1,
  W4A16_DTYPE_F32 = 2
};

enum w4a16_regime_id {
  W4A16_REGIME_NONE = 0,   /* M == 0: nothing to launch */
  W4A16_REGIME_DECODE = 1, /* M < 32: split-K, HBM-bound kernel */
  W4A16_REGIME_TILE = 2    /* larger M: LDS-tiled bf16 MFMA GEMM */
};

/* ABI version of the loaded library (W4A16_ABI_VERSION). No reference counterpart. */
int w4a16_abi_version(void);

/* Thread-local text of the last error on this thread ("" if none).
 * Replaces the TORCH_CHECK messages of awq_w4a16.cu:249-334. */
const char* w4a16_last_error(void);

/* Unpack int32 [R, C] AWQ words into int32 [R, 8C] in logical column order.
 * Replaces unpack_awq_int4 (awq.py:184-200).  Requires R, C > 0. */
int w4a16_unpack_int4(const int32_t* packed, int32_t* out, int rows, int cols, void* stream);

/* Dequantize the AutoAWQ tensors into bf16 W [K, N], bit-exact with the reference.
 * Replaces dequantize_awq_gemm (awq.py:235-248).  Any group_size > 0 dividing K; N % 8 == 0. */
int w4a16_dequant(const int32_t* qweight, const int32_t* qzeros, const uint16_t* scales,
                  uint16_t* w_out, int K, int N, int group_size, void* stream);

/* Rearrange qweight [K, N/8] into the group-tile layout consumed by w4a16_gemm (same
 * 4-bit values, same byte size K*N/2).  One 1 KiB tile per (128-row group g, 16-column
 * tile t); word [((g*(N/16) + t)*64 + lane)*4 + js] holds, at bit 8h + 4(k/2) + 16(k%2),
 * the value of row 128g + 32js + 8(lane/16) + 4h + lane%4 and column
 * 16t + 4((lane/4)%4) + k, for h = 0..1 and k = 0..3.  K % 128 == 0, N % 16 == 0.
 * Replaces repack_qweight (awq_w4a16.cu:81-109, 256-272) / repack_awq_qweight_cuda
 * (awq_cuda.py:129-132).  qzeros need no reorder: the kernels read them as stored, so
 * reorder_qzeros (awq_w4a16.cu:111-118, 274-286) has no counterpart. */
int w4a16_repack_qweight(const int32_t* qweight, int32_t* packed, int K, int N, void* stream);

/* Dequantize from the repacked layout through the GEMM kernels' matrix-core dequant
 * (same bits as w4a16_dequant for every finite scale with |s| < 2^123, zero signs aside);
 * exists to verify that path bit-exactly.  K % 128 == 0, N % 16 == 0.  No reference
 * counterpart beyond dequantize_awq_gemm (awq.py:235-248). */
int w4a16_dequant_packed(const int32_t* packed, const int32_t* qzeros, const uint16_t* scales,
                         uint16_t* w_out, int K, int N, int group_size, void* stream);

/* Group-wise asymmetric int4 quantization of weight [out_features, in_features] (row-major,
 * element type dtype) into the AutoAWQ GEMM layout: qweight [in_features, out_features/8],
 * qzeros [in_features/group_size, out_features/8] (int32), scales
 * [in_features/group_size, out_features] of type dtype.  Per (output row, group):
 * s = max(max - min, 1e-5) / 15, z = clamp(-round(min / s), 0, 15),
 * q = clamp(round(w / s) + z, 0, 15) in fp32, round half to even -- bit-exact with the
 * reference for finite weights.  out_features % 8 == 0, 1 <= group_size <= 128 dividing
 * in_features, in_features / group_size <= 65535; weight 2- or 4-byte aligned by type.
 * Replaces quantize_awq_weight (awq_calibration.py:35-62). */
int w4a16_quantize(const void* weight, int dtype, int32_t* qweight, int32_t* qzeros, void* scales,
                   int out_features, int in_features, int group_size, void* stream);

/* Pack int32 values [rows, cols] (cols % 8 == 0; each value's low 4 bits) into AutoAWQ words
 * [rows, cols/8]: nibble i of word [r, j] holds column 8j + (0,2,4,6,1,3,5,7)[i].  values
 * 16-byte aligned.  Range checks on the values stay with the caller.
 * Replaces _pack_int4 (awq_calibration.py:19-32). */
int w4a16_pack_int4(const int32_t* values, int32_t* packed, int rows, int cols, void* stream);

/* Bytes of workspace w4a16_gemm needs for this problem (0 = none), and, when N % 128 == 0,
 * w4a16_gemm_silu_mul too (the larger of the two).  The workspace must be
 * zero-filled once when first allocated; the kernels leave its counter words at zero.
 * Two GEMMs in flight at the same time must not share one workspace.
 * Replaces the workspace sizing of awq.py:168-180 and awq_cuda.py:157-176. */
size_t w4a16_workspace_bytes(int M, int K, int N, int group_size);

/* The largest w4a16_workspace_bytes(M, K, N, group_size) over 1 <= M <= M_max: one buffer of
 * this size, allocated and zero-filled at load time, serves every call with M <= M_max at
 * this shape (e.g. M_max = the engine's max_num_batched_tokens, 16384 by default), so the
 * GEMM calls never allocate.  0 for M_max < 1 or an invalid shape.
 * Replaces the load-time workspace allocation of process_weights_after_loading
 * (awq.py:168-180), which the reference sizes for its M <= 16 split-K kernel only. */
size_t w4a16_workspace_bytes_max(int M_max, int K, int N, int group_size);

/* y[M, N] = x[M, K] @ W with W given as (packed, qzeros, scales); bf16 in and out, fp32
 * accumulation.  M >= 0 (M == 0 is a no-op), K % 128 == 0, N % 64 == 0, group_size == 128,
 * K * N / 2 < 2^31 bytes of packed weights; x, packed, y 16-byte and qzeros, scales 4-byte
 * aligned.
 * Replaces linear (awq_w4a16.cu:288-371) / awq_cuda_linear (awq_cuda.py:141-185) and the
 * reference backend awq_reference_linear (awq.py:251-276). */
int w4a16_gemm(const uint16_t* x, const int32_t* packed, const int32_t* qzeros,
               const uint16_t* scales, uint16_t* y, int M, int K, int N, int group_size,
               void* workspace, size_t workspace_bytes, void* stream);

/* w4a16_gemm for callers that cannot allocate device memory (code under HIP graph capture,
 * tight serving loops, harnesses that forbid allocation): no workspace argument; the split-K
 * workspace is a 48 MiB device array of the library itself, one per GPU, held until the
 * process ends, set up on the first call on each device (symbol lookup, its counters
 * cleared by a kernel on `stream`): that first call must not be under graph capture
 * (W4A16_ERR_LAUNCH, nothing enqueued); later calls may be.  Allocates nothing.  Problems whose plan needs more
 * than 48 MiB of workspace (w4a16_workspace_bytes) are rejected with W4A16_ERR_WORKSPACE
 * before anything is enqueued (every Qwen3-8B projection at M <= 16384 fits).  Calls that
 * overlap on one GPU (two streams at once) share the array and race: serialize them.
 * Arguments, limits and results otherwise as w4a16_gemm (same kernels, same bits).
 * No counterpart in the reference: an allocation-free entry for the callers above. */
int w4a16_gemm_noalloc(const uint16_t* x, const int32_t* packed, const int32_t* qzeros,
                       const uint16_t* scales, uint16_t* y, int M, int K, int N, int group_size,
                       void* stream);

/* y[M, N] = bf16(bf16(x[M, K] @ W) + residual[M, N]): the GEMM with the residual add that
 * follows the O and down projections (the reference's add_rms_forward: x.float() +
 * residual.float() then bf16, layernorm.py:35-36) done in the epilogue.  residual may be y itself
 * (in place); 16-byte aligned.  Otherwise as w4a16_gemm; same workspace.  Replaces
 * o_proj / down_proj followed by that add (qwen3.py:170-174). */
int w4a16_gemm_residual(const uint16_t* x, const int32_t* packed, const int32_t* qzeros,
                        const uint16_t* scales, const uint16_t* residual, uint16_t* y, int M, int K,
                        int N, int group_size, void* workspace, size_t workspace_bytes, void* stream);

/* y[M, N/2] = SiLU(g) * u with [g | u] = x[M, K] @ W for a gate|up weight W [K, N] whose
 * first N/2 columns are the gate projection and last N/2 the up projection (the layout of
 * MergedColumnParallelLinear's gate_up_proj); g and u are rounded to bf16 as that layer
 * returns them, and SiLU(g) * u is computed in fp32 and rounded once, the reference's two
 * steps in one kernel.  Same arguments and limits as w4a16_gemm, plus N % 128 == 0; y is
 * [M, N/2], 16-byte aligned; workspace from w4a16_workspace_bytes(M, K, N, 128).
 * Replaces gate_up_proj followed by SiluAndMul (qwen3.py:126-130, activation.py:8-11):
 * the [M, N] gate|up intermediate is never written. */
int w4a16_gemm_silu_mul(const uint16_t* x, const int32_t* packed, const int32_t* qzeros,
                        const uint16_t* scales, uint16_t* y, int M, int K, int N, int group_size,
                        void* workspace, size_t workspace_bytes, void* stream);

/* RMSNorm of each row of x [M, K], with the residual add in front when residual is not NULL:
 *   s = float(x) + float(residual)  (s = float(x) without a residual), in fp32;
 *   residual_out = bf16(s);
 *   x_norm = bf16(float(bf16(s * rsqrt(mean(s * s) + eps))) * float(weight)).
 * weight is bf16 [K].  residual and residual_out are both given or both NULL; residual_out
 * may be residual or x (in place), x_norm may be x, x_norm != residual_out.  K % 8 == 0,
 * K <= 16384, every pointer 16-byte aligned, 0 <= eps <= 1.  rsqrt is evaluated in fp64
 * and the sum of squares is an fp32 tree sum, so bf16(s * r) can differ from another fp32
 * implementation by one bf16 ulp where s * r lies next to a rounding boundary (up to two
 * ulps of x_norm after the weight product).
 * Replaces RMSNorm.rms_forward / add_rms_forward (layernorm.py:16-40). */
int w4a16_add_rmsnorm(const uint16_t* x, const uint16_t* residual, const uint16_t* weight, float eps,
                      uint16_t* x_norm, uint16_t* residual_out, int M, int K, void* stream);

/* RMSNorm without a residual (as w4a16_add_rmsnorm with residual == NULL) of rows read
 * through two strides: row r of x starts at element
 * (r / rows_inner) * stride_outer + (r % rows_inner) * stride_inner; x_norm is contiguous
 * [M, K].  Strides are multiples of 8 elements, x 16-byte aligned; other limits as
 * w4a16_add_rmsnorm.  Rows of K <= 512 share a wave (8 .. 64 lanes per row).
 * Replaces RMSNorm.rms_forward (layernorm.py:16-25) on a non-contiguous view: q_norm and
 * k_norm over q.view(-1, heads, head_dim) of the split QKV output (qwen3.py:87-94). */
int w4a16_rmsnorm_strided(const uint16_t* x, int rows_inner, int64_t stride_outer, int64_t stride_inner,
                          const uint16_t* weight, float eps, uint16_t* x_norm, int M, int K, void* stream);

/* The RMSNorm(+residual) prologue of w4a16_add_rmsnorm followed, on the same stream and in
 * the same call, by w4a16_gemm (silu_mul == 0) or w4a16_gemm_silu_mul (silu_mul == 1) of
 * x_norm: y = x_norm @ W, or SiLU(g) * u of it.  x_norm [M, K] (a caller buffer) and
 * residual_out receive the norm's outputs.  At M <= 2 on decode plans without a K split
 * (the Qwen3-8B QKV and gate|up shapes) and with x_norm / residual_out overlapping neither x
 * nor residual, the norm runs inside the GEMM kernel (one launch); otherwise the norm kernel
 * writes x_norm and the GEMM reads it back (from L2 at decode sizes).  Arguments as for
 * those two calls; y must overlap none of x, residual, x_norm and residual_out
 * (W4A16_ERR_ARG).  The workspace is w4a16_workspace_bytes(M, K, N, 128).  Argument, shape
 * and workspace errors are reported before anything is enqueued.
 * Replaces input_layernorm / post_attention_layernorm followed by qkv_proj / gate_up_proj
 * (qwen3.py:166-173 with layernorm.py:28-40, qwen3.py:126-130). */
int w4a16_gemm_rmsnorm(const uint16_t* x, const uint16_t* residual, const uint16_t* norm_weight, float eps,
                       uint16_t* x_norm, uint16_t* residual_out, const int32_t* packed,
                       const int32_t* qzeros, const uint16_t* scales, uint16_t* y, int M, int K, int N,
                       int group_size, int silu_mul, void* workspace, size_t workspace_bytes,
                       void* stream);

/* The RMSNorm that follows the O or down projection, split across that GEMM and the next
 * one so that no norm launch sits between them (decode sizes, 0 <= M <= 8; M > 8 is
 * W4A16_ERR_SHAPE: use w4a16_gemm_residual / w4a16_gemm and w4a16_gemm_rmsnorm there).
 * Producer: h = bf16(x[M, K] @ W) is added to residual [M, N] in fp32 in the epilogue, as
 * the reference's add_rms_forward does (layernorm.py:35-36): s_out[M, N] (fp32) =
 * float(h) + float(residual), residual_out = bf16(s_out) (may be residual itself, in place),
 * and ssq_out[M, N / 16] (fp32) holds, per row, the sum of s^2 over each 16-column tile.  h
 * itself is not stored.  x, W, workspace as w4a16_gemm; every pointer 16-byte aligned; the
 * outputs overlap neither each other (but for residual_out == residual) nor the inputs.
 * Replaces o_proj / down_proj followed by the residual add and the sum of squares of the
 * next RMSNorm (qwen3.py:170-174 with layernorm.py:35-38). */
int w4a16_gemm_residual_stats(const uint16_t* x, const int32_t* packed, const int32_t* qzeros,
                              const uint16_t* scales, const uint16_t* residual, float* s_out,
                              uint16_t* residual_out, float* ssq_out, int M, int K, int N,
                              int group_size, void* workspace, size_t workspace_bytes,
                              void* stream);

/* Consumer of w4a16_gemm_residual_stats: the norm's scaling and the QKV GEMM (silu_mul == 0)
 * or the gate|up GEMM with SiLU * up (silu_mul == 1) in one decode kernel, whose workgroups
 * normalize the M rows of their K range once into LDS.  s [M, K] and
 * ssq [M, K / 16] are the producer's s_out and ssq_out (K its N); per row, rstd =
 * 1 / sqrt(sum(ssq) / K + eps) with the K / 16 tile sums added in a fixed order (rsqrt in
 * fp64, rounded once), then x_norm = bf16(float(bf16(s * rstd)) * float(norm_weight)) and
 * y = x_norm @ W (or SiLU(g) * u of it).  x_norm (may be NULL) receives the normalized
 * activations.  The sum of squares is added in another order than w4a16_add_rmsnorm's, so
 * x_norm can differ from it by one bf16 unit where s * rstd lies next to a rounding
 * boundary.  0 <= M <= 8, eps in [0, 1], every pointer 16-byte aligned; y overlaps none of
 * the inputs; workspace as w4a16_gemm (w4a16_workspace_bytes(M, K, N, 128) suffices).
 * Replaces post_attention_layernorm / input_layernorm followed by gate_up_proj / qkv_proj
 * (qwen3.py:166-173 with layernorm.py:28-40). */
int w4a16_gemm_rmsnorm_stats(const float* s, const float* ssq, const uint16_t* norm_weight, float eps,
                             uint16_t* x_norm, const int32_t* packed, const int32_t* qzeros,
                             const uint16_t* scales, uint16_t* y, int M, int K, int N, int group_size,
                             int silu_mul, void* workspace, size_t workspace_bytes, void* stream);

/* Kernel family w4a16_gemm launches for (M, K, N): a w4a16_regime_id.
 * Replaces the dispatch rule of select_awq_cuda_split_k (awq_cuda.py:17-26) and
 * AWQLinearMethod.apply (awq.py:115-154) as the thing a caller can query. */
int w4a16_regime(int M, int K, int N);

/* Number of K splits w4a16_gemm uses for (M, K, N) (1 = no cross-workgroup reduction).
 * Counterpart of select_awq_cuda_split_k (awq_cuda.py:17-26). */
int w4a16_split_k(int M, int K, int N);

/* The kernel configuration an entry point chooses for (M, K, N), written to out[5] as
 * {regime, p0, p1, p2, split} in w4a16_gemm_config's terms.  entry: 0 = w4a16_gemm (and
 * w4a16_gemm_residual, w4a16_gemm_residual_stats), 1 = w4a16_gemm_silu_mul, 2 and 3 =
 * w4a16_gemm_rmsnorm_stats without and with silu_mul (M <= 8), 4 = the decode kernel's own
 * plan (M <= 64), which w4a16_gemm runs below M = 32.  No reference counterpart: an
 * introspection hook for tuning and benchmarks. */
int w4a16_plan(int M, int K, int N, int entry, int* out);

/* w4a16_gemm with the kernel configuration forced instead of chosen: regime
 * W4A16_REGIME_DECODE (p0 = 16-column tiles per workgroup in {1,2,3,4,6} dividing N/16,
 * p1 = waves per workgroup in {4,8} (or 12 with p0 = 1), p2 = 128-row groups in flight per
 * wave in {1,2,4}, M <= 64; configurations whose LDS exceeds 156 KiB or whose accumulators and load ring
 * exceed 176 registers per lane are rejected) or W4A16_REGIME_TILE (p0 = 16-row tiles per
 * wave in {2,4,6,8}, p1 = waves per SIMD the register allocation targets, p2 = wave layout: 0 or 1 =
 * 4 waves of 64 columns, 2 = 2 x 4 waves of 64 columns, 3 = 8 waves of 32 columns,
 * 4 = 4 K slices x 2 waves of 32 columns, 5 = 2 K slices x 4 waves of 32 columns,
 * 6 = 2 K slices x 2 waves of 32 columns, 7 = 4 K slices x 1 wave of 32 columns,
 * 9 = 4 K slices x 3 waves of 32 columns, 10 = 2 K slices x 6 waves of 32 columns, the K
 * slices of a workgroup summed through LDS, 8 = 8 waves of 64 columns, 11 = 8 waves of 48
 * columns (plain GEMM only, N a multiple of 48); the compiled (p0, p2, p1) are (4,1,1),
 * (4,1,2), (8,1,1), (4,2,2), (4,3,2), (8,3,2), (2,4,2), (4,4,2), (2,5,2), (4,5,2), (8,5,2),
 * (4,6,1), (8,6,1), (2,7,1), (4,7,1), (8,8,2), (4,9,3), (2,9,3), (4,10,3), (8,11,2),
 * (4,11,2), (6,3,2), (6,8,2), (6,11,2));
 * 1 <= split <= K/128.  No reference counterpart: a tuning and testing hook (it exercises
 * every split-K reduction path at small sizes). */
int w4a16_gemm_config(const uint16_t* x, const int32_t* packed, const int32_t* qzeros,
                      const uint16_t* scales, uint16_t* y, int M, int K, int N, int group_size,
                      int regime, int p0, int p1, int p2, int split, void* workspace,
                      size_t workspace_bytes, void* stream);

/* w4a16_gemm_silu_mul with the kernel configuration forced, as w4a16_gemm_config (decode
 * p0 must be even).  No reference counterpart: a testing hook. */
int w4a16_gemm_silu_mul_config(const uint16_t* x, const int32_t* packed, const int32_t* qzeros,
                               const uint16_t* scales, uint16_t* y, int M, int K, int N,
                               int group_size, int regime, int p0, int p1, int p2, int split,
                               void* workspace, size_t workspace_bytes, void* stream);

/* Workspace bytes w4a16_gemm_config needs for that configuration (for the tile regime,
 * enough for every wave layout).  No reference counterpart. */
size_t w4a16_workspace_bytes_config(int M, int N, int regime, int p0, int split);

/* ---------------------------------------------------------------------------
 * Attention over a key/value cache held in 4 bits.  The reference keeps its cache in bf16 and
 * calls flash-attn (attention.py:21-133); these entry points take the place of that store and
 * attention, and of the slot maps and block tables that its model runner builds on the host.
 *
 * Cache: bytes [num_blocks, KV, block_size * (D + 8)], one page per (block, kv head), D in
 * {64, 128}, block_size a power of two in 16 .. 256.  A row (one token of one kv head) is D
 * codes c in 0 .. 15 with one bf16 scale s and one zero point z in 0 .. 15; a channel's value is
 * s * (c - z).  A page holds, in 32-bit words of eight channels (AutoAWQ's nibble order), the
 * tokens' keys [token][word], then their values [token / 4][word][token % 4], then one word a
 * token for the keys and one for the values: bf16(s) in the high half, bf16(128 + z) in the low.
 * A slot is block * block_size + token; slots outside the cache name no row.  Tables, slots and
 * lengths are int32 on the device and are never trusted: an id or length that points outside
 * the cache, the tables or the packed rows reads and writes nothing there.  A table's row reaches at
 * most 2^31 - 2^19 - 1 tokens (width * block_size).
 * ------------------------------------------------------------------------- */

/* One step's bookkeeping from the request lengths.  Request r has context_lens[r] tokens in the
 * cache and brings query_lens[r] new ones (0 for a padded request; negative lengths count as 0);
 * its cached tokens' blocks are the first ones of tables[r].  Writes cu_query_lens [R + 1] (the
 * requests' offsets among the packed rows), seq_lens [R] = context + query, and, for each of T
 * packed rows, its position in its sequence and its cache slot; rows behind the last request
 * get position 0 and slot -1.  Blocks that new tokens open are taken from free_blocks
 * [num_free], in order of request and position, and entered in tables (row stride table_stride
 * elements); blocks_used [1] receives how many are needed.  A token whose block the free list or
 * the table's width lacks gets slot -1 (and -1 in the table).  The lists are not consumed: the
 * same call again gives the same result.  R <= 4096, T <= 2^18, and a query counts as at most 2^18
 * rows.  T < sum(query_lens) drops the last rows: they have no position and no slot, but offsets,
 * lengths, blocks_used and tables count them.  Replaces the host loops of prepare_prefill /
 * prepare_decode (model_runner.py:279-333). */
int w4a16_kv_step(const int32_t* query_lens, const int32_t* context_lens, int32_t* tables,
                  int64_t table_stride, const int32_t* free_blocks, int32_t* cu_query_lens,
                  int32_t* seq_lens, int32_t* positions, int32_t* slots, int32_t* blocks_used, int R,
                  int width, int num_free, int block_size, int T, void* stream);

/* Quantize rows k, v [T, KV, D] (bf16, unit stride along D, the other strides in elements and
 * multiples of 8, 16-byte aligned) into the cache at slots [T]; rows of a slot outside the cache
 * are skipped, live slots must differ.  Per row: the range [min(x, 0), max(x, 0)] in 15 steps,
 * s = bf16(range / 15), z = min(round(-min / s), 15), c = clamp(round(x / s) + z, 0, 15), round
 * half to even.  A row with a NaN or infinity is stored as NaN; one whose scale rounds to zero
 * as zeros.  Replaces store_kvcache (attention.py:21-57). */
int w4a16_kv_store(const uint16_t* k, int64_t k_stride_t, int64_t k_stride_h, const uint16_t* v,
                   int64_t v_stride_t, int64_t v_stride_h, uint8_t* cache, const int32_t* slots, int T,
                   int KV, int D, int num_blocks, int block_size, void* stream);

/* The rows at slots [T] as bf16(s * (c - z)), k and v [T, KV, D] contiguous and 16-byte aligned;
 * zeros for a slot outside the cache.  No reference counterpart (its cache is bf16). */
int w4a16_kv_load(const uint8_t* cache, const int32_t* slots, uint16_t* k, uint16_t* v, int T, int KV,
                  int D, int num_blocks, int block_size, void* stream);

/* Ints that w4a16_kv_attention counts its workgroups' arrivals in: zero when a call starts, left
 * zero by it.  Calls in flight at the same time must not share them. */
#define W4A16_KV_COUNTERS 1024

/* Bytes of workspace w4a16_kv_attention needs (its contents need no initialization and are not
 * kept; calls in flight at the same time must not share one). */
size_t w4a16_kv_attention_workspace(int T, int R, int H, int KV, int D, int block_size, int width,
                                    int max_query_len);

/* Causal attention of packed query rows q [T, H, D] (bf16, strides as in w4a16_kv_store) over
 * their sequences' cached keys and values, those of the rows themselves included (store first):
 * request r owns rows cu_query_lens[r] .. cu_query_lens[r + 1] - 1, the last tokens of its
 * seq_lens[r] (at most width * block_size are reached) on the pages of tables[r]; query head h
 * reads kv head h / (H / KV).  out [T, H, D] (bf16, contiguous) = softmax(scale * q k^T) v with
 * fp32 scores, statistics and sums.  The second product's operands are p * s_v in 16 bits and exact
 * codes; for requests of more than 64 rows a kv head, all operands are fp16 with a power of two
 * taken out of each query row and of every 16 keys: a key or value whose scale is 2^-24 of the
 * largest among its 16, seen by the row or not, loses bits.  Sums are fp32 and have terms of up to
 * 143 |q| and 143 scales of values: a row with queries or values of 2^110 and more may be infinite
 * or NaN.  A row with a score beyond 2^26 (2^30 for requests of up to 64 rows a kv head) may be NaN
 * or zero: the exponents' own rounding leaves the weights' range there.  tree_mask (may be null) [T]: row t then sees its request's cached tokens and, instead of
 * the earlier new ones, those new ones j < 64 whose bit j is set.
 * A row that sees no key gives zeros; keys on a page id outside the cache are not seen; NaN and
 * infinities in keys that a row does not see have no effect on it.  Rows of no request (before
 * cu_query_lens[0], behind cu_query_lens[R]) are set to zero if zero_tail, else left as they are;
 * offsets that decrease anywhere name no rows at all.  max_query_len (>= 1) is a hint that chooses
 * kernels and grid: the longest query of the batch; results are right for any, if not the same bits.
 * out may be q where that is contiguous, and overlaps no other operand.  scale > 0 and scale * log2(e)
 * finite; H % KV == 0.  Replaces flash_attn_varlen_func / flash_attn_with_kvcache (attention.py:
 * 118-132). */
int w4a16_kv_attention(const uint16_t* q, int64_t q_stride_t, int64_t q_stride_h, const uint8_t* cache,
                       const int32_t* tables, int64_t table_stride, const int32_t* seq_lens,
                       const int32_t* cu_query_lens, const uint64_t* tree_mask, uint16_t* out, float scale,
                       int T, int R, int H, int KV, int D, int num_blocks, int block_size, int width,
                       int max_query_len, int zero_tail, void* workspace, size_t workspace_bytes,
                       int32_t* counters, void* stream);

/* ---------------------------------------------------------------------------
 * From the QKV projection to attention: per-head norms and position rotation, the same on the way
 * into the 4-bit cache, and attention of whole prompts over their own keys and values.
 * ------------------------------------------------------------------------- */

/* Per-head RMSNorm and position rotation of q [T, H, D] and k [T, KV, D] (bf16, strides as in
 * w4a16_kv_store, D in {64, 128}) into q_out and k_out (contiguous, overlapping no input), T up to 2^26 - 32.  A row x
 * becomes y = x * r * w with r = 1 / sqrt(mean(x^2) + eps) and the weight w [D] (q_weight, k_weight;
 * null: y = x), and channels i and i + rotary / 2 of y turn by the angle of the row's position:
 *   z[i] = y[i] cos - y[i + rotary / 2] sin,  z[i + rotary / 2] = y[i + rotary / 2] cos + y[i] sin;
 * channels from rotary on are y.  table [table_rows, rotary] (fp32) holds a position's rotary / 2
 * cosines, then its sines; rotary is a multiple of 16 up to D.  A row whose position [T] lies outside
 * the table becomes NaN.  The sum of squares is fp64, r the nearest fp32, every other step one fp32
 * operation in the order written, and z is rounded to bf16 once (a row whose mean square passes fp32's
 * range, of sizes from 2^64 on, becomes zero).  Replaces q_norm, k_norm and
 * rotary_emb of the reference's attention (qwen3.py:87-94, rotary_embedding.py:37-48), which round
 * after each of their steps. */
int w4a16_qk_norm_rope(const uint16_t* q, int64_t q_stride_t, int64_t q_stride_h, const uint16_t* k,
                       int64_t k_stride_t, int64_t k_stride_h, const int32_t* positions,
                       const float* table, int table_rows, int rotary, const uint16_t* q_weight,
                       const uint16_t* k_weight, float eps, uint16_t* q_out, uint16_t* k_out, int T,
                       int H, int KV, int D, void* stream);

/* w4a16_qk_norm_rope, and w4a16_kv_store of the keys it gives (the bf16 ones) and of v, in one
 * launch: the same bits.  k_out may be null.  Rows of a slot outside the cache are not stored (q_out
 * and k_out get them). */
int w4a16_kv_append(const uint16_t* q, int64_t q_stride_t, int64_t q_stride_h, const uint16_t* k,
                    int64_t k_stride_t, int64_t k_stride_h, const uint16_t* v, int64_t v_stride_t,
                    int64_t v_stride_h, uint8_t* cache, const int32_t* slots, const int32_t* positions,
                    const float* table, int table_rows, int rotary, const uint16_t* q_weight,
                    const uint16_t* k_weight, float eps, uint16_t* q_out, uint16_t* k_out, int T, int H,
                    int KV, int D, int num_blocks, int block_size, void* stream);

/* Bytes of workspace w4a16_prompt_attention needs (as w4a16_kv_attention_workspace); fewer rows and
 * requests need no more. */
size_t w4a16_prompt_attention_workspace(int T, int R, int H, int KV, int D);

/* Causal attention of whole prompts over their own keys and values: q [T, H, D], k and v [T, KV, D]
 * (bf16, strides as in w4a16_kv_store; rows 0 to 2^22 elements apart, q's heads of a kv head within
 * 2^28; H <= 2^14), sequence r being rows cu_query_lens[r] .. cu_query_lens[r + 1] - 1 of all three.
 * Its row t sees its rows 0 .. t; query head h reads kv head h / (H / KV).  out [T, H, D] (bf16,
 * contiguous) = softmax(scale * q k^T) v with fp32 scores, statistics and sums; the weights, up to 2^8
 * of the row's largest, are rounded to bf16 for the second product (so that values beyond 2^119
 * divided by the row's number of keys may overflow in the sum).  NaN and infinities in keys and
 * values that a row does not see have no effect on it; an infinite value that it sees gives infinity in
 * its channel, or NaN where its weight underflows.  Scores, also times scale log2(e), are fp32: a row
 * all of whose scores are minus infinity or below that range is zero, as in w4a16_kv_attention, and one
 * that has a score above it is NaN.  T up to 2^18 with any R, H up to 128 and H / KV up to 16; other
 * sizes while their work counts in 32 bits (W4A16_ERR_SHAPE otherwise).  Rows of no sequence,
 * offsets that decrease, zero_tail, workspace and counters are as in w4a16_kv_attention.  out may be q
 * where that is contiguous, and overlaps no other operand.  Replaces the reference's attention of
 * prompts where nothing is cached (attention.py:118-125). */
int w4a16_prompt_attention(const uint16_t* q, int64_t q_stride_t, int64_t q_stride_h, const uint16_t* k,
                           int64_t k_stride_t, int64_t k_stride_h, const uint16_t* v, int64_t v_stride_t,
                           int64_t v_stride_h, const int32_t* cu_query_lens, uint16_t* out, float scale,
                           int T, int R, int H, int KV, int D, int zero_tail, void* workspace,
                           size_t workspace_bytes, int32_t* counters, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* W4A16_H_ */
