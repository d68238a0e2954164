/*
 * nemo_ops.h -- kernel-level C ABI of libnemo_b200.so.
 *
 * One entry point per device kernel of the forward pass, on caller-owned
 * device memory (plain device pointers as void*), so each kernel can be
 * checked on its own against the CPU oracle. These stand where the
 * reference's per-kernel `createRun` / `encode` pairs stand
 * (src/webgpu/ops.ts, src/webgpu/quant-matmul.ts): same inputs, same
 * outputs, packed valid-token rows instead of padded [batch x sequence] rows.
 * Unless its comment says otherwise, a call launches on the legacy default
 * stream and synchronises before it returns; errors follow nemo.h.
 */
#ifndef NEMO_OPS_H
#define NEMO_OPS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Weight block formats for nemo_op_decode. */
#define NEMO_FMT_Q4_K 0         /* GGUF row-major 144-byte blocks, quantization.ts:19-38 */
#define NEMO_FMT_Q6_K 1         /* GGUF row-major 210-byte blocks, quantization.ts:46-74 */
#define NEMO_FMT_Q4_0 2         /* GGUF row-major 18-byte blocks, quantization.ts:40-44 */
#define NEMO_FMT_Q4_0_TILE32 3  /* q4_0-tile32-compact, format.ts:65-99 / quant-matmul.ts:99-108 */

/* Decodes a [rows x k] quantised matrix: out16 receives f16(value) (the
 * effective weights of every reference matmul pipeline), out32 (optional)
 * the exact f32 value of the CPU decoders. */
int nemo_op_decode(int fmt, const void* d_src, int rows, int k, void* d_out16, void* d_out32);

/* Size in bytes of the per-run metadata block the ops below take. */
size_t nemo_op_meta_bytes(void);
/* Builds the metadata of a run from d_lengths [batch] (model.ts:226-233). */
int nemo_op_meta(const void* d_lengths, int batch, int sequence, void* d_meta);
/* Device ints inside the metadata block: valid tokens before / after the merge. */
void* nemo_op_meta_tokens(void* d_meta, int merged);

/* ops.ts:680-725: d_ids [batch*sequence] u32 padded rows, Q6_K table ->
 * d_x [tokens x 2048] f16 (packed valid tokens). */
int nemo_op_embedding(const void* d_ids, const void* d_table, int vocab, const void* d_meta,
                      int max_tokens, void* d_x);

/* ops.ts:21-72: x (+)= residual (stored f16), norm = f16(x*rsqrt(mean x^2+1e-5)*w).
 * d_residual may be NULL; *d_rows (device int) rows of width 2048. */
int nemo_op_rmsnorm(void* d_x, const void* d_residual, const void* d_w, void* d_norm,
                    const void* d_rows, int max_rows);

/* model.ts:95-107 on the host: the YaRN RoPE table [sequence x 64 x (cos,sin)] f32. */
int nemo_rope_table(int sequence, float* out);

/* ops.ts:168-194: d_qkv [tokens x 5120] -> d_q [tokens x 3072], d_k [tokens x 1024]. */
int nemo_op_rope(const void* d_qkv, const void* d_table, const void* d_meta, int merged,
                 int max_tokens, void* d_q, void* d_k);

/* ops.ts:213-362: bidirectional GQA attention with the >2048 stride-3 key
 * sampling; V read from d_qkv columns 4096..5119. d_out [tokens x 3072]. */
int nemo_op_attention(const void* d_q, const void* d_k, const void* d_qkv, const void* d_meta,
                      int merged, int batch, int max_len, void* d_out);

/* Same attention on the tcgen05 tensor cores (the kernel the plans run).
 * d_q, d_k, d_qkv hold `rows` token rows (rows >= the metadata's token count);
 * sampled layers (> 2048 valid keys) gather their keys into scratch buffers
 * this call allocates. */
int nemo_op_attention_tc(const void* d_q, const void* d_k, const void* d_qkv, const void* d_meta, int merged,
                         int batch, int max_len, int rows, void* d_out);

/* nemo_op_attention_tc without any device allocation. No counterpart in the
 * reference: it is for hosts that cannot call cudaMalloc/cudaFree where
 * attention runs (device memory owned by another allocator or reserved up
 * front; cudaFree would synchronise the whole device under a latency-bound
 * server). Its scratch is one fixed device array of 8 MiB + 256 B per GPU,
 * held until exit. The call reads d_meta back to learn how many sampled key
 * rows the run needs (requests longer than 2048 keep every third key; none in
 * exact-attention metadata) and fails with NEMO_ERR_ARGS when that exceeds
 * 2048. All calls share the array: calls that overlap on the GPU race. The
 * first call on a device looks up the array's address; make it before any
 * stream capture. Same arguments and results as nemo_op_attention_tc. */
int nemo_op_attention_tc_noalloc(const void* d_q, const void* d_k, const void* d_qkv, const void* d_meta, int merged,
                                 int batch, int max_len, int rows, void* d_out);

/* ops.ts:74-89: [rows x 12288] (gate | up) -> [rows x 6144]. */
int nemo_op_swiglu(const void* d_gate_up, const void* d_rows, int max_rows, void* d_out);

/* ops.ts:629-661 applied to x and normalized: -> d_xm, d_nm [merged tokens x 2048]. */
int nemo_op_merge(const void* d_x, const void* d_norm, const void* d_meta, int max_out, void* d_xm,
                  void* d_nm);

/* ops.ts:596-616: d_norm merged rows -> d_out [batch x 2048] f32, L2-normalised. */
int nemo_op_pool(const void* d_norm, const void* d_meta, int batch, void* d_out);

/* Projection GEMM Y[M x N] = X[M x K] . W[N x K]^T (f16 in, f32 accumulate,
 * f16 out; quant-matmul.ts:438-563 with f32 accumulation). impl 0 = CUDA-core
 * validation kernel, impl 1 = tcgen05 tensor-core kernel (bn = 64/128/256).
 * M = *d_rows <= max_rows; d_x has max_rows rounded up to 128 rows. */
int nemo_op_gemm(int impl, const void* d_x, const void* d_w, void* d_y, const void* d_rows,
                 int max_rows, int n, int k, int bn);

/* Standalone quantised matmul, the operation of the reference's
 * QuantMatmulKernel (src/webgpu/quant-matmul.ts:438-563: a GGUF Q4_K / Q6_K /
 * Q4_0 or q4_0-tile32-compact weight buffer, an [m x k] f16 activation buffer,
 * K divisible by 256, quant-matmul.ts:513), with f32 output:
 *   Y[m x n] = X[m x k] . W[n x k]^T, W = f16(decode(blocks)).
 * fmt is a NEMO_FMT_* value; n must be a multiple of 128.
 *
 * nemo_op_qmatmul_image_bytes / nemo_op_qmatmul_image re-tile the blocks on
 * the device into the tile-slab image the projection kernels stream (what
 * model load does for every projection); d_image is 256-byte aligned device
 * memory of that size. nemo_op_qmatmul_enqueue runs the matmul on an image
 * asynchronously on `stream` (a cudaStream_t, NULL = legacy default stream):
 * the fused-dequant split-K kernel for m <= 64, the dequant-fused batched GEMM
 * above. d_err is a zeroed 4-byte device word that becomes nonzero if a
 * bounded wait gave up. nemo_op_qmatmul does all of it on packed blocks and
 * synchronises (it allocates the image and error word and frees them). */
size_t nemo_op_qmatmul_image_bytes(int fmt, int n, int k);
int nemo_op_qmatmul_image(int fmt, const void* d_packed, int n, int k, void* d_image);
int nemo_op_qmatmul_enqueue(int fmt, const void* d_image, const void* d_x, int m, int n, int k, void* d_y,
                            void* d_err, void* stream);
int nemo_op_qmatmul(int fmt, const void* d_packed, const void* d_x, int m, int n, int k, void* d_y);

/* Decode of a tile-slab image by the per-row decoders every projection kernel
 * runs (the same launch model load uses to build the batched path's f16
 * weights): d_w16 = f16(decode(blocks)) as a row-major [n x k] f16 matrix,
 * 16-byte aligned. Replaces the reference's dequantisation for parity checks:
 * src/gguf/quantization.ts:19-74 rounded to f16 as quant-matmul.ts:106 does.
 * Synchronises. */
int nemo_op_qmatmul_image_decode(int fmt, const void* d_image, int n, int k, void* d_w16);

/* --- Layer operators beside the fixed-shape encoder -------------------------
 * Operators of a transformer layer for other shapes and types than the
 * encoder's own: residual RMSNorm with an 8-bit output, rotary embedding,
 * 4-bit group-quantised matrix-vector product, windowed attention. No
 * counterpart in the reference.
 *
 * They are asynchronous: each enqueues its kernel on `stream` (a cudaStream_t,
 * NULL = legacy default stream) and returns. They allocate nothing, keep
 * nothing between calls, use no workspace and can be captured into CUDA
 * graphs; calls on different streams are independent of one another. Every
 * buffer is device memory of one device, which need not be the current one;
 * `stream` belongs to that device. Leading dimensions (ld*) count elements
 * between the starts of consecutive rows. Zero rows, tokens or requests is a
 * valid call that does nothing. Inputs and outputs do not overlap unless an
 * entry says so. Results do not depend on the launch: the same call on the
 * same inputs gives the same bits. */
#define NEMO_DTYPE_F16 0
#define NEMO_DTYPE_BF16 1
#define NEMO_DTYPE_F32 2
#define NEMO_DTYPE_E4M3 3 /* 8-bit float, 4 exponent and 3 mantissa bits, largest value 448 */
#define NEMO_DTYPE_I8 4

/* Residual RMSNorm with an 8-bit output. For each row of `width` columns, in
 * f32:
 *   s = x + residual (s = x with d_residual NULL); d_sum = s rounded to dtype;
 *   u = s * w; for each group of `group` columns top = max|u| and
 *   q = round(u * (Q / top)), scale = top / Q / sqrt(mean(s^2) + eps),
 * Q = 448 for NEMO_DTYPE_E4M3 and 127 for NEMO_DTYPE_I8, both rounded to
 * nearest even, so that q * scale is the normalised row. dtype (x, residual,
 * sum) is F16 or BF16, d_w f32 [width]. group is 32, 64 or 128 (the last group
 * of a row may be shorter), or 0 for one scale per row; d_scales is f32
 * [rows x ceil(width / group)]. d_sum is NULL exactly when d_residual is; it
 * may be d_x or d_residual themselves (with the same ld). A group whose top is
 * at most 1e-30 has codes 0; one that holds an infinity or a NaN has codes 0
 * and a NaN scale. mean(s^2) is an f32 sum too: values whose squares leave its
 * range (above 1e19 / sqrt(width); with eps 0, below 1e-19) have no useful
 * scale. width <= 32768. Rows of 16-byte multiples with 16-byte
 * aligned buffers (8-byte for d_q) are read and written as vectors; others
 * work, slower. */
int nemo_op_rmsnorm_q8(int dtype, const void* d_x, int64_t ldx, const void* d_residual, int64_t ldr, const void* d_w,
                       int rows, int width, float eps, void* d_sum, int64_t lds, int out_dtype, int group, void* d_q,
                       int64_t ldq, void* d_scales, void* stream);

/* Rotary embedding of q and k: element pair i of the first rotary_dim columns
 * of each head turns by t = position * inv_freq[i],
 *   (a, b) -> magnitude * (a cos t - b sin t, a sin t + b cos t),
 * computed in f32 with t reduced in 64 bits (positions up to 2^31 - 1 keep
 * their angle); columns from rotary_dim to head_dim are copied. layout
 * NEMO_ROPE_PAIRS pairs columns (2i, 2i + 1), NEMO_ROPE_HALVES (i,
 * i + rotary_dim / 2). q rows hold q_heads heads of head_dim columns, k rows
 * k_heads; heads follow one another, rows are ldq / ldk apart (a column range
 * of a QKV buffer is fine). d_k may be NULL with k_heads 0. d_inv_freq f64
 * [rotary_dim / 2], d_positions int32 [tokens]. d_qo may be d_q with ldqo ==
 * ldq, and d_ko d_k (in place). dtype F16 or BF16; rotary_dim even and at most
 * head_dim; head_dim <= 512. */
#define NEMO_ROPE_PAIRS 0
#define NEMO_ROPE_HALVES 1
int nemo_op_rope_apply(int dtype, int layout, const void* d_q, int64_t ldq, int q_heads, const void* d_k, int64_t ldk,
                       int k_heads, int head_dim, int rotary_dim, const void* d_inv_freq, float magnitude,
                       const void* d_positions, int tokens, void* d_qo, int64_t ldqo, void* d_ko, int64_t ldko,
                       void* stream);

/* Inverse frequencies for nemo_op_rope_apply, on the host: out [rotary_dim / 2]
 * f64 and *magnitude. With f_i = theta^(-2i / rotary_dim):
 *   NEMO_ROPE_PLAIN   f_i
 *   NEMO_ROPE_LINEAR  f_i / factor
 *   NEMO_ROPE_NTK     theta' = theta * factor^(r / (r - 2)), r = rotary_dim >= 4
 *   NEMO_ROPE_YARN    f_i / factor blended into f_i over the pairs that turn
 *                     between `slow` (1) and `fast` (32) times in
 *                     original_context positions (boundaries rounded outwards
 *                     to whole pairs, as in nemo_rope_table), *magnitude =
 *                     0.1 ln(factor) + 1
 *   NEMO_ROPE_RAMP    the same blend over the number of turns itself
 *                     (slow 1, fast 4): f_i / factor below `slow` turns, f_i
 *                     above `fast`, magnitude 1
 * *magnitude is 1 for the others. factor >= 1; original_context, slow and fast
 * (0 < slow < fast) are read by the last two only. */
#define NEMO_ROPE_PLAIN 0
#define NEMO_ROPE_LINEAR 1
#define NEMO_ROPE_NTK 2
#define NEMO_ROPE_YARN 3
#define NEMO_ROPE_RAMP 4
int nemo_rope_inv_freq(int scaling, double theta, int rotary_dim, double factor, double original_context, double slow,
                       double fast, double* out, float* magnitude);

/* Matrix-vector products with 4-bit weights and group scales, for up to 16
 * rows of x at once:
 *   y[m x n] = x[m x k] . W[n x k]^T,  W[r][c] = scale[r][c / group] * (q[r][c] - zero[r][c / group]).
 * d_w4 holds two columns per byte, the even one in the low four bits
 * ([n x k / 2] bytes, 16-byte aligned); d_scales [n x k / group] of scale_dtype
 * (F16 or BF16); d_zeros packs the zero points the same way ([n x
 * ceil(k / group / 2)] bytes), NULL = 8 everywhere. group is 32, 64 or 128 and
 * divides k. x is F16, BF16, E4M3 or I8; 8-bit codes take d_x_scales f32
 * [m x ceil(k / x_group)], x_group 32, 64 or 128, or >= k for one scale per
 * row (as nemo_op_rmsnorm_q8 writes them, where group 0 is x_group >= k);
 * 16-bit x takes NULL. y is F16, BF16 or F32. Sums are f32 or finer and y is
 * rounded once; 16-bit elements of x below 2^-19 of the largest of their 32 to
 * 128 neighbours may be rounded to 2^-30 of it. A sum of x * (q - zero) over one
 * group must stay within f32 (it does for |x| up to 2^116). An infinity or NaN in a row of
 * x makes its row of y infinite or NaN. m > 16 is refused: more rows take a call
 * for each 16 of them, which reads the weights each time (no other entry takes
 * this format). n and k are at most 2^30. d_x and ldx need the alignment of one
 * element only. */
int nemo_op_w4_matvec(int x_dtype, const void* d_x, int64_t ldx, const void* d_x_scales, int x_group, const void* d_w4,
                      int scale_dtype, const void* d_scales, const void* d_zeros, int group, int m, int n, int k,
                      int y_dtype, void* d_y, int64_t ldy, void* stream);

/* On the host, how nemo_op_w4_matvec runs a call of these sizes on a device of
 * `sms` SMs: *digits 1 if x goes as 8-bit digits, 0 as 16-bit products; *rows
 * weight rows and one of *slices column slices a warp; rows of x in *panels;
 * *blocks blocks of *shared_bytes. (x_group is read for 8-bit x only.) */
int nemo_op_w4_matvec_form(int x_dtype, int x_group, int group, int m, int n, int k, int sms, int* digits, int* rows,
                           int* slices, int* panels, int* blocks, int* shared_bytes);

/* Grouped-query attention with a sliding window and first tokens that stay
 * visible, for prompts, whole documents and single tokens against a cache.
 * Request b has the query rows d_q_off[b] .. d_q_off[b + 1] - 1 (int32
 * [batch + 1], ascending) and the key rows d_k_start[b] .. + d_k_len[b] - 1
 * (int32 [batch] each), so keys may be packed like the queries or lie in a
 * cache with room behind them. Its queries are the last ones of its keys:
 * query i has position p = i + key length - query length, and sees key j iff
 *   j < key length  and  (right < 0 or j <= p + right)
 *   and  (left < 0 or j >= p - left or j < sinks).
 * right 0 is causal, right < 0 with left < 0 bidirectional. A query that sees
 * no key, or whose scores are all -infinity, gets zeros. Scores are q . k *
 * scale with an f32 softmax, weights are rounded to dtype for the product with
 * v, which sums in f32. Infinities and NaN in keys or values that a query does
 * not see do not reach its row; a NaN that it sees makes its columns of the row
 * NaN, or the whole row if it is in a score (as does a score of +infinity).
 * Finite values never give an infinite result. dtype F16 or BF16; head_dim 64 or 128; q_heads
 * a multiple of kv_heads; heads follow one another within a row; batch and
 * heads at most 65535; buffers 16-byte aligned, leading dimensions multiples
 * of 8. q_rows, k_rows: rows of the buffers, in which the offsets have to lie.
 * Requests may share keys. max_q: the longest query length (rows past it are
 * not written). max_k: about the longest key length, which only steers the
 * split of the work. Rows of d_out that no request covers stay as they are.
 * d_err is a zeroed 4-byte device word that becomes nonzero if a bounded wait
 * gave up. */
int nemo_op_attention_window(int dtype, const void* d_q, int64_t ldq, const void* d_k, int64_t ldk, const void* d_v,
                             int64_t ldv, int q_heads, int kv_heads, int head_dim, const void* d_q_off,
                             const void* d_k_start, const void* d_k_len, int batch, int q_rows, int k_rows, int max_q,
                             int max_k, int left, int right, int sinks, float scale, void* d_out, int64_t ldo,
                             void* d_err, void* stream);

/* On the host, how nemo_op_attention_window runs a call of these sizes on a
 * device of `sms` SMs that can place clusters of max_cluster blocks (16 on a
 * whole B200): *tiles 1 on 128-query tensor-core tiles, 0 on 16-row ones, whose
 * keys *splits blocks of a cluster share. */
int nemo_op_attention_window_form(int q_heads, int kv_heads, int head_dim, int batch, int q_rows, int k_rows, int max_q,
                                  int max_k, int left, int right, int sinks, int sms, int max_cluster, int* tiles,
                                  int* splits);

/* Routing of the head-parallel path (no reference counterpart; the index
 * functions its QKV GEMM and attention epilogues use, exported for layout
 * tests without a GPU), n_devices in {2, 4, 8}:
 * nemo_hp_qkv_route: for each QKV column c < 5120, the device that owns its
 *   head group, the buffer there (0 Q, 1 K, 2 V) and the column in it;
 * nemo_hp_row_owner: for positions 0..n_positions-1 of a request sharded in
 *   rows_per_device-row shards (the last one shorter), the owning device. */
int nemo_hp_qkv_route(int n_devices, int* device, int* buffer, int* column);
int nemo_hp_row_owner(int n_devices, int rows_per_device, int n_positions, int* device);

#ifdef __cplusplus
}
#endif
#endif /* NEMO_OPS_H */
