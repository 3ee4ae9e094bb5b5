/*
 * dionw_hip.h — C ABI of libdionw_hip.so, the MI355X (gfx950) kernels of the
 * Dion optimizer step.
 *
 * Conventions
 *  - Every function returns 0 on success, 1 for a rejected argument and 2 for
 *    a failed launch; dionw_last_error() holds the message (per thread).
 *  - Pointers are device pointers unless named otherwise; pointer *arrays*
 *    (grads, params, ...) are host arrays of device pointers, copied into the
 *    kernel arguments (no device table, no host synchronization).
 *  - Every launch is asynchronous on `stream`. The library never allocates,
 *    frees or synchronizes: buffers and workspaces come from the caller.
 *  - Matrices are row-major. A bucket run's momentum is [blocks, rows, cols]
 *    float32 and contiguous; every tensor of a run holds blocks_per_tensor
 *    blocks (rows_per_tensor = blocks_per_tensor * rows rows).
 *  - Element codes: 0 = float16, 1 = bfloat16, 2 = float32.
 *
 * Citations are to the reference implementation (JTriggerFish/dionw, src/dionw).
 */
#ifndef DIONW_HIP_H
#define DIONW_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct ihipStream_t* dionw_stream_t; /* hipStream_t */

/* Last error message of the calling thread ("" when none). */
const char* dionw_last_error(void);

/* ABI revision of this header (2). */
int dionw_abi_version(void);

/*
 * Norm element type (the `elem` argument of the functions that form the
 * Newton-Schulz normalization): the element code of the iteration the sums
 * normalize. 0 (float16 Gram) and 2: sums of squares of the float32 values and
 * den = sqrt(sum) * safety + eps (the norm of x.float(), _gram.py:85-86).
 * 1 (bfloat16 quintics): sums of squares of the values rounded to bfloat16 and
 * den = float(bf16(sqrt(sum))) * safety + eps, the norm of the bf16 input taken
 * as a bf16 tensor (_polar_express.py:57-58, 89-92).
 */

/*
 * M += G for every row of a run, with each row's l1 norm (the top-k score) and
 * sum of squares. Replaces accumulate_row_l1 (_momentum_kernels.py:89-103)
 * and the per-parameter loop of _accumulate_with_scores (_matrix_step.py:188-199).
 * The score is an fp32 sum in a fixed order (per-lane float4 partials in
 * column order, then an xor butterfly over the 64 lanes).
 *   grads[count]: float32 gradients, rows_per_tensor x cols each, contiguous.
 *   momentum: [count * rows_per_tensor, cols]; scores, row_sumsq: one per row.
 *   elem: the norm element type (row_sumsq of the bf16-rounded sums when 1).
 */
int dionw_accumulate_scores(const float* const* grads, int32_t count, int64_t rows_per_tensor,
                            int64_t cols, float* momentum, float* scores, float* row_sumsq,
                            int32_t elem, dionw_stream_t stream);

/*
 * Per-row sum of squares of the every-row Newton-Schulz input U = M + G
 * (heavy ball) or G + mu (M + G) (Nesterov), without writing anything: the
 * first of the two passes that replace accumulate_copy_decay
 * (_momentum_kernels.py:106-133; _matrix_step.py:217-237). momentum may be
 * NULL (U = G: the standalone orthogonalization of a given matrix).
 */
int dionw_full_sumsq(const float* const* grads, int32_t count, int64_t rows_per_tensor,
                     int64_t cols, const float* momentum, float mu, int32_t nesterov,
                     float* row_sumsq, int32_t elem, dionw_stream_t stream);

/* den[b] = sqrt(sum of row_sumsq over block b's rows) * safety + eps (the
 * square root rounded to bf16 first for elem 1): the Frobenius normalization
 * of _gram.py:86 (safety 1) and _polar_express.py:92 (safety 1.02 for Polar
 * Express, 1 for Keller). */
int dionw_block_denom(const float* row_sumsq, int64_t blocks, int64_t rows, float safety,
                      float eps, float* den, int32_t elem, dionw_stream_t stream);

/*
 * The normalization prologue of the Orthogonalize plugin on a contiguous
 * [blocks, rows, cols] input x of elem x_elem (0 fp16, 1 bf16, 2 fp32), read
 * as it is: row sums of squares as dionw_full_sumsq forms them (into
 * row_sumsq, blocks * rows floats), den as dionw_block_denom (both with the
 * norm element type elem), then
 * X = 16-bit(x / den) of type elem (0 or 1) written as dionw_prepare_ns_input
 * writes it in every-row mode without momentum (out_rowmajor and/or
 * out_transposed, padded to p_pad x j_pad). Bit-identical to those three calls
 * on a float32 copy of x, without the copy. Replaces x.float() and the
 * division by the norm of _gram.py:85-86 and _polar_express.py:89-92.
 */
int dionw_normalize_input(const void* x, int32_t x_elem, int64_t blocks, int64_t rows,
                          int64_t cols, float safety, float eps, float* row_sumsq, float* den,
                          int64_t p_pad, int64_t j_pad, int32_t elem, void* out_rowmajor,
                          void* out_transposed, dionw_stream_t stream);

/*
 * Top-k rows of each block by score: replaces torch.topk(sorted=False) and the
 * index bookkeeping of _selected_update (_matrix_step.py:172-180).
 * Exact: ties at the k-th score take the lowest row indices.
 *   idx [blocks, k]: selected rows, ascending; slot [blocks, rows]: position
 *   of each row in idx or -1; den [blocks]: sqrt(sum of the selected rows'
 *   row_sumsq) * safety + eps, as dionw_block_denom forms it for elem.
 */
int dionw_select_rows(const float* scores, const float* row_sumsq, int64_t blocks, int64_t rows,
                      int64_t k, float safety, float eps, int32_t* idx, int32_t* slot,
                      float* den, int32_t elem, dionw_stream_t stream);

/*
 * One pass writing the decayed momentum and the Newton-Schulz input.
 * Selected mode (idx != NULL): U = M[idx] (pre-decay) and M[idx] *= mu
 * (_matrix_step.py:176-179). Every-row mode (idx == NULL, grads given):
 * M = mu (M + G), U = M + G or, with nesterov, G + mu (M + G).
 * Then X = U / den[b] rounded to float16 (elem 0), or bf16(bf16(U) / den)
 * (elem 1, the Keller / Polar Express input), written, if out_rowmajor !=
 * NULL, as [blocks, p_pad, j_pad] (row p = selected row p) and, if
 * out_transposed != NULL, as its transpose [blocks, j_pad, p_pad], zeros in
 * the padding; at least one must be given. In every-row mode momentum may be
 * NULL with write_m == 0 (U = G). elem 2 writes the raw float32 U as
 * [blocks, k, cols] (out_rowmajor required) for a user-supplied
 * orthogonalization.
 * Replaces the prologue of gram_polar_express (_gram.py:83-87) and the
 * normalization of quintic_triton (_polar_express.py:89-92).
 */
int dionw_prepare_ns_input(const float* const* grads, int32_t count, float* momentum,
                           const int32_t* idx, const float* den, int64_t blocks, int64_t rows,
                           int64_t cols, int64_t k, int64_t p_pad, int64_t j_pad, float mu,
                           int32_t nesterov, int32_t write_m, int32_t elem, void* out_rowmajor,
                           void* out_transposed, dionw_stream_t stream);

/*
 * Batched C = alpha * A B^T + beta * D on MFMA (fp32 accumulation, one
 * rounding). A [m, k], B [n, k], D and C [m, n], all row-major with the given
 * leading dimensions and batch strides (elements); ct (optional) receives C^T
 * [n, m]. symmetric: only the tiles on and above the diagonal are computed and
 * mirrored (m == n, output c only). elem 0 or 1: k, lda, ldb and the operand
 * batch strides must be multiples of 8 and the operands 16-byte aligned.
 * elem 2: float32 operands and output, products and sums in float32 on the
 * fp32 MFMA (the reference's "ieee" dot for float32 inputs), any sizes and
 * strides.
 * Replaces ns_line_1 (alpha A A^T, _symmetric_kernels.py:252-277), ns_line_2
 * (c A A^T + b A, :280-312) and the baddbmm/bmm products of _gram.py:46-69
 * and _polar_express.py:98-103.
 */
int dionw_gemm_nt(int32_t elem, int64_t batch, int64_t m, int64_t n, int64_t k, const void* a,
                  int64_t lda, int64_t stride_a, const void* b, int64_t ldb, int64_t stride_b,
                  const void* d, int64_t ldd, int64_t stride_d, float alpha, float beta, void* c,
                  int64_t ldc, int64_t stride_c, void* ct, int64_t ldct, int64_t stride_ct,
                  int32_t symmetric, dionw_stream_t stream);

/*
 * The five (a, b, c) rows dionw_newton_schulz uses for kind (out: 15 doubles,
 * row-major; the kernels take them rounded to float): the Gram table of
 * _gram.py:24-35 with the 1.05 safety folded in as (a/s, b/s^3, c/s^5), the
 * Polar Express table of _polar_express.py:28-34, Keller's row of
 * _keller.py:20. Host only: no device work.
 */
int dionw_ns_coefficients(int32_t kind, double* out);

/* Workspace bytes dionw_newton_schulz needs. */
size_t dionw_newton_schulz_workspace(int32_t kind, int64_t batch, int64_t r, int64_t c);

/*
 * Newton-Schulz orthogonalization of a batch of wide, normalized matrices:
 * the Orthogonalize plugin (newton_schulz.py:30, 43-68) after its prologue.
 *   kind 0 (GRAM): fp16 Gram Newton-Schulz with restart at iteration 2 when
 *     c > r (_gram.py:50-69), the standard Polar Express iteration when
 *     c == r (_gram.py:41-47); output bf16(fp16(.)).
 *   kind 1 (POLAR_EXPRESS_TRITON) / 2 (KELLER_TRITON): the bf16 quintic with
 *     each line rounded once (_polar_express.py:74-104; _keller.py:20-34).
 *   kind 3 (POLAR_EXPRESS) / 4 (KELLER): the bf16 quintic with the products
 *     A A and P X rounded to bf16 before the elementwise terms, as the
 *     reference's cuBLAS variant computes it (_polar_express.py:43-71).
 *   x [batch, r, c] and xt [batch, c, r] (the input and its transpose, both
 *   overwritten), r <= c multiples of 8. With r a multiple of 32 the products
 *   read x itself where they multiply it from the left: xt is then neither
 *   read nor written and may be NULL. The real r_real x c_real region of
 *   the result goes to out (bf16) with leading dimension out_ld and batch
 *   stride out_stride, transposed when out_transposed (tall blocks).
 */
int dionw_newton_schulz(int32_t kind, int64_t batch, int64_t r, int64_t c, void* x, void* xt,
                        int64_t r_real, int64_t c_real, void* out, int32_t out_transposed,
                        int64_t out_ld, int64_t out_stride, void* workspace,
                        size_t workspace_bytes, dionw_stream_t stream);

/*
 * dionw_newton_schulz for count independent bucket runs at once: element i of
 * every array is run i's argument. Runs whose product sequences match (same
 * kind and shape class) execute together, up to 8 at a time, one launch per
 * product of the sequence, so that small runs fill the CUs a large run's
 * launches leave idle. Results are bit-identical to count separate calls.
 * The runs' workspaces must not overlap (checked); all arguments are checked
 * before anything is launched. Replaces the per-run orthogonalize calls of a
 * step (_matrix_step.py:254-265, one per run of optimizer.py:351-369).
 */
int dionw_newton_schulz_group(int32_t count, const int32_t* kind, const int64_t* batch,
                              const int64_t* r, const int64_t* c, void* const* x,
                              void* const* xt, const int64_t* r_real, const int64_t* c_real,
                              void* const* out, const int32_t* out_transposed,
                              const int64_t* out_ld, const int64_t* out_stride,
                              void* const* workspace, const size_t* workspace_bytes,
                              dionw_stream_t stream);

/*
 * Product launches dionw_newton_schulz_group would issue for runs of these
 * shapes (which of their products it groups), or -1 for invalid arguments;
 * nothing is launched and no memory is touched. For one run it is the length
 * of that run's product sequence. Callers use it to keep runs apart when
 * grouping would save nothing (each run's passes then follow its own
 * iteration while its output is still in cache).
 */
int64_t dionw_newton_schulz_group_launches(int32_t count, const int32_t* kind,
                                           const int64_t* batch, const int64_t* r,
                                           const int64_t* c, const int64_t* r_real,
                                           const int64_t* c_real);

/*
 * NorMuon statistics of the orthogonalized rows O (bf16 [blocks, k, cols]):
 * v = lerp(v, mean(O^2), 1 - beta2) written back into variance [blocks, rows]
 * at the selected rows (idx [blocks, k], or every row when idx == NULL),
 * rowd [blocks, k] = sqrt(v) + 1e-8, and scale [blocks] =
 * ||O||_F / max(||O / rowd||_F, 1e-8) * step. scratch: 2 * blocks * k floats.
 * Replaces normalize_rows (_row_normalization.py:41-60).
 */
int dionw_normuon_stats(const void* orthogonal, int64_t blocks, int64_t k, int64_t rows,
                        int64_t cols, const int32_t* idx, float* variance, float beta2,
                        float step, float* rowd, float* scratch, float* scale,
                        dionw_stream_t stream);

/*
 * dionw_normuon_stats without the scratch argument: the per-row partial sums
 * go to a device array inside the library (4 MiB per GPU, held until the
 * process ends), so the call allocates nothing. No counterpart in the
 * reference: it is for callers that cannot allocate device memory (code under
 * HIP graph capture, tight serving loops, harnesses that forbid hipMalloc).
 * Limit: blocks * k <= 524288 selected rows; larger calls are rejected.
 * The stream must belong to the current device. Calls that overlap on one GPU
 * (two streams, two threads) race on the shared array.
 */
int dionw_normuon_stats_noalloc(const void* orthogonal, int64_t blocks, int64_t k, int64_t rows,
                                int64_t cols, const int32_t* idx, float* variance, float beta2,
                                float step, float* rowd, float* scale, dionw_stream_t stream);

/*
 * The weight update of a run: W *= decay on every row when apply_decay, then
 * W[row] += O[slot] / rowd[slot] * scale[b] on the selected rows (rowd == NULL:
 * W[row] += O[slot] * (scale ? scale[b] : step)). Replaces _apply and
 * _add_blocks_ (_matrix_step.py:274-311) and finish()'s product with the step
 * (_row_normalization.py:18-38).
 */
int dionw_apply_update(float* const* params, int32_t count, int64_t blocks_per_tensor,
                       int64_t rows, int64_t cols, int64_t k, const void* orthogonal,
                       const int32_t* idx, const int32_t* slot, const float* rowd,
                       const float* scale, float step, float decay, int32_t apply_decay,
                       dionw_stream_t stream);

/*
 * dionw_apply_update with the GPU EMA fused in: after a row's new weights are
 * formed, its float32 shadow (same layout as the parameter, shadows[i] for
 * params[i]) becomes lerp(shadow, W_new, ema_weight), on every row (also those
 * only decayed or unchanged). Replaces the apply pass followed by
 * foreach_ema_update_ over the same parameters (_matrix_step.py:274-311, then
 * ema/_update.py:32-70 from ema/tracker.py:217-227) with one pass: 4 bytes per
 * element less than the two.
 */
int dionw_apply_update_ema(float* const* params, float* const* shadows, int32_t count,
                           int64_t blocks_per_tensor, int64_t rows, int64_t cols, int64_t k,
                           const void* orthogonal, const int32_t* idx, const int32_t* slot,
                           const float* rowd, const float* scale, float step, float decay,
                           int32_t apply_decay, float ema_weight, dionw_stream_t stream);

/*
 * dionw_apply_update that also writes every row's new weights (also the rows
 * only decayed or unchanged) into staged[i], a pinned host buffer laid out like
 * params[i] (hipHostMalloc or torch pin_memory=True; other memory is rejected
 * before any launch): the CPU EMA's snapshot of the parameters taken by the pass
 * that forms them. Replaces the apply pass followed by the side-stream
 * tmp_cpu.copy_(param, non_blocking=True) of every parameter
 * (_matrix_step.py:274-311, then ema/tracker.py:229-248). The snapshot is
 * complete once the work enqueued on `stream` up to this call has finished.
 */
int dionw_apply_update_stage(float* const* params, float* const* staged, int32_t count,
                             int64_t blocks_per_tensor, int64_t rows, int64_t cols, int64_t k,
                             const void* orthogonal, const int32_t* idx, const int32_t* slot,
                             const float* rowd, const float* scale, float step, float decay,
                             int32_t apply_decay, dionw_stream_t stream);

/* steps[i] += 1 (float32 device scalars): the _foreach_add_ of _adamw.py:47. */
int dionw_increment_steps(float* const* steps, int32_t count, dionw_stream_t stream);

/*
 * Multi-tensor AdamW with decoupled weight decay, bit-compatible with
 * torch._fused_adamw_ (called by adamw_step, _adamw.py:25-61): reads each
 * tensor's (already incremented) float32 step.
 */
int dionw_adamw(float* const* params, const float* const* grads, float* const* exp_avgs,
                float* const* exp_avg_sqs, const float* const* steps, const int64_t* numels,
                int32_t count, double lr, double beta1, double beta2, double weight_decay,
                double eps, dionw_stream_t stream);

/*
 * dionw_adamw with the GPU EMA fused in: shadows[i] = lerp(shadows[i], new
 * params[i], ema_weight). Replaces _fused_adamw_ followed by
 * foreach_ema_update_ over the same tensors (_adamw.py:45-61, then
 * ema/_update.py:32-70 from ema/tracker.py:217-227) with one pass.
 */
int dionw_adamw_ema(float* const* params, const float* const* grads, float* const* exp_avgs,
                    float* const* exp_avg_sqs, const float* const* steps, float* const* shadows,
                    const int64_t* numels, int32_t count, double lr, double beta1, double beta2,
                    double weight_decay, double eps, float ema_weight, dionw_stream_t stream);

/*
 * Multi-tensor AdamW with the moments in 8 bits (not in the reference). The state of
 * `tensors` tensors lies in shared arrays of `blocks` blocks of 256 elements: exp_avg
 * (e4m3 bytes) and rms (the root of the second moment: unsigned bytes of 4 exponent bits,
 * bias 8, and 4 fraction bits), 256 a block, and one float32 power of two a block in
 * exp_avg_scale and rms_scale. Tensor i of the call has numels[i] contiguous elements, its
 * blocks from first_blocks[i] on and its step at steps[ids[i]]. No two tensors of a call may
 * share blocks or an id. Increments the steps, then
 *   m = beta1 m + (1 - beta1) g;   v = beta2 v + (1 - beta2) g^2
 *   p = p (1 - lr weight_decay) - lr / (1 - beta1^t) m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
 * and stores m and sqrt(v) rounded stochastically by a hash of (step, id, element).
 * shadows (may be NULL): EMA shadows, lerped towards the new parameters by ema_weight.
 * scalars: float32 scratch, 4 for each of the `tensors`.
 */
int dionw_adamw_8bit(float* const* params, const float* const* grads, float* const* shadows,
                     const int64_t* numels, const int64_t* first_blocks, const int32_t* ids,
                     int32_t count, int64_t blocks, int32_t tensors, void* exp_avg,
                     float* exp_avg_scale, void* rms, float* rms_scale, float* steps,
                     float* scalars, double lr, double beta1, double beta2, double weight_decay,
                     double eps, float ema_weight, dionw_stream_t stream);

/* The float32 values of that state for `count` tensors, one after another in the outputs. */
int dionw_adamw_8bit_values(const int64_t* numels, const int64_t* first_blocks, int32_t count,
                            int64_t blocks, const void* exp_avg, const float* exp_avg_scale,
                            const void* rms, const float* rms_scale, float* exp_avg_out,
                            float* rms_out, dionw_stream_t stream);

/*
 * 8-bit matrices (not in the reference). A quantized matrix [rows, cols] is e4m3 codes
 * [rows][data_ld] (data_ld a multiple of 16, at least cols rounded up to 128; 16-byte aligned;
 * the columns up to that multiple of 128 hold zeros) and the exponent bytes of float32 powers
 * of two [blocks of 128 columns][scale_ld], scale_ld >= rows.
 *
 * dionw_float8_quantize rounds x [rows, cols] (row pitch ld, element code elem) to nearest:
 * into data/scale by rows, and into data_t/scale_t as the transpose [cols, rows]; either may
 * be NULL. One scale for each row (of the transpose: column of x) and block of 128, or for
 * each 128 x 128 tile when tiles != 0. Values that are not finite become NaN and leave their
 * block's scale alone. expanded: bit 0 for data, bit 1 for data_t: they take bfloat16 halves of
 * the values (see dionw_float8_expand; pitches in elements) and the scales are not used. sums (may
 * be NULL): float32 [ceil(rows / 128)][cols], the column sums of each 128 rows.
 */
int dionw_float8_quantize(int32_t elem, const void* x, int64_t rows, int64_t cols, int64_t ld,
                          int32_t tiles, void* data, int64_t data_ld, void* scale,
                          int64_t scale_ld, void* data_t, int64_t data_t_ld, void* scale_t,
                          int64_t scale_t_ld, int32_t expanded, float* sums,
                          dionw_stream_t stream);

/* out[c] = parts[0][c] + parts[1][c] + ..., a quarter of them at a time, in a fixed order, in
 * element code elem. */
int dionw_sum_parts(const float* parts, int64_t count, int64_t cols, int32_t elem, void* out,
                    dionw_stream_t stream);

/*
 * The codes [rows][data_ld] of a quantized matrix expanded: bfloat16 halves of the values,
 * out [rows][out_ld] (16-byte aligned, out_ld a multiple of 8), `depth` columns (a multiple
 * of 128).
 */
int dionw_float8_expand(const void* data, int64_t data_ld, const void* scale, int64_t scale_ld,
                        int64_t rows, int64_t depth, void* out, int64_t out_ld,
                        dionw_stream_t stream);

/*
 * C [m, n] = A B^T + bias for quantized A [m, depth] and B [n, depth] (depth: a multiple of
 * 128), summed in float32 and rounded once to element code elem; bias: n floats or NULL.
 * expanded 0: codes with their scales (pitches a multiple of 16, 4-byte aligned), float16 or
 * bfloat16 output; the products of each 8 columns are cut to 13 bits below the exponent of
 * the largest of them before they are added. expanded 1: operands from dionw_float8_expand
 * (or dionw_float8_quantize), float32 output, every product exact. Pitches in elements, rows
 * of less than 8 MB at multiples of 16 bytes. workspace: float32 scratch of
 * dionw_float8_gemm_workspace bytes (0: none needed). dionw_float8_gemm_plan writes what a product
 * of these extents runs on: the side of its tiles (256, 128 or 64) and in how many ranges its depth
 * is summed (1: whole).
 */
int dionw_float8_gemm_plan(int32_t expanded, int64_t m, int64_t n, int64_t depth, int32_t* side,
                           int32_t* ranges);
size_t dionw_float8_gemm_workspace(int32_t expanded, int64_t m, int64_t n, int64_t depth);
int dionw_float8_gemm(int32_t expanded, int64_t m, int64_t n, int64_t depth, const void* a,
                      int64_t lda, const void* a_scale, int64_t a_scale_ld, const void* b,
                      int64_t ldb, const void* b_scale, int64_t b_scale_ld, const float* bias,
                      int32_t elem, void* c, int64_t ldc, void* workspace, size_t workspace_bytes,
                      dionw_stream_t stream);

/*
 * A linear layer on 8-bit operands: y [m, n] = x [m, k] W [n, k]^T + bias in x's element code
 * (x_elem), from float x and W (pitches in elements). x is quantized by rows, W by tiles.
 * saved (NULL where both needs are 0) keeps, for the backward, W's transpose (need_x) and x's
 * (need_w) in codes. The backward gives dx (x_elem) = dy W when need_x, dw (w_elem) = dy^T x
 * when need_w, dy quantized by rows and by columns, and db (bias_elem) = the column sums of dy
 * when db is not NULL; float32 results are summed in float32, 16-bit ones on the 8-bit
 * instructions (dionw_float8_gemm). dionw_float8_linear_sizes writes the bytes of saved and of
 * the two calls' scratch.
 */
void dionw_float8_linear_sizes(int32_t x_elem, int32_t w_elem, int64_t m, int64_t n, int64_t k,
                               int32_t need_x, int32_t need_w, int32_t need_b, size_t* sizes);
int dionw_float8_linear_forward(int32_t x_elem, const void* x, int64_t x_ld, int32_t w_elem,
                                const void* w, int64_t w_ld, const float* bias, int64_t m,
                                int64_t n, int64_t k, int32_t need_x, int32_t need_w, void* y,
                                void* saved, void* scratch, size_t scratch_bytes,
                                dionw_stream_t stream);
int dionw_float8_linear_backward(int32_t x_elem, const void* dy, int64_t dy_ld, int32_t w_elem,
                                 int64_t m, int64_t n, int64_t k, int32_t need_x, int32_t need_w,
                                 const void* saved, void* dx, void* dw, int32_t bias_elem,
                                 void* db, void* scratch, size_t scratch_bytes,
                                 dionw_stream_t stream);

/*
 * The same y from a kept W: codes [n][w_ld] with their scales [ceil(k / 128)][w_scale_ld]. Up
 * to 16 rows of x (32 float32 ones, 64 of at most 4096 columns) are quantized by the product
 * itself, in one launch and no scratch.
 */
size_t dionw_float8_linear_kept_scratch(int32_t x_elem, int64_t m, int64_t n, int64_t k);
int dionw_float8_linear_kept(int32_t x_elem, const void* x, int64_t x_ld, const void* w,
                             int64_t w_ld, const void* w_scale, int64_t w_scale_ld,
                             const float* bias, int64_t m, int64_t n, int64_t k, void* y,
                             void* scratch, size_t scratch_bytes, dionw_stream_t stream);

/*
 * 4-bit matrices (not in the reference). A quantized matrix [rows, cols] is e2m1 codes, two a byte
 * (the first column's in the low half), rows of depth / 2 bytes one behind the other, depth being
 * cols rounded up to 256 (zeros from cols on), and the exponent bytes of float32 powers of two
 * [depth / 32][scale_ld], scale_ld >= rows and a multiple of 16; 255 makes a block NaN. Codes and
 * scales are 16-byte aligned.
 *
 * dionw_float4_quantize rounds x [rows, cols] (row pitch ld, element code elem) into data/scale by
 * rows and into data_t/scale_t as the transpose [cols, rows]; either data may be NULL. rounding 0:
 * to nearest, one scale for each row (of the transpose: column of x) and block of 32; 1: to
 * nearest, one for each 32 x 32 tile; 2: as 0, stochastically, with bits from a hash of seed (of
 * *seed_at in device memory, read by the kernel, where that is not NULL) and the element's place. A
 * block with a value that is not finite is NaN. dionw_float4_values writes the float32 values,
 * [rows][cols].
 */
int dionw_float4_quantize(int32_t elem, const void* x, int64_t rows, int64_t cols, int64_t ld,
                          int32_t rounding, int64_t seed, const int64_t* seed_at, void* data,
                          void* scale, int64_t scale_ld, void* data_t, void* scale_t,
                          int64_t scale_t_ld, dionw_stream_t stream);
int dionw_float4_values(const void* data, const void* scale, int64_t scale_ld, int64_t rows,
                        int64_t cols, float* out, dionw_stream_t stream);

/*
 * C [m, n] = A B^T + bias for quantized A [m, depth] and B [n, depth] (depth: a multiple of 256, of
 * less than 16 M), summed in float32 and rounded once to element code elem; bias: n floats or NULL.
 * workspace: float32 scratch of dionw_float4_gemm_workspace bytes (0: none needed).
 * dionw_float4_gemm_plan writes what a product of these extents runs on: the side of its tiles (256,
 * 128 or 64) and in how many ranges its depth is summed (1: whole).
 */
int dionw_float4_gemm_plan(int64_t m, int64_t n, int64_t depth, int32_t* side, int32_t* ranges);
size_t dionw_float4_gemm_workspace(int64_t m, int64_t n, int64_t depth);
int dionw_float4_gemm(int64_t m, int64_t n, int64_t depth, const void* a, const void* a_scale,
                      int64_t a_scale_ld, const void* b, const void* b_scale, int64_t b_scale_ld,
                      const float* bias, int32_t elem, void* c, int64_t ldc, void* workspace,
                      size_t workspace_bytes, dionw_stream_t stream);

/*
 * A linear layer on 4-bit operands: y [m, n] = x [m, k] W [n, k]^T + bias in x's element code
 * (x_elem), from float x and W (pitches in elements). x is quantized by rows, W by tiles. saved
 * (NULL where both needs are 0) keeps, for the backward, W's transpose (need_x) and x's (need_w) in
 * codes. The backward gives dx (x_elem) = dy W when need_x, dw (w_elem) = dy^T x when need_w, dy
 * rounded stochastically by rows and by columns, and db (bias_elem) = the column sums of dy when db
 * is not NULL. dionw_float4_linear_sizes writes the bytes of saved and of the two calls' scratch.
 */
void dionw_float4_linear_sizes(int64_t m, int64_t n, int64_t k, int32_t need_x, int32_t need_w,
                               int32_t need_b, size_t* sizes);
int dionw_float4_linear_forward(int32_t x_elem, const void* x, int64_t x_ld, int32_t w_elem,
                                const void* w, int64_t w_ld, const float* bias, int64_t m,
                                int64_t n, int64_t k, int32_t need_x, int32_t need_w, void* y,
                                void* saved, void* scratch, size_t scratch_bytes,
                                dionw_stream_t stream);
int dionw_float4_linear_backward(int32_t x_elem, const void* dy, int64_t dy_ld, int32_t w_elem,
                                 int64_t m, int64_t n, int64_t k, int32_t need_x, int32_t need_w,
                                 int64_t seed, const int64_t* seed_at, const void* saved, void* dx,
                                 void* dw, int32_t bias_elem, void* db, void* scratch,
                                 size_t scratch_bytes, dionw_stream_t stream);

/*
 * The same y from a kept W: codes [n] rows with their scales [depth / 32][w_scale_ld]. Up to 8 rows
 * of x (16 of up to 8192 columns where W has 4096 rows or less, of up to 2048 where it has 5105 to 16384,
 * of up to 4096 elsewhere) are quantized by the product itself, in one launch and no scratch.
 */
size_t dionw_float4_linear_kept_scratch(int64_t m, int64_t n, int64_t k);
int dionw_float4_linear_kept(int32_t x_elem, const void* x, int64_t x_ld, const void* w,
                             const void* w_scale, int64_t w_scale_ld, const float* bias, int64_t m,
                             int64_t n, int64_t k, void* y, void* scratch, size_t scratch_bytes,
                             dionw_stream_t stream);

/*
 * Layer norm of the rows of x [rows, cols] (row pitch x_ld, element code elem): y [rows][cols] in x's
 * code, (x - mean) / sqrt(variance + eps) * weight + bias, the parameters in codes of their own
 * (NULL: ones, zeros). mean and rstd (both or neither): float32 [rows], for the backward.
 * dionw_layer_norm_float4 writes the same y, not rounded to a type of its own first, quantized by rows
 * to nearest (dionw_float4_quantize).
 * The backward gives dx (x's code), dg (w_elem) and db (b_elem), each where it is not NULL; dg and db
 * take scratch of dionw_layer_norm_backward_scratch bytes.
 */
int dionw_layer_norm_forward(int32_t elem, const void* x, int64_t x_ld, int64_t rows, int64_t cols,
                             int32_t w_elem, const void* weight, int32_t b_elem, const void* bias,
                             float eps, void* y, float* mean, float* rstd, dionw_stream_t stream);
int dionw_layer_norm_float4(int32_t elem, const void* x, int64_t x_ld, int64_t rows, int64_t cols,
                            int32_t w_elem, const void* weight, int32_t b_elem, const void* bias,
                            float eps, void* data, void* scale, int64_t scale_ld,
                            dionw_stream_t stream);
size_t dionw_layer_norm_backward_scratch(int64_t rows, int64_t cols);
int dionw_layer_norm_backward(int32_t elem, const void* x, int64_t x_ld, const void* dy, int64_t dy_ld,
                              int64_t rows, int64_t cols, int32_t w_elem, const void* weight,
                              const float* mean, const float* rstd, void* dx, void* dg,
                              int32_t b_elem, void* db, void* scratch, size_t scratch_bytes,
                              dionw_stream_t stream);

/*
 * GPU EMA of float32 sources: shadow = lerp(shadow, source, weight), or a
 * copy when copy != 0. Replaces foreach_ema_update_ (ema/_update.py:32-70)
 * and the first-update _foreach_copy_ (ema/tracker.py:142-145).
 */
int dionw_ema_update(float* const* shadows, const float* const* sources, const int64_t* numels,
                     int32_t count, float weight, int32_t copy, dionw_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* DIONW_HIP_H */
