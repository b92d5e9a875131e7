/* Kernel-level C-ABI of libns_b200.so: the hot-path kernels on caller-owned
 * DEVICE pointers, one call per kernel family, for tests, benchmarks and
 * integrators that drive their own buffers. Each entry names the reference
 * computation it replaces (file:line in MrModelOS/NeuralScript). `stream` is
 * a cudaStream_t (NULL = legacy default stream). Returns 0 on success, a
 * negative value on a bad argument or launch failure. Nothing here
 * allocates device memory: scratch, where a kernel needs it, is passed in
 * and its size is given by the matching *_scratch_bytes query.
 */
#ifndef NS_B200_OPS_H
#define NS_B200_OPS_H

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

/* dtype codes */
#define NSB_F32 0
#define NSB_BF16 1

/* engine codes */
#define NSB_ENGINE_AUTO 0   /* tcgen05 when operands allow, else SIMT */
#define NSB_ENGINE_SIMT 1   /* exact fp32 FMA, sequential in k */
#define NSB_ENGINE_TENSOR 2 /* tcgen05 only (error if not possible) */

/* C[M,N] = act(alpha * A[M,K] B[N,K]^T + add) with
 *   A element (i,k) at A[i*lda + k] (a_mn = 0) or A[k*lda + i] (a_mn = 1),
 *   B element (n,k) at B[n*ldb + k] (b_mn = 0) or B[k*ldb + n] (b_mn = 1).
 * Replaces ns_gemm_kernel / ns_grad_a_kernel / ns_grad_w_kernel
 * (src/codegen/cuda_backend.cpp:58-79, 446-467) and ns_matmul /
 * ns_matmul_grad_a / ns_matmul_grad_w (src/codegen/codegen.cpp:1257-1337).
 * act: 0 identity .. 6 GELU (codegen.cpp:1244-1255). add (fp32, ld_add) may be
 * NULL. c32 / c16 outputs (either may be NULL). workspace: fp32 scratch of
 * nsb_op_gemm_workspace_floats(...) floats (may be NULL when that is 0). */
int nsb_op_gemm(int M, int N, int K, const void* A, int a_dtype, long long lda, int a_mn, const void* B, int b_dtype,
                long long ldb, int b_mn, float alpha, const float* add, long long ld_add, int act, float* c32,
                long long ldc32, void* c16, long long ldc16, int engine, float* workspace, size_t workspace_floats,
                int* dev_err, void* stream);
size_t nsb_op_gemm_workspace_floats(int M, int N, int K, const void* A, int a_dtype, long long lda, int a_mn,
                                    const void* B, int b_dtype, long long ldb, int b_mn, int engine);
/* 1 when nsb_op_gemm would run on tcgen05 tensor cores for these operands. */
int nsb_op_gemm_uses_tensor_cores(int M, int N, int K, const void* A, int a_dtype, long long lda, int a_mn,
                                  const void* B, int b_dtype, long long ldb, int b_mn, int engine);

/* out = W[(int)ids[r]] (ids fp32; out-of-range -> row 0).
 * Replaces ns_embedding_kernel (cuda_backend.cpp:172-181), ns_embedding
 * (codegen.cpp:1711-1718). */
int nsb_op_embedding_fwd(const float* W, const float* ids, int M, int V, int D, float* out32, void* out16,
                         void* stream);
/* dW = deterministic sort-then-segment scatter-add of dout rows by id
 * (rows in increasing order; out-of-range ids skipped). Replaces
 * ns_embedding_grad_w_kernel (cuda_backend.cpp:500-512) and
 * ns_embedding_grad_w (codegen.cpp:1374-1383). */
size_t nsb_op_embedding_bwd_scratch_bytes(int M, int V);
int nsb_op_embedding_bwd(const float* dout, const float* ids, int M, int V, int D, float* dW, void* scratch,
                         void* stream);

/* Allocation-free variant of nsb_op_embedding_bwd (same result, bit for
 * bit). No counterpart in the reference: it exists for callers that cannot
 * allocate device memory when they need this gradient - code running inside
 * a memory-pool or allocator callback, hosts that have given all device
 * memory to their own pool, runtimes that forbid cudaMalloc after start-up.
 * Its sort scratch is a fixed array in the library's device memory, so it
 * calls no cudaMalloc, cudaFree or allocating library routine.
 * Limits: M <= 262144 rows and V <= 65536 vocabulary rows; larger sizes
 * return -2 without launching anything. The work runs on the current device:
 * a non-NULL `stream` must belong to it (otherwise -4, nothing launched).
 * Every GPU that loads the library
 * holds the 1.75 MB array until the process exits. The first call on a
 * device looks up the array's device address (cudaGetSymbolAddress, once per
 * device, with that device current); make that first call before any CUDA
 * stream capture. All calls share the one array: calls that overlap on the
 * same GPU (for example on two streams) race on it, so serialise them on one
 * stream. Counters are cleared by every call. */
int nsb_op_embedding_bwd_noalloc(const float* dout, const float* ids, int M, int V, int D, float* dW, void* stream);

/* LayerNorm, no affine, eps 1e-5. Replaces ns_layernorm_kernel /
 * ns_layernorm_grad_kernel (cuda_backend.cpp:420-431, 473-499),
 * ns_layernorm / ns_layernorm_grad (codegen.cpp:1280-1291, 1346-1371). */
int nsb_op_layernorm_fwd(const float* x, int M, int D, float* out32, void* out16, void* stream);
int nsb_op_layernorm_bwd(const float* dy, const float* x, const float* add, int M, int D, float* dx32, void* dx16,
                         void* stream);

/* Attention core on qkv [B*S, ld_qkv] (Q | K | V column blocks, heads
 * concatenated) -> ctx [B*S, ld_ctx]; lse [B*H*S] saved for the backward.
 * Replaces ns_attention_core_kernel / ns_attention_grad_kernel
 * (cuda_backend.cpp:186-366) and the per-head core of ns_attention_fwd /
 * ns_attention_bwd (codegen.cpp:1724-1907). dvec: [B*H*S] fp32 scratch. */
int nsb_op_attention_fwd(int B, int S, int H, int D, int dtype, const void* qkv, long long ld_qkv, void* ctx,
                         long long ld_ctx, float* lse, void* stream);
int nsb_op_attention_bwd(int B, int S, int H, int D, int dtype, const void* qkv, long long ld_qkv, const void* ctx,
                         long long ld_ctx, const float* lse, const void* dctx, long long ld_dctx, void* dqkv,
                         long long ld_dqkv, float* dvec, void* stream);

/* Softmax cross-entropy forward + seed gradient: row_loss[r] and
 * d = (softmax - y) / denom. labels one-hot [M,C] fp32, or targets int32 [M]
 * when labels is NULL. Replaces ns_ce_row_kernel + ns_loss_grad_kernel
 * (cuda_backend.cpp:690-719), ns_cross_entropy / ns_loss_grad
 * (codegen.cpp:1582-1613). */
int nsb_op_cross_entropy(const float* logits, const float* labels, const int* targets, int M, int C, float denom,
                         float* row_loss, float* d32, void* d16, void* stream);
/* Second half of the fused head loss: logits16 holds fp16 logits [M,C]
 * (16-byte aligned, C % 8 == 0) as the head GEMM writes them, tlogit the
 * fp32 target logit of each row; writes row_loss[r] = lse - tlogit[r] (0 for
 * a target outside [0,C)) and overwrites the row in place with the bf16 seed
 * (softmax - onehot) / denom. Same arithmetic as nsb_op_cross_entropy with
 * targets (ns_ce_row_kernel + ns_loss_grad_kernel, cuda_backend.cpp:690-719). */
int nsb_op_cross_entropy_finish(void* logits16, int M, int C, const int* targets, const float* tlogit, float denom,
                                float* row_loss, void* stream);
/* out[0] = scale * sum(x[0..n)), fixed reduction order. */
int nsb_op_reduce_sum(const float* x, int n, float scale, float* out, void* stream);

/* One AdamW step of one tensor (step counter t >= 1). Replaces
 * ns_adamw_kernel (cuda_backend.cpp:720-733) / codegen.cpp:3108-3120. */
int nsb_op_adamw(float* w, const float* g, float* m, float* v, long long n, long long t, float lr, float beta1,
                 float beta2, float one_minus_beta1, float one_minus_beta2, float eps, float decay, void* stream);
/* Modified Gram-Schmidt in place on an r x c matrix (columns if r >= c, rows
 * otherwise). Replaces ns_orthonom_kernel (cuda_backend.cpp:747-773) /
 * ns_orthonom (codegen.cpp:1617-1633). */
int nsb_op_mgs(float* G, int r, int c, void* stream);

/* Top-1 MoE router: logits x.Wg accumulated with fmaf in increasing k (the
 * reference's scalar order, so the logits are bit-identical to its CPU emit),
 * softmax over live experts (active[e] != 0; NULL = all live), best = first
 * maximum of the exp'd logits (-1 if none live), pb = its probability, probs
 * [M,E] (may be NULL) the live softmax. Replaces the routing of ns_moe_kernel
 * (cuda_backend.cpp:371-407) and ns_moe_fwd (codegen.cpp:1915-1931). */
int nsb_op_moe_route(const float* x, const float* Wg, const unsigned char* active, int M, int D, int E, int* best,
                     float* pb, float* probs, void* stream);

/* Activation forward / derivative product. Replaces ns_act_kernel /
 * ns_act_grad_kernel (cuda_backend.cpp:80-84, 468-472). */
int nsb_op_act_fwd(const float* x, size_t n, int act, float* out32, void* out16, void* stream);
int nsb_op_act_bwd(const float* dy, const float* z, int act, size_t n, float* out32, void* stream);

/* Y[M,512] = LayerNorm(alpha * A[M,K] B[K,512] + add) row by row (no affine,
 * eps 1e-5), the LayerNorm in the GEMM's epilogue: a 128 x 512 tile holds
 * whole rows. A K-major (element (i,k) at A[i*lda + k]), B row-major
 * [K, 512] (B[k*ldb + n]), both bf16 or both fp32 (TF32); add fp32 (may be
 * NULL); c32 / c16 receive Y (either may be NULL), rstd[M] the rows'
 * 1 / sqrt(var + eps). Replaces a Dense / attention output GEMM, the
 * residual ns_binop and ns_layernorm_kernel in sequence
 * (cuda_backend.cpp:58-79, 408-431). */
int nsb_op_gemm_layernorm(int M, int K, const void* A, int dtype, long long lda, const void* B, long long ldb,
                          float alpha, const float* add, long long ld_add, float* c32, long long ldc32, void* c16,
                          long long ldc16, float* rstd, int* dev_err, void* stream);

/* y = 2^x for x <= 0 by the FMA-pipe exponential the attention softmax and
 * the loss pass use for part of their exponentials (Cody-Waite reduction and
 * a fitted cubic; relative error <= 7.5e-5; x below -125 gives 2^-125).
 * No reference counterpart: exposed so its error bound can be tested. */
int nsb_op_exp2_poly3(const float* x, float* y, size_t n, void* stream);

/* Row softmax (max-subtracted, exp, normalised). Replaces ns_softmax_kernel
 * (cuda_backend.cpp:432-441) / ns_softmax (codegen.cpp CPU helper). */
int nsb_op_softmax(const float* x, int M, int C, float* out32, void* out16, void* stream);

/* out = a (op) b over n elements, code 0 + 1 - 2 * 3 /, full-size b.
 * Replaces ns_binop_kernel (cuda_backend.cpp:408-419) / ns_binop
 * (codegen.cpp:1267-1278). The backward (no reference counterpart: the
 * reference has no binop gradient) writes da and/or db (either may be NULL). */
int nsb_op_binop(const float* a, const float* b, size_t n, int code, float* out32, void* out16, void* stream);
int nsb_op_binop_bwd(const float* dout, const float* a, const float* b, size_t n, int code, float* da, float* db,
                     void* stream);

/* Inverted dropout with a counter-based mask: element i keeps its value with
 * probability 1 - rate (scaled by 1/(1 - rate)), decided by Philox4x32-10 of
 * (i, step, site) under key (key0, key1); the backward regenerates the same
 * mask. Replaces ns_dropout_fwd_kernel / ns_dropout_mul_kernel
 * (cuda_backend.cpp:778-793), whose curand mask (and the CPU emit's
 * std::mt19937 mask, codegen.cpp:2874-2893) it does not reproduce. */
int nsb_op_dropout_fwd(const float* x, size_t n, float rate, unsigned key0, unsigned key1, unsigned step,
                       unsigned site, float* out32, void* out16, void* stream);
int nsb_op_dropout_bwd(const float* dy, size_t n, float rate, unsigned key0, unsigned key1, unsigned step,
                       unsigned site, float* dx, void* stream);

/* Data movement on row-major fp32 tensors. axis 1: column forms on [rows,
 * cols]; axis 0: row forms. Indices are int64. A scatter keeps the last
 * update of a repeated index (the reference CPU helpers' order); an index
 * outside the source reads 0. Replace ns_transpose2d_kernel,
 * ns_concat2/0_kernel, ns_slice2/slicerows_kernel, ns_index/indexrows_kernel
 * and ns_scatter/scatterrows_kernel (cuda_backend.cpp:93-171). */
int nsb_op_transpose(const float* in, int R, int C, float* out, void* stream);
int nsb_op_concat(const float* a, const float* b, int axis, int rows_a, int rows_b, int ca, int cb, float* out,
                  void* stream);
int nsb_op_slice(const float* in, int axis, int rows, int cols, int start, int end, float* out, void* stream);
int nsb_op_index(const float* in, int axis, int rows, int cols, const long long* idx, int L, float* out,
                 void* stream);
int nsb_op_scatter(const float* in, int axis, int rows, int cols, const long long* idx, int L, const float* upd,
                   float* out, void* stream);

/* ---- Mixture of experts with k experts a token (no reference counterpart:
 * its layer sends a token to one expert) --------------------------------- */
#define NSB_SCORE_SOFTMAX 0
#define NSB_SCORE_SIGMOID 1

/* Routing. logits [M, ld] (F32 or BF16), scores s = softmax over the live
 * experts or sigmoid, both in fp32; active[e] = 0 marks a dead expert, whose
 * logit is not looked at (NULL = all live). The choice goes by s + bias
 * (bias [E], may be NULL). With groups > 1 (a divisor of E, at least two
 * experts each) a group's score is the sum of its two best s + bias (of live
 * experts; of its one where only one lives), and only the topk_groups best
 * groups stay. The k largest are chosen, in falling order; ties go to the
 * lower expert, and group. idx [M, k] receives the experts, w [M, k] their
 * weights
 *   w = scale * s / (sum of the k chosen s + 1e-20)     (renorm)
 *   w = scale * s                                       (otherwise).
 * A row with fewer than k candidates has idx -1 and w 0 in the rest; an
 * expert whose s + bias is NaN or -inf is no candidate (a softmax row with a
 * NaN or +inf logit, or with -inf in every live one, has none).
 * Limits: E <= 1024, k <= 32, k <= E. */
int nsb_op_moe_topk_route(const void* logits, int dtype, long long ld, int M, int E, int k, int score,
                          const float* bias, const unsigned char* active, int groups, int topk_groups, int renorm,
                          float scale, int* idx, float* w, void* stream);
/* Its gradient: dlogits [M, ld_dlogits] (the logits' type) from dw [M, k],
 * the same logits and the choice idx, which is constant. Entries of dw beside
 * idx -1 are not looked at; a row without any expert gets zeros. */
int nsb_op_moe_topk_route_bwd(const float* dw, const void* logits, int dtype, long long ld, int M, int E, int k,
                              int score, const unsigned char* active, int renorm, float scale, const int* idx,
                              void* dlogits, long long ld_dlogits, void* stream);

/* Order of the pairs (token t, choice j), numbered t * k + j, by expert:
 * expert e owns rows [offsets[e], offsets[e] + counts[e]) in rising pair
 * order, offsets[e] a multiple of align, offsets[E] the end of the last.
 * rows[r] = the pair in row r or -1 (all of nsb_op_moe_dispatch_rows(...)
 * rows are written), pos[t * k + j] = its row, -1 for idx outside [0, E).
 * E <= 1024, k <= 32; more than 2^31 - 1 rows return -2. */
size_t nsb_op_moe_dispatch_rows(int M, int k, int E, int align);
int nsb_op_moe_dispatch(const int* idx, int M, int k, int E, int align, int* offsets, int* counts, int* rows, int* pos,
                        void* stream);

/* y[t] = sum over j of w[t,j] * o[pos[t,j]] in fp32, rounded once (w NULL:
 * all 1, the gradient of a gather by rows; negative pos are left out). o, y:
 * [*, D] of one dtype. */
int nsb_op_moe_combine(const void* o, int dtype, long long ld_o, const int* pos, const float* w, int M, int k, int D,
                       void* y, long long ld_y, void* stream);
/* The same where o has R rows: a pos past them is left out, and reported by
 * nsb_op_device_error (above, pos is trusted). */
int nsb_op_moe_combine_rows(const void* o, int dtype, long long ld_o, int R, const int* pos, const float* w, int M,
                            int k, int D, void* y, long long ld_y, void* stream);
/* Its gradient: d_o[r] = w[pair] * dy[pair / k] for pair = rows[r], zeros for
 * a negative rows[r], or one past the last pair, which is reported (R rows),
 * and dw[pair] = <o[r], dy[pair / k]>, 0 for pairs without a row (dw and o may
 * be NULL together). */
int nsb_op_moe_combine_bwd(const void* dy, const void* o, int dtype, long long ld_dy, long long ld_o, const int* rows,
                           const int* pos, const float* w, int M, int k, int R, int D, void* d_o, long long ld_do,
                           float* dw, void* stream);

/* ---- 8-bit floating point (e4m3) with a scale for each block of 128 ------
 * (no reference counterpart)
 *   scale = max(max |x| * (1 / 448), 2^-100),  code = e4m3(x * (1 / scale)),
 * rounded to nearest even, the value read back code * scale. NaN gives a NaN
 * code and does not count in the maximum; an infinity turns its block to NaN.
 * Code arrays: 16-byte aligned, rows on 16-byte boundaries (leading
 * dimensions multiples of 16). Scales of rows are block-major: row r,
 * columns [128 b, 128 b + 128) at s[b * ld_s + r]; scales of 128 x 128 blocks
 * lie row by row.
 *
 * x [*, ld] (F32 or BF16, any alignment) with act(x) quantised (act 0: x
 * itself): q [M, ld_q] with s (a scale for each 1 x 128), and / or the
 * transpose qt [K, ld_qt] with st (a scale for each 128 rows of a column).
 * rows (NULL: none) gathers first: row r of the result is row
 * rows[r] / row_div of x (row_div 0: row r), zeros for a negative entry. */
int nsb_op_fp8_quantize(const void* x, int dtype, long long ld, int M, int K, int act, const int* rows, int row_div,
                        void* q, long long ld_q, float* s, long long ld_s, void* qt, long long ld_qt, float* st,
                        long long ld_st, void* stream);
/* The same where x has x_rows rows (at least M of them without a row list or
 * with row_div 0): an entry of rows past them counts as a negative one, and is
 * reported by nsb_op_device_error (above, rows is trusted). */
int nsb_op_fp8_quantize_rows(const void* x, int dtype, long long ld, int x_rows, int M, int K, int act, const int* rows,
                             int row_div, void* q, long long ld_q, float* s, long long ld_s, void* qt, long long ld_qt,
                             float* st, long long ld_st, void* stream);
/* A scale for each 128 x 128: q [M, ld_q], s [M / 128, ld_s], and / or the
 * transpose of the same codes and scales, qt [K, ld_qt], st [K / 128, ld_st]. */
int nsb_op_fp8_quantize_block(const void* x, int dtype, long long ld, int M, int K, void* q, long long ld_q, float* s,
                              long long ld_s, void* qt, long long ld_qt, float* st, long long ld_st, void* stream);

/* What went wrong on the current device since the last call, in a product
 * below whose caller gave no dev_err or with an index past its tensor's rows:
 * 0, or the first error's code, which is cleared (101 to 104: a bounded wait
 * ran out and the product's result is not to be used; 111: an index was left
 * out). Waits for the stream; not inside a capture. */
int nsb_op_device_error(int* code, void* stream);

/* C[M,N] = A[M,K] B[N,K]^T of the values that codes and scales stand for:
 * exact products, fp32 sums over 128 k, these scaled and added in fp32 (the
 * product of two blocks' scales is to be a finite fp32 number), rounded once
 * to c_dtype. A has row scales; B 128 x 128 scales (b_rows 0: a
 * weight; its transposed codes serve the input gradient) or row scales
 * (b_rows 1: the weight gradient, from two transposed quantisations). */
int nsb_op_gemm_fp8(int M, int N, int K, const void* A, long long lda, const float* sa, long long ld_sa,
                    const void* B, long long ldb, const float* sb, long long ld_sb, int b_rows, void* C, int c_dtype,
                    long long ldc, int* dev_err, void* stream);
/* The experts' products: rows [offsets[e], offsets[e] + counts[e]) of C
 * [R, ldc] are those of A times B[e]^T (b_stride codes and sb_stride scales
 * from expert to expert, 128 x 128 scales); other rows of C are not written.
 * rows (NULL: A is in C's order): row r reads row rows[r] / row_div of A,
 * which has a_rows rows (the last one where the entry is past it). E <= 1024. */
int nsb_op_moe_gemm_fp8(int R, int E, int N, int K, const void* A, long long lda, int a_rows, const float* sa,
                        long long ld_sa, const int* rows, int row_div, const int* offsets, const int* counts,
                        const void* B, long long ldb, long long b_stride, const float* sb, long long ld_sb,
                        long long sb_stride, void* C, int c_dtype, long long ldc, int* dev_err, void* stream);
/* The experts' weight gradients: C[e] (c_stride elements apart) =
 * sum over r in [offsets[e], offsets[e] + counts[e]) of A[:, r] B[:, r]^T, A
 * [M, R] and B [N, R] with row scales, both zero in the columns between an
 * expert's last row and the next multiple of 128; offsets multiples of 128.
 * An expert without rows gets zeros. */
int nsb_op_moe_wgrad_fp8(int M, int N, int R, int E, const void* A, long long lda, const float* sa, long long ld_sa,
                         const void* B, long long ldb, const float* sb, long long ld_sb, const int* offsets,
                         const int* counts, void* C, int c_dtype, long long ldc, long long c_stride, int* dev_err,
                         void* stream);

/* ---- Attention that answers token by token (no reference counterpart: its
 * attention is bidirectional, without positions, and keeps nothing between
 * calls) --------------------------------------------------------------------
 * Tensors of heads [rows, heads, dh]: `_row` and `_head` are the strides in
 * elements from row to row and head to head, a head's columns lie side by
 * side. Hq query heads share Hkv key heads (a divisor of Hq): query head h
 * reads key head h / (Hq / Hkv). dtype is that of every tensor of heads.
 *
 * A cache of keys (of values) has `pages` pages of `page` places: place p of
 * page n, head h, at n * _page + p * _slot + h * _head. table [B, ld_table]
 * lists the pages of every sequence (`width` of them): key j of sequence b is
 * at place j % page of page table[b, j / page]. */

/* Rotary positions. Pair i < pairs of a head of x [T, H, dh] is columns
 * (i, i + pairs), or (2 i, 2 i + 1) where interleaved, and becomes
 *   scale * (x0 cos a - x1 sin a, x1 cos a + x0 sin a),  a = pos[axis, t] * freq[i],
 * the angle in 64 bits. pos [axes, ld_pos] holds up to four coordinates of
 * each token; the first sections[0] pairs turn by the first, the next
 * sections[1] by the second and so on (sections: `axes` ints in host memory
 * whose sum is pairs; NULL with one axis). Columns from 2 * pairs on are
 * copied. y may be x. dh is even, at most 1024, H * dh at most 2^26. */
int nsb_op_rope(const void* x, int dtype, long long x_row, long long x_head, int T, int H, int dh, const int* pos,
                long long ld_pos, int axes, const int* sections, const float* freq, int pairs, int interleaved, float scale,
                void* y, long long y_row, long long y_head, void* stream);
/* Its gradient: dx from dy, the rotation back. */
int nsb_op_rope_bwd(const void* dy, int dtype, long long dy_row, long long dy_head, int T, int H, int dh, const int* pos,
                    long long ld_pos, int axes, const int* sections, const float* freq, int pairs, int interleaved,
                    float scale, void* dx, long long dx_row, long long dx_head, void* stream);

/* Keys k and values v [T, Hkv, dh] into their caches, token t at key at[t] of
 * sequence seq[t], keys rotated as above on the way (pairs 0: as they are),
 * and queries q [T, Hq, dh], rotated, to q_out (both may be NULL; q_out may be
 * q). A token with a negative seq[t] is padding: nothing of its keys, values
 * and queries is read or written. One whose place is outside the table or the
 * cache is left out too, and reported by nsb_op_device_error. No two tokens of
 * one call go to the same place. (2 Hkv + Hq) * dh is at most 2^26. */
int nsb_op_kv_append(const void* k, long long k_row, long long k_head, const void* v, long long v_row, long long v_head,
                     int dtype, int T, int Hkv, int dh, const int* seq, const int* at, const int* table, long long ld_table,
                     int B, int width, int pages, int page, void* k_cache, long long kc_page, long long kc_slot,
                     long long kc_head, void* v_cache, long long vc_page, long long vc_slot, long long vc_head,
                     const int* pos, long long ld_pos, int axes, const int* sections, const float* freq, int pairs,
                     int interleaved, float scale, const void* q, long long q_row, long long q_head, int Hq, void* q_out,
                     long long qo_row, long long qo_head, void* stream);

/* Attention of one new token a sequence: q, out [B, Hq, dh] over the first
 * lens[b] keys of the cache (the new token's own among them),
 *   out = sum_j p_j v_j,  p = softmax(scale * q . k_j),  lse = log sum_j exp(scale * q . k_j)
 * over j < lens[b] and, where window > 0, j >= lens[b] - window or j < sinks.
 * lse [B, Hq] may be NULL. Without a key (or with none but scores of -inf):
 * zeros and -inf; a negative length is one of 0. A length that the table has no
 * room for, or above 2^31 - 16, is cut, and a page outside the cache left out;
 * both are reported by nsb_op_device_error. What the cache holds behind a
 * sequence's end is not looked at. dh <= 128, B <= 8192, B * Hq < 2^31,
 * scale > 0. workspace (16-byte aligned) of at least
 * nsb_op_attention_paged_workspace_bytes(...) bytes: of this call alone until
 * it is done. */
size_t nsb_op_attention_paged_workspace_bytes(int B, int Hq, int Hkv, int dh);
int nsb_op_attention_paged(const void* q, long long q_row, long long q_head, int dtype, int B, int Hq, int Hkv, int dh,
                           const void* k_cache, long long kc_page, long long kc_slot, long long kc_head, const void* v_cache,
                           long long vc_page, long long vc_slot, long long vc_head, int pages, int page, const int* table,
                           long long ld_table, int width, const int* lens, int window, int sinks, float scale, void* out,
                           long long out_row, long long out_head, float* lse, void* workspace, size_t workspace_bytes,
                           void* stream);

/* Causal attention of packed sequences: rows [offsets[b], offsets[b + 1]) of
 * q, out [T, Hq, dh] and k, v [T, Hkv, dh] are sequence b (offsets [B + 1]
 * rising from 0 on, at most T; NULL with B = 1: one of T rows), in which
 * query i sees key j where
 *   j <= i  and  (window == 0  or  i - j < window  or  j < sinks).
 * lse [Hq, ld_lse] receives the log-sum-exp (may be NULL). Rows behind the
 * last sequence are neither read nor written. Offsets that do not rise are
 * cut and reported by nsb_op_device_error. dh <= 128, scale > 0, T <= 2^30,
 * Hq <= 65535. What is infinite or NaN in a sequence can reach its rows that it
 * is hidden from too: values the outputs, keys the gradients of queries, queries
 * and dout those of keys and values. */
int nsb_op_attention_window(const void* q, long long q_row, long long q_head, const void* k, long long k_row,
                            long long k_head, const void* v, long long v_row, long long v_head, int dtype, int T, int Hq,
                            int Hkv, int dh, const int* offsets, int B, int window, int sinks, float scale, void* out,
                            long long out_row, long long out_head, float* lse, long long ld_lse, void* stream);
/* Its gradients from dout, the forward pass's out and lse: dq, and dk, dv
 * summed over the query heads that share a key head, in a fixed order.
 * workspace (16-byte aligned) of at least
 * nsb_op_attention_window_bwd_workspace_bytes(...) bytes: of this call alone
 * until it is done. */
size_t nsb_op_attention_window_bwd_workspace_bytes(int T, int Hq, int Hkv, int dh, int dtype);
int nsb_op_attention_window_bwd(const void* q, long long q_row, long long q_head, const void* k, long long k_row,
                                long long k_head, const void* v, long long v_row, long long v_head, int dtype, int T,
                                int Hq, int Hkv, int dh, const int* offsets, int B, int window, int sinks, float scale,
                                const void* out, long long out_row, long long out_head, const float* lse, long long ld_lse,
                                const void* dout, long long do_row, long long do_head, void* dq, long long dq_row,
                                long long dq_head, void* dk, long long dk_row, long long dk_head, void* dv,
                                long long dv_row, long long dv_head, void* workspace, size_t workspace_bytes,
                                void* stream);

/* The calls from nsb_op_rope on with their arguments in one block, in order
 * and each aligned as in a struct (`bytes` up to the end of the last), for
 * bindings that pay by the argument. -1 where `which` or `bytes` does not
 * fit. */
#define NSB_CALL_ROPE 0
#define NSB_CALL_ROPE_BWD 1
#define NSB_CALL_KV_APPEND 2
#define NSB_CALL_ATTENTION_PAGED 3
#define NSB_CALL_ATTENTION_WINDOW 4
#define NSB_CALL_ATTENTION_WINDOW_BWD 5
int nsb_op_from_block(int which, const void* args, size_t bytes);

#ifdef __cplusplus
}
#endif

#endif /* NS_B200_OPS_H */
