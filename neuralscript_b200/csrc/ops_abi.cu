// Kernel-level C-ABI (include/ns_b200_ops.h): thin argument marshalling onto
// the launchers in gemm.cu, kernels.cu and attention.cu.
#include <cuda_bf16.h>
#include <math.h>
#include <string.h>

#include <tuple>

#include "../../include/ns_b200_ops.h"
#include "attention.h"
#include "attention_cache.h"
#include "elementwise.h"
#include "engine.h"
#include "fp8.h"
#include "gemm.h"
#include "kernels.h"
#include "moe.h"
#include "moe_topk.h"

using namespace nsb;

// A call of f with its arguments read from a block in which they stand in
// order, each on a multiple of its size.
template <typename... A>
static int from_block(int (*f)(A...), const void* block, size_t bytes) {
    std::tuple<A...> args{};
    size_t at = 0;
    auto next = [&](auto& to) {
        at = (at + sizeof(to) - 1) / sizeof(to) * sizeof(to);
        if (at + sizeof(to) <= bytes) memcpy(&to, static_cast<const char*>(block) + at, sizeof(to));
        at += sizeof(to);
    };
    std::apply([&](auto&... to) { (next(to), ...); }, args);
    return at == bytes ? std::apply(f, args) : -1;
}

static GemmDesc make_desc(int M, int N, int K, const void* A, int a_dtype, long long lda, int a_mn, const void* B,
                          int b_dtype, long long ldb, int b_mn, int engine) {
    GemmDesc d;
    d.M = M;
    d.N = N;
    d.K = K;
    d.a.ptr = A;
    d.a.dtype = a_dtype;
    d.a.ld = lda;
    d.a.mn_major = a_mn != 0;
    d.b.ptr = B;
    d.b.dtype = b_dtype;
    d.b.ld = ldb;
    d.b.mn_major = b_mn != 0;
    d.engine = engine;
    return d;
}

namespace {
__global__ void exp2_poly3_kernel(const float* __restrict__ x, float* __restrict__ y, size_t n) {
    for (size_t i = blockIdx.x * (size_t)blockDim.x + threadIdx.x; i < n; i += (size_t)gridDim.x * blockDim.x)
        y[i] = exp2_poly3(x[i]);
}

}  // namespace

extern "C" {

int nsb_op_gemm(int M, int N, int K, const void* A, int a_dtype, long long lda, int a_mn, const void* B, int b_dtype,
                long long ldb, int b_mn, float alpha, const float* add, long long ld_add, int act, float* c32,
                long long ldc32, void* c16, long long ldc16, int engine, float* workspace, size_t workspace_floats,
                int* dev_err, void* stream) {
    if (M < 0 || N < 0 || K <= 0 || !A || !B) return -1;
    GemmDesc d = make_desc(M, N, K, A, a_dtype, lda, a_mn, B, b_dtype, ldb, b_mn, engine);
    d.ep.alpha = alpha;
    d.ep.add = add;
    d.ep.ld_add = (int)ld_add;
    d.ep.act = act;
    d.ep.c32 = c32;
    d.ep.ld_c32 = (int)ldc32;
    d.ep.c16 = reinterpret_cast<__nv_bfloat16*>(c16);
    d.ep.ld_c16 = (int)ldc16;
    d.workspace = workspace;
    d.workspace_floats = workspace_floats;
    launch_counter() += 1;
    return gemm(d, (cudaStream_t)stream, dev_err);
}

size_t nsb_op_gemm_workspace_floats(int M, int N, int K, const void* A, int a_dtype, long long lda, int a_mn,
                                    const void* B, int b_dtype, long long ldb, int b_mn, int engine) {
    GemmDesc d = make_desc(M, N, K, A, a_dtype, lda, a_mn, B, b_dtype, ldb, b_mn, engine);
    return gemm_workspace_floats(d);
}

int nsb_op_gemm_uses_tensor_cores(int M, int N, int K, const void* A, int a_dtype, long long lda, int a_mn,
                                  const void* B, int b_dtype, long long ldb, int b_mn, int engine) {
    GemmDesc d = make_desc(M, N, K, A, a_dtype, lda, a_mn, B, b_dtype, ldb, b_mn, engine);
    return gemm_uses_tensor_cores(d) ? 1 : 0;
}

int nsb_op_embedding_fwd(const float* W, const float* ids, int M, int V, int D, float* out32, void* out16,
                         void* stream) {
    return embedding_fwd(W, ids, M, V, D, out32, reinterpret_cast<__nv_bfloat16*>(out16), (cudaStream_t)stream);
}

size_t nsb_op_embedding_bwd_scratch_bytes(int M, int V) { return embedding_bwd_scratch_bytes(M, V); }

int nsb_op_embedding_bwd(const float* dout, const float* ids, int M, int V, int D, float* dW, void* scratch,
                         void* stream) {
    if (!scratch) return -1;
    return embedding_bwd(dout, ids, M, V, D, dW, scratch, (cudaStream_t)stream);
}

int nsb_op_layernorm_fwd(const float* x, int M, int D, float* out32, void* out16, void* stream) {
    return layernorm_fwd(x, M, D, out32, reinterpret_cast<__nv_bfloat16*>(out16), (cudaStream_t)stream);
}

int nsb_op_layernorm_bwd(const float* dy, const float* x, const float* add, int M, int D, float* dx32, void* dx16,
                         void* stream) {
    return layernorm_bwd(dy, x, add, M, D, dx32, reinterpret_cast<__nv_bfloat16*>(dx16), (cudaStream_t)stream);
}

static AttnArgs attn_args(int B, int S, int H, int D, int dtype) {
    AttnArgs a;
    a.B = B;
    a.S = S;
    a.H = H;
    a.D = D;
    a.dh = H > 0 ? D / H : 0;
    a.scale = a.dh > 0 ? 1.0f / sqrtf((float)a.dh) : 1.f;
    a.dtype = dtype;
    return a;
}

int nsb_op_attention_fwd(int B, int S, int H, int D, int dtype, const void* qkv, long long ld_qkv, void* ctx,
                         long long ld_ctx, float* lse, void* stream) {
    if (H <= 0 || D % H) return -1;
    AttnArgs a = attn_args(B, S, H, D, dtype);
    a.qkv = qkv;
    a.ld_qkv = ld_qkv;
    a.ctx = ctx;
    a.ld_ctx = ld_ctx;
    a.lse = lse;
    return attention_fwd(a, (cudaStream_t)stream);
}

int nsb_op_attention_bwd(int B, int S, int H, int D, int dtype, const void* qkv, long long ld_qkv, const void* ctx,
                         long long ld_ctx, const float* lse, const void* dctx, long long ld_dctx, void* dqkv,
                         long long ld_dqkv, float* dvec, void* stream) {
    if (H <= 0 || D % H || !lse || !dvec) return -1;
    AttnArgs a = attn_args(B, S, H, D, dtype);
    a.qkv = qkv;
    a.ld_qkv = ld_qkv;
    a.ctx = const_cast<void*>(ctx);
    a.ld_ctx = ld_ctx;
    a.lse = const_cast<float*>(lse);
    a.dctx = dctx;
    a.ld_dctx = ld_dctx;
    a.dqkv = dqkv;
    a.ld_dqkv = ld_dqkv;
    a.dvec = dvec;
    return attention_bwd(a, (cudaStream_t)stream);
}

int nsb_op_cross_entropy(const float* logits, const float* labels, const int* targets, int M, int C, float denom,
                         float* row_loss, float* d32, void* d16, void* stream) {
    if (!labels && !targets) return -1;
    return cross_entropy_fwd_bwd(logits, labels, targets, M, C, denom, row_loss, d32,
                                 reinterpret_cast<__nv_bfloat16*>(d16), (cudaStream_t)stream);
}

int nsb_op_cross_entropy_finish(void* logits16, int M, int C, const int* targets, const float* tlogit, float denom,
                                float* row_loss, void* stream) {
    if (!logits16 || !targets || !tlogit || !row_loss || M < 0 || C <= 0) return -1;
    launch_counter() += 1;
    return cross_entropy_finish(logits16, M, C, targets, tlogit, denom, row_loss, (cudaStream_t)stream);
}

int nsb_op_reduce_sum(const float* x, int n, float scale, float* out, void* stream) {
    return reduce_sum(x, n, scale, out, (cudaStream_t)stream);
}

int nsb_op_adamw(float* w, const float* g, float* m, float* v, long long n, long long t, float lr, float beta1,
                 float beta2, float one_minus_beta1, float one_minus_beta2, float eps, float decay, void* stream) {
    if (t < 1 || n < 0) return -1;
    AdamTensor a;
    a.w = w;
    a.g = g;
    a.m = m;
    a.v = v;
    a.n = n;
    a.b1t = 1.f - powf(beta1, (float)t);
    a.b2t = 1.f - powf(beta2, (float)t);
    AdamHyper h{lr, beta1, beta2, one_minus_beta1, one_minus_beta2, eps, decay};
    return adamw_single(a, h, (cudaStream_t)stream);
}

int nsb_op_mgs(float* G, int r, int c, void* stream) { return mgs_orthonormalize(G, r, c, (cudaStream_t)stream); }

int nsb_op_moe_route(const float* x, const float* Wg, const unsigned char* active, int M, int D, int E, int* best,
                     float* pb, float* probs, void* stream) {
    if (E <= 0 || E > 64 || D <= 0) return -1;
    return moe_route(x, Wg, active, M, D, E, best, pb, probs, (cudaStream_t)stream);
}

int nsb_op_act_fwd(const float* x, size_t n, int act, float* out32, void* out16, void* stream) {
    return act_fwd_f32(x, n, act, out32, reinterpret_cast<__nv_bfloat16*>(out16), (cudaStream_t)stream);
}

int nsb_op_act_bwd(const float* dy, const float* z, int act, size_t n, float* out32, void* stream) {
    return act_bwd(dy, z, kF32, act, nullptr, n, out32, nullptr, (cudaStream_t)stream);
}


int nsb_op_exp2_poly3(const float* x, float* y, size_t n, void* stream) {
    if (!x || !y) return -1;
    if (n == 0) return 0;
    launch_counter() += 1;
    const unsigned blocks = (unsigned)((n + 255) / 256 < 4096 ? (n + 255) / 256 : 4096);
    exp2_poly3_kernel<<<blocks, 256, 0, (cudaStream_t)stream>>>(x, y, n);
    return cudaGetLastError() == cudaSuccess ? 0 : -5;
}

int nsb_op_softmax(const float* x, int M, int C, float* out32, void* out16, void* stream) {
    if (!x || M < 0 || C <= 0) return -1;
    launch_counter() += 1;
    return softmax_rows(x, M, C, out32, reinterpret_cast<__nv_bfloat16*>(out16), (cudaStream_t)stream);
}

int nsb_op_binop(const float* a, const float* b, size_t n, int code, float* out32, void* out16, void* stream) {
    launch_counter() += 1;
    return binop_fwd(a, b, n, code, out32, reinterpret_cast<__nv_bfloat16*>(out16), (cudaStream_t)stream);
}

int nsb_op_binop_bwd(const float* dout, const float* a, const float* b, size_t n, int code, float* da, float* db,
                     void* stream) {
    launch_counter() += 1;
    return binop_bwd(dout, a, b, n, code, nullptr, da, nullptr, db, (cudaStream_t)stream);
}

static DropoutSite site_of(float rate, unsigned key0, unsigned key1, unsigned step, unsigned site) {
    DropoutSite d;
    d.rate = rate;
    d.key0 = key0;
    d.key1 = key1;
    d.step = step;
    d.site = site;
    return d;
}

int nsb_op_dropout_fwd(const float* x, size_t n, float rate, unsigned key0, unsigned key1, unsigned step,
                       unsigned site, float* out32, void* out16, void* stream) {
    launch_counter() += 1;
    return dropout_fwd(x, n, site_of(rate, key0, key1, step, site), out32, reinterpret_cast<__nv_bfloat16*>(out16),
                       (cudaStream_t)stream);
}

int nsb_op_dropout_bwd(const float* dy, size_t n, float rate, unsigned key0, unsigned key1, unsigned step,
                       unsigned site, float* dx, void* stream) {
    launch_counter() += 1;
    return dropout_bwd(dy, n, site_of(rate, key0, key1, step, site), nullptr, dx, (cudaStream_t)stream);
}

int nsb_op_transpose(const float* in, int R, int C, float* out, void* stream) {
    launch_counter() += 1;
    return transpose2d(in, R, C, out, (cudaStream_t)stream);
}

int nsb_op_concat(const float* a, const float* b, int axis, int rows_a, int rows_b, int ca, int cb, float* out,
                  void* stream) {
    launch_counter() += 1;
    if (axis == 0) {
        if (ca != cb) return -1;
        return concat_rows(a, rows_a, b, rows_b, ca, out, (cudaStream_t)stream);
    }
    if (rows_a != rows_b) return -1;
    return concat_cols(a, ca, b, cb, rows_a, out, nullptr, (cudaStream_t)stream);
}

int nsb_op_slice(const float* in, int axis, int rows, int cols, int start, int end, float* out, void* stream) {
    launch_counter() += 1;
    if (axis == 0) {
        if (start < 0 || end > rows) return -1;
        return slice_rows(in, cols, start, end, out, (cudaStream_t)stream);
    }
    return slice_cols(in, rows, cols, start, end, out, nullptr, (cudaStream_t)stream);
}

int nsb_op_index(const float* in, int axis, int rows, int cols, const long long* idx, int L, float* out,
                 void* stream) {
    launch_counter() += 1;
    const int64_t* ix = reinterpret_cast<const int64_t*>(idx);
    if (axis == 0) return index_rows(in, rows, cols, ix, L, out, (cudaStream_t)stream);
    return index_cols(in, rows, cols, ix, L, out, nullptr, (cudaStream_t)stream);
}

int nsb_op_scatter(const float* in, int axis, int rows, int cols, const long long* idx, int L, const float* upd,
                   float* out, void* stream) {
    launch_counter() += 1;
    const int64_t* ix = reinterpret_cast<const int64_t*>(idx);
    if (axis == 0) return scatter_rows(in, rows, cols, ix, L, upd, out, (cudaStream_t)stream);
    return scatter_cols(in, rows, cols, ix, L, upd, out, nullptr, (cudaStream_t)stream);
}

int nsb_op_gemm_layernorm(int M, int K, const void* A, int dtype, long long lda, const void* B, long long ldb,
                          float alpha, const float* add, long long ld_add, float* c32, long long ldc32, void* c16,
                          long long ldc16, float* rstd, int* dev_err, void* stream) {
    if (M < 0 || K <= 0 || !A || !B || !rstd || (!c32 && !c16)) return -1;
    GemmDesc d = make_desc(M, 512, K, A, dtype, lda, 0, B, dtype, ldb, 1, kEngineTensor);
    d.ep.alpha = alpha;
    d.ep.add = add;
    d.ep.ld_add = (int)ld_add;
    d.ep.c32 = c32;
    d.ep.ld_c32 = (int)ldc32;
    d.ep.c16 = reinterpret_cast<__nv_bfloat16*>(c16);
    d.ep.ld_c16 = (int)ldc16;
    d.ep.ln_rstd = rstd;
    launch_counter() += 1;
    return gemm(d, (cudaStream_t)stream, dev_err);
}

static RouteDesc make_route(const void* logits, int dtype, long long ld, int M, int E, int k, int score,
                            const float* bias, const unsigned char* active, int groups, int topk_groups, int renorm,
                            float scale) {
    RouteDesc d;
    d.logits = logits;
    d.dtype = dtype;
    d.ld = ld;
    d.M = M;
    d.E = E;
    d.k = k;
    d.sigmoid = score == NSB_SCORE_SIGMOID;
    d.bias = bias;
    d.active = active;
    d.groups = groups;
    d.topk_groups = topk_groups;
    d.renorm = renorm != 0;
    d.scale = scale;
    return d;
}

int nsb_op_moe_topk_route(const void* logits, int dtype, long long ld, int M, int E, int k, int score,
                          const float* bias, const unsigned char* active, int groups, int topk_groups, int renorm,
                          float scale, int* idx, float* w, void* stream) {
    if (score != NSB_SCORE_SOFTMAX && score != NSB_SCORE_SIGMOID) return -1;
    launch_counter() += 1;
    return moe_topk_route(make_route(logits, dtype, ld, M, E, k, score, bias, active, groups, topk_groups, renorm, scale),
                          idx, w, (cudaStream_t)stream);
}

int nsb_op_moe_topk_route_bwd(const float* dw, const void* logits, int dtype, long long ld, int M, int E, int k,
                              int score, const unsigned char* active, int renorm, float scale, const int* idx,
                              void* dlogits, long long ld_dlogits, void* stream) {
    if (score != NSB_SCORE_SOFTMAX && score != NSB_SCORE_SIGMOID) return -1;
    launch_counter() += 1;
    return moe_topk_route_bwd(make_route(logits, dtype, ld, M, E, k, score, nullptr, active, 1, 1, renorm, scale), dw,
                              idx, dlogits, ld_dlogits, (cudaStream_t)stream);
}

size_t nsb_op_moe_dispatch_rows(int M, int k, int E, int align) { return moe_dispatch_rows(M, k, E, align); }

int nsb_op_moe_dispatch(const int* idx, int M, int k, int E, int align, int* offsets, int* counts, int* rows, int* pos,
                        void* stream) {
    launch_counter() += 1;
    return moe_dispatch(idx, M, k, E, align, offsets, counts, rows, pos, (cudaStream_t)stream);
}

int nsb_op_moe_combine(const void* o, int dtype, long long ld_o, const int* pos, const float* w, int M, int k, int D,
                       void* y, long long ld_y, void* stream) {
    return nsb_op_moe_combine_rows(o, dtype, ld_o, 0x7fffffff, pos, w, M, k, D, y, ld_y, stream);
}

int nsb_op_moe_combine_rows(const void* o, int dtype, long long ld_o, int R, const int* pos, const float* w, int M,
                            int k, int D, void* y, long long ld_y, void* stream) {
    launch_counter() += 1;
    return moe_combine(o, dtype, ld_o, R, pos, w, M, k, D, y, ld_y, op_error_word(), (cudaStream_t)stream);
}

int nsb_op_moe_combine_bwd(const void* dy, const void* o, int dtype, long long ld_dy, long long ld_o, const int* rows,
                           const int* pos, const float* w, int M, int k, int R, int D, void* d_o, long long ld_do,
                           float* dw, void* stream) {
    launch_counter() += 1;
    return moe_combine_bwd(dy, o, dtype, ld_dy, ld_o, rows, pos, w, M, k, R, D, d_o, ld_do, dw, op_error_word(),
                           (cudaStream_t)stream);
}

int nsb_op_device_error(int* code, void* stream) {
    int* word = op_error_word();
    cudaStream_t st = (cudaStream_t)stream;
    if (!code) return -1;
    if (!word || cudaMemcpyAsync(code, word, sizeof(int), cudaMemcpyDeviceToHost, st) != cudaSuccess ||
        cudaStreamSynchronize(st) != cudaSuccess)
        return -5;
    if (*code && cudaMemsetAsync(word, 0, sizeof(int), st) != cudaSuccess) return -5;
    return 0;
}

int nsb_op_fp8_quantize(const void* x, int dtype, long long ld, int M, int K, int act, const int* rows, int row_div,
                        void* q, long long ld_q, float* s, long long ld_s, void* qt, long long ld_qt, float* st,
                        long long ld_st, void* stream) {
    return nsb_op_fp8_quantize_rows(x, dtype, ld, 0x7fffffff, M, K, act, rows, row_div, q, ld_q, s, ld_s, qt, ld_qt, st,
                                    ld_st, stream);
}

int nsb_op_fp8_quantize_rows(const void* x, int dtype, long long ld, int x_rows, int M, int K, int act, const int* rows,
                             int row_div, void* q, long long ld_q, float* s, long long ld_s, void* qt, long long ld_qt,
                             float* st, long long ld_st, void* stream) {
    QuantDesc d;
    d.x = x;
    d.dtype = dtype;
    d.ld = ld;
    d.x_rows = x_rows;
    d.err = rows ? op_error_word() : nullptr;
    d.M = M;
    d.K = K;
    d.act = act;
    d.rows = rows;
    d.row_div = row_div;
    d.q = reinterpret_cast<uint8_t*>(q);
    d.ld_q = ld_q;
    d.s = s;
    d.ld_s = ld_s;
    d.qt = reinterpret_cast<uint8_t*>(qt);
    d.ld_qt = ld_qt;
    d.st = st;
    d.ld_st = ld_st;
    launch_counter() += 1;
    return fp8_quantize(d, (cudaStream_t)stream);
}

int nsb_op_fp8_quantize_block(const void* x, int dtype, long long ld, int M, int K, void* q, long long ld_q, float* s,
                              long long ld_s, void* qt, long long ld_qt, float* st, long long ld_st, void* stream) {
    QuantDesc d;
    d.x = x;
    d.dtype = dtype;
    d.ld = ld;
    d.M = M;
    d.K = K;
    d.q = reinterpret_cast<uint8_t*>(q);
    d.ld_q = ld_q;
    d.s = s;
    d.ld_s = ld_s;
    d.qt = reinterpret_cast<uint8_t*>(qt);
    d.ld_qt = ld_qt;
    d.st = st;
    d.ld_st = ld_st;
    launch_counter() += 1;
    return fp8_quantize_block(d, (cudaStream_t)stream);
}

int nsb_op_gemm_fp8(int M, int N, int K, const void* A, long long lda, const float* sa, long long ld_sa,
                    const void* B, long long ldb, const float* sb, long long ld_sb, int b_rows, void* C, int c_dtype,
                    long long ldc, int* dev_err, void* stream) {
    Fp8Gemm d;
    d.M = M;
    d.N = N;
    d.K = K;
    d.a = reinterpret_cast<const uint8_t*>(A);
    d.lda = lda;
    d.a_rows = M;
    d.sa = sa;
    d.ld_sa = ld_sa;
    d.b = reinterpret_cast<const uint8_t*>(B);
    d.ldb = ldb;
    d.sb = sb;
    d.ld_sb = ld_sb;
    d.b_rows = b_rows != 0;
    d.c = C;
    d.c_dtype = c_dtype;
    d.ldc = ldc;
    d.err = dev_err ? dev_err : op_error_word();
    launch_counter() += 1;
    return fp8_gemm(d, (cudaStream_t)stream);
}

int nsb_op_moe_gemm_fp8(int R, int E, int N, int K, const void* A, long long lda, int a_rows, const float* sa,
                        long long ld_sa, const int* rows, int row_div, const int* offsets, const int* counts,
                        const void* B, long long ldb, long long b_stride, const float* sb, long long ld_sb,
                        long long sb_stride, void* C, int c_dtype, long long ldc, int* dev_err, void* stream) {
    if (E <= 0 || a_rows < 0 || (!rows && a_rows < R)) return -1;
    Fp8Gemm d;
    d.M = R;
    d.N = N;
    d.K = K;
    d.a = reinterpret_cast<const uint8_t*>(A);
    d.lda = lda;
    d.a_rows = a_rows;
    d.sa = sa;
    d.ld_sa = ld_sa;
    d.b = reinterpret_cast<const uint8_t*>(B);
    d.ldb = ldb;
    d.b_stride = b_stride;
    d.sb = sb;
    d.ld_sb = ld_sb;
    d.sb_stride = sb_stride;
    d.c = C;
    d.c_dtype = c_dtype;
    d.ldc = ldc;
    d.groups = E;
    d.offsets = offsets;
    d.counts = counts;
    d.rows = rows;
    d.row_div = row_div;
    d.err = dev_err ? dev_err : op_error_word();
    launch_counter() += 1;
    return fp8_gemm(d, (cudaStream_t)stream);
}

int nsb_op_moe_wgrad_fp8(int M, int N, int R, int E, const void* A, long long lda, const float* sa, long long ld_sa,
                         const void* B, long long ldb, const float* sb, long long ld_sb, const int* offsets,
                         const int* counts, void* C, int c_dtype, long long ldc, long long c_stride, int* dev_err,
                         void* stream) {
    if (E <= 0) return -1;
    Fp8Gemm d;
    d.M = M;
    d.N = N;
    d.K = R;
    d.a = reinterpret_cast<const uint8_t*>(A);
    d.lda = lda;
    d.a_rows = M;
    d.sa = sa;
    d.ld_sa = ld_sa;
    d.b = reinterpret_cast<const uint8_t*>(B);
    d.ldb = ldb;
    d.sb = sb;
    d.ld_sb = ld_sb;
    d.b_rows = 1;
    d.c = C;
    d.c_dtype = c_dtype;
    d.ldc = ldc;
    d.c_stride = c_stride;
    d.groups = E;
    d.group_k = 1;
    d.offsets = offsets;
    d.counts = counts;
    d.err = dev_err ? dev_err : op_error_word();
    launch_counter() += 1;
    return fp8_gemm(d, (cudaStream_t)stream);
}

static Heads heads(const void* p, long long row, long long head) {
    Heads h;
    h.p = const_cast<void*>(p);
    h.row = row;
    h.head = head;
    return h;
}
static Pages cache(const void* p, long long page, long long slot, long long head) {
    Pages c;
    c.p = const_cast<void*>(p);
    c.page = page;
    c.slot = slot;
    c.head = head;
    return c;
}

// Sections become the pairs' ends, axis by axis; false where they do not add up.
static bool make_turn(Turn* t, const int* pos, long long ld_pos, int axes, const int* sections, const float* freq, int pairs,
                      int interleaved, float scale, float sign) {
    t->n = pairs;
    if (pairs == 0) return true;
    if (axes < 1 || axes > kMaxAxes || (!sections && axes > 1)) return false;
    long long end = 0;
    for (int i = 0; i < axes; i++) {
        if (sections && sections[i] < 0) return false;
        end += sections ? sections[i] : pairs;
        if (end > pairs) return false;
        t->end[i] = (int)end;
    }
    t->pos = pos;
    t->ld_pos = ld_pos;
    t->axes = axes;
    t->freq = freq;
    t->interleaved = interleaved != 0;
    t->scale = scale;
    t->sign = sign;
    return end == pairs;
}

static int turn_heads(const void* x, int dtype, long long x_row, long long x_head, int T, int H, int dh, const int* pos,
                      long long ld_pos, int axes, const int* sections, const float* freq, int pairs, int interleaved,
                      float scale, float sign, void* y, long long y_row, long long y_head, void* stream) {
    Turn t;
    if (!make_turn(&t, pos, ld_pos, axes, sections, freq, pairs, interleaved, scale, sign)) return -1;
    launch_counter() += 1;
    return rope(t, dtype, heads(x, x_row, x_head), heads(y, y_row, y_head), T, H, dh, (cudaStream_t)stream);
}

int nsb_op_rope(const void* x, int dtype, long long x_row, long long x_head, int T, int H, int dh, const int* pos,
                long long ld_pos, int axes, const int* sections, const float* freq, int pairs, int interleaved, float scale,
                void* y, long long y_row, long long y_head, void* stream) {
    return turn_heads(x, dtype, x_row, x_head, T, H, dh, pos, ld_pos, axes, sections, freq, pairs, interleaved, scale, 1.f, y,
                      y_row, y_head, stream);
}

int nsb_op_rope_bwd(const void* dy, int dtype, long long dy_row, long long dy_head, int T, int H, int dh, const int* pos,
                    long long ld_pos, int axes, const int* sections, const float* freq, int pairs, int interleaved,
                    float scale, void* dx, long long dx_row, long long dx_head, void* stream) {
    return turn_heads(dy, dtype, dy_row, dy_head, T, H, dh, pos, ld_pos, axes, sections, freq, pairs, interleaved, scale,
                      -1.f, dx, dx_row, dx_head, stream);
}

int nsb_op_kv_append(const void* k, long long k_row, long long k_head, const void* v, long long v_row, long long v_head,
                     int dtype, int T, int Hkv, int dh, const int* seq, const int* at, const int* table, long long ld_table,
                     int B, int width, int pages, int page, void* k_cache, long long kc_page, long long kc_slot,
                     long long kc_head, void* v_cache, long long vc_page, long long vc_slot, long long vc_head,
                     const int* pos, long long ld_pos, int axes, const int* sections, const float* freq, int pairs,
                     int interleaved, float scale, const void* q, long long q_row, long long q_head, int Hq, void* q_out,
                     long long qo_row, long long qo_head, void* stream) {
    AppendDesc d;
    if (!make_turn(&d.turn, pos, ld_pos, axes, sections, freq, pairs, interleaved, scale, 1.f)) return -1;
    d.dtype = dtype;
    d.T = T;
    d.dh = dh;
    d.Hkv = Hkv;
    d.Hq = Hq;
    d.k = heads(k, k_row, k_head);
    d.v = heads(v, v_row, v_head);
    d.q = heads(q, q_row, q_head);
    d.q_out = heads(q_out, qo_row, qo_head);
    d.seq = seq;
    d.at = at;
    d.table = table;
    d.ld_table = ld_table;
    d.B = B;
    d.width = width;
    d.pages = pages;
    d.page = page;
    d.kc = cache(k_cache, kc_page, kc_slot, kc_head);
    d.vc = cache(v_cache, vc_page, vc_slot, vc_head);
    d.err = op_error_word();
    launch_counter() += 1;
    return kv_append(d, (cudaStream_t)stream);
}

size_t nsb_op_attention_paged_workspace_bytes(int B, int Hq, int Hkv, int dh) {
    return attention_paged_workspace(B, Hq, Hkv, dh);
}

int nsb_op_attention_paged(const void* q, long long q_row, long long q_head, int dtype, int B, int Hq, int Hkv, int dh,
                           const void* k_cache, long long kc_page, long long kc_slot, long long kc_head, const void* v_cache,
                           long long vc_page, long long vc_slot, long long vc_head, int pages, int page, const int* table,
                           long long ld_table, int width, const int* lens, int window, int sinks, float scale, void* out,
                           long long out_row, long long out_head, float* lse, void* workspace, size_t workspace_bytes,
                           void* stream) {
    PagedDesc d;
    d.dtype = dtype;
    d.B = B;
    d.Hq = Hq;
    d.Hkv = Hkv;
    d.dh = dh;
    d.q = heads(q, q_row, q_head);
    d.out = heads(out, out_row, out_head);
    d.kc = cache(k_cache, kc_page, kc_slot, kc_head);
    d.vc = cache(v_cache, vc_page, vc_slot, vc_head);
    d.pages = pages;
    d.page = page;
    d.table = table;
    d.ld_table = ld_table;
    d.width = width;
    d.lens = lens;
    d.window = window;
    d.sinks = sinks;
    d.scale = scale;
    d.lse = lse;
    d.workspace = workspace;
    d.workspace_bytes = workspace_bytes;
    d.err = op_error_word();
    launch_counter() += attention_paged_launches();
    return attention_paged(d, (cudaStream_t)stream);
}

static WindowDesc make_window(const void* q, long long q_row, long long q_head, const void* k, long long k_row,
                              long long k_head, const void* v, long long v_row, long long v_head, int dtype, int T, int Hq,
                              int Hkv, int dh, const int* offsets, int B, int window, int sinks, float scale) {
    WindowDesc d;
    d.dtype = dtype;
    d.T = T;
    d.Hq = Hq;
    d.Hkv = Hkv;
    d.dh = dh;
    d.offsets = offsets;
    d.B = B;
    d.window = window;
    d.sinks = sinks;
    d.scale = scale;
    d.q = heads(q, q_row, q_head);
    d.k = heads(k, k_row, k_head);
    d.v = heads(v, v_row, v_head);
    d.err = op_error_word();
    return d;
}

int nsb_op_attention_window(const void* q, long long q_row, long long q_head, const void* k, long long k_row,
                            long long k_head, const void* v, long long v_row, long long v_head, int dtype, int T, int Hq,
                            int Hkv, int dh, const int* offsets, int B, int window, int sinks, float scale, void* out,
                            long long out_row, long long out_head, float* lse, long long ld_lse, void* stream) {
    WindowDesc d = make_window(q, q_row, q_head, k, k_row, k_head, v, v_row, v_head, dtype, T, Hq, Hkv, dh, offsets, B,
                               window, sinks, scale);
    d.out = heads(out, out_row, out_head);
    d.lse = lse;
    d.ld_lse = ld_lse;
    launch_counter() += 1;
    return attention_window(d, (cudaStream_t)stream);
}

size_t nsb_op_attention_window_bwd_workspace_bytes(int T, int Hq, int Hkv, int dh, int dtype) {
    return attention_window_bwd_workspace(T, Hq, Hkv, dh, dtype);
}

int nsb_op_attention_window_bwd(const void* q, long long q_row, long long q_head, const void* k, long long k_row,
                                long long k_head, const void* v, long long v_row, long long v_head, int dtype, int T,
                                int Hq, int Hkv, int dh, const int* offsets, int B, int window, int sinks, float scale,
                                const void* out, long long out_row, long long out_head, const float* lse, long long ld_lse,
                                const void* dout, long long do_row, long long do_head, void* dq, long long dq_row,
                                long long dq_head, void* dk, long long dk_row, long long dk_head, void* dv,
                                long long dv_row, long long dv_head, void* workspace, size_t workspace_bytes,
                                void* stream) {
    WindowDesc d = make_window(q, q_row, q_head, k, k_row, k_head, v, v_row, v_head, dtype, T, Hq, Hkv, dh, offsets, B,
                               window, sinks, scale);
    d.out = heads(out, out_row, out_head);
    d.lse = const_cast<float*>(lse);
    d.ld_lse = ld_lse;
    d.dout = heads(dout, do_row, do_head);
    d.dq = heads(dq, dq_row, dq_head);
    d.dk = heads(dk, dk_row, dk_head);
    d.dv = heads(dv, dv_row, dv_head);
    d.workspace = workspace;
    d.workspace_bytes = workspace_bytes;
    launch_counter() += attention_window_bwd_launches(d);
    return attention_window_bwd(d, (cudaStream_t)stream);
}

int nsb_op_from_block(int which, const void* args, size_t bytes) {
    if (!args) return -1;
    switch (which) {
        case NSB_CALL_ROPE: return from_block(nsb_op_rope, args, bytes);
        case NSB_CALL_ROPE_BWD: return from_block(nsb_op_rope_bwd, args, bytes);
        case NSB_CALL_KV_APPEND: return from_block(nsb_op_kv_append, args, bytes);
        case NSB_CALL_ATTENTION_PAGED: return from_block(nsb_op_attention_paged, args, bytes);
        case NSB_CALL_ATTENTION_WINDOW: return from_block(nsb_op_attention_window, args, bytes);
        case NSB_CALL_ATTENTION_WINDOW_BWD: return from_block(nsb_op_attention_window_bwd, args, bytes);
    }
    return -1;
}

}  // extern "C"
