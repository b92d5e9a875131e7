// Mixture of experts with k experts a token (no counterpart in the
// reference, whose layer sends a token to one expert): routing, ordering of
// the pairs, weighted sum of the experts' outputs, and their gradients.
#include <cuda_bf16.h>
#include <math.h>

#include "gemm.h"
#include "moe_topk.h"

namespace nsb {

namespace {

constexpr unsigned kAll = 0xffffffffu;

inline int launched() { return cudaGetLastError() == cudaSuccess ? 0 : -5; }

// Order-preserving map of a float that is no NaN to unsigned (both zeros to
// the same value); 0 is left for "not eligible".
__device__ __forceinline__ unsigned ordered(float v) {
    const unsigned u = __float_as_uint(v + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(unsigned u) {
    return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
    return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
    return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kAll, v, o));
    return v;
}

// Scores of this lane's NV consecutive experts, from lane * NV on. Dead
// experts score 0. The softmax's sum is held in 64 bits and rounded once, so
// that the scores, and with them the choice, do not depend on the order of
// the sum.
template <int NV>
__device__ __forceinline__ void scores(const RouteDesc& d, int row, int lane, float* s, unsigned& live) {
    float x[NV];
    live = 0;
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int e = lane * NV + i;
        const bool on = e < d.E && (!d.active || d.active[e]);
        x[i] = on ? ld_any(d.logits, d.dtype, (size_t)row * d.ld + e) : -INFINITY;
        live |= on ? 1u << i : 0u;
    }
    if (d.sigmoid) {
#pragma unroll
        for (int i = 0; i < NV; i++) s[i] = live >> i & 1 ? 1.f / (1.f + expf(-x[i])) : 0.f;
        return;
    }
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < NV; i++) m = fmaxf(m, x[i]);
    m = warp_max(m);
    double sum = 0.;
#pragma unroll
    for (int i = 0; i < NV; i++) {
        s[i] = live >> i & 1 ? expf(x[i] - m) : 0.f;
        sum += s[i];
    }
    const float total = (float)warp_sum(sum);
#pragma unroll
    for (int i = 0; i < NV; i++) s[i] = s[i] / total;
}

// One warp a token; a lane holds NV consecutive experts.
template <int NV>
__global__ void __launch_bounds__(128) route_kernel(const RouteDesc d, int* __restrict__ idx, float* __restrict__ w) {
    const int row = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (row >= d.M) return;
    float s[NV];
    unsigned live, key[NV];
    scores<NV>(d, row, lane, s, live);
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const float v = s[i] + (d.bias && lane * NV + i < d.E ? d.bias[lane * NV + i] : 0.f);
        key[i] = (live >> i & 1) && v > -INFINITY ? ordered(v) : 0u;
    }
    if (d.groups > 1) {
        // A group's score is the sum of its two best keys; lane g (and g + 32,
        // ...) keeps that of group g. The topk_groups best stay.
        const int per = d.E / d.groups;
        unsigned gs[(kTopkMaxE / 2) / 32];
#pragma unroll
        for (int q = 0; q < (kTopkMaxE / 2) / 32; q++) gs[q] = 0;
        for (int g = 0; g < d.groups; g++) {
            unsigned b1 = 0, b2 = 0;
#pragma unroll
            for (int i = 0; i < NV; i++) {
                const int e = lane * NV + i;
                const unsigned v = e / per == g ? key[i] : 0u;
                b2 = max(b2, min(b1, v));
                b1 = max(b1, v);
            }
            const unsigned m1 = __reduce_max_sync(kAll, b1);
            const int owner = __ffs(__ballot_sync(kAll, b1 == m1)) - 1;
            const unsigned m2 = __reduce_max_sync(kAll, lane == owner ? b2 : b1);
            float v = m1 ? unordered(m1) : 0.f;
            if (m2) v += unordered(m2);
#pragma unroll
            for (int q = 0; q < (kTopkMaxE / 2) / 32; q++)
                if (q * 32 + lane == g) gs[q] = m1 ? ordered(v) : 0u;
        }
        for (int t = 0; t < d.groups; t++) {
            unsigned b = 0;
            int bq = 0;
#pragma unroll
            for (int q = 0; q < (kTopkMaxE / 2) / 32; q++)
                if (gs[q] > b) {
                    b = gs[q];
                    bq = q;
                }
            const unsigned m = __reduce_max_sync(kAll, b);
            if (m == 0) break;
            const int g = (int)__reduce_min_sync(kAll, b == m ? (unsigned)(bq * 32 + lane) : ~0u);
#pragma unroll
            for (int q = 0; q < (kTopkMaxE / 2) / 32; q++)
                if (q * 32 + lane == g) gs[q] = 0;
            if (t < d.topk_groups) continue;
#pragma unroll
            for (int i = 0; i < NV; i++)
                if ((lane * NV + i) / per == g) key[i] = 0;
        }
    }
    int mine = -1;
    float got = 0.f;
    for (int j = 0; j < d.k; j++) {
        unsigned b = 0;
        int bi = 0;
#pragma unroll
        for (int i = 0; i < NV; i++)
            if (key[i] > b) {
                b = key[i];
                bi = i;
            }
        const unsigned m = __reduce_max_sync(kAll, b);
        if (m == 0) break;
        const int owner = __ffs(__ballot_sync(kAll, b == m)) - 1;
        float sv = 0.f;
#pragma unroll
        for (int i = 0; i < NV; i++)
            if (i == bi) {
                sv = s[i];
                if (lane == owner) key[i] = 0;
            }
        const int e = __shfl_sync(kAll, lane * NV + bi, owner);
        sv = __shfl_sync(kAll, sv, owner);
        if (lane == j) {
            mine = e;
            got = sv;
        }
    }
    const float total = d.renorm ? warp_sum(got) + 1e-20f : 1.f;
    if (lane < d.k) {
        idx[(size_t)row * d.k + lane] = mine;
        w[(size_t)row * d.k + lane] = d.scale * got / total;
    }
}

__device__ __forceinline__ void st_any(void* p, int dtype, size_t i, float v) {
    if (dtype == kBF16) reinterpret_cast<__nv_bfloat16*>(p)[i] = f2bf(v);
    else reinterpret_cast<float*>(p)[i] = v;
}

// One warp a token: the row's other experts first, then lane j the j-th
// chosen one.
template <int NV>
__global__ void __launch_bounds__(128)
    route_bwd_kernel(const RouteDesc d, const float* __restrict__ dw, const int* __restrict__ idx, void* dlogits,
                     long long ld_d) {
    const int row = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (row >= d.M) return;
    float s[NV];
    unsigned live;
    scores<NV>(d, row, lane, s, live);
    int e = lane < d.k ? idx[(size_t)row * d.k + lane] : -1;
    if (e >= d.E) e = -1;
    float sj = 0.f;
    for (int j = 0; j < d.k; j++) {
        const int ej = __shfl_sync(kAll, e, j);
        float v = 0.f;
#pragma unroll
        for (int i = 0; i < NV; i++)
            if (ej >= 0 && i == ej % NV) v = s[i];
        v = __shfl_sync(kAll, v, ej >= 0 ? ej / NV : 0);
        if (lane == j) sj = v;
    }
    const float g = e >= 0 ? dw[(size_t)row * d.k + lane] : 0.f;
    float ds = d.scale * g;
    if (d.renorm) {
        const float total = warp_sum(sj) + 1e-20f;
        ds = d.scale * (g - warp_sum(g * sj) / total) / total;
    }
    if (e < 0) ds = 0.f;
    const bool any = __any_sync(kAll, e >= 0);
    const float dot = d.sigmoid || !any ? 0.f : warp_sum(ds * sj);
    const size_t base = (size_t)row * ld_d;
#pragma unroll
    for (int i = 0; i < NV; i++)
        if (lane * NV + i < d.E) st_any(dlogits, d.dtype, base + lane * NV + i, dot == 0.f ? 0.f : -s[i] * dot);
    __syncwarp();
    if (e >= 0) st_any(dlogits, d.dtype, base + e, d.sigmoid ? ds * sj * (1.f - sj) : sj * (ds - dot));
}

bool route_ok(const RouteDesc& d) {
    if (d.M < 0 || d.E <= 0 || d.E > kTopkMaxE || d.k <= 0 || d.k > kTopkMaxK || d.k > d.E) return false;
    if (!d.logits || d.ld < d.E || (d.dtype != kF32 && d.dtype != kBF16)) return false;
    if (d.groups < 1 || d.E % d.groups || d.topk_groups < 1 || d.topk_groups > d.groups) return false;
    return d.groups == 1 || d.E / d.groups >= 2;
}

// ---------------------------------------------------------------------------
// Order of the pairs by expert
// ---------------------------------------------------------------------------
constexpr int kOrderThreads = 1024;
constexpr int kOrderWarps = kOrderThreads / 32;

// One block: every warp counts a contiguous share of the pairs, the counts
// are summed over warps and experts, and every warp places its share in the
// same order.
__global__ void __launch_bounds__(kOrderThreads)
    dispatch_kernel(const int* __restrict__ idx, long long P, int E, int align, long long cap, int* offsets, int* counts,
                    int* rows, int* pos) {
    extern __shared__ int sh[];  // [kOrderWarps][E] counts, [E + 1] starts
    int* start = sh + kOrderWarps * E;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int i = threadIdx.x; i < kOrderWarps * E; i += kOrderThreads) sh[i] = 0;
    __syncthreads();
    const long long share = (P + kOrderThreads - 1) / kOrderThreads * 32;
    const long long p0 = share * warp, p1 = min(P, p0 + share);
    int* mine = sh + warp * E;
    for (long long p = p0; p < p1; p += 32) {
        const int e = p + lane < p1 ? idx[p + lane] : -1;
        const unsigned peers = __match_any_sync(kAll, e);
        if (e >= 0 && e < E && lane == __ffs(peers) - 1) mine[e] += __popc(peers);
        __syncwarp();
    }
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += kOrderThreads) {
        int run = 0;
        for (int q = 0; q < kOrderWarps; q++) {
            const int c = sh[q * E + e];
            sh[q * E + e] = run;
            run += c;
        }
        start[e] = run;
        counts[e] = run;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        int at = 0;
        for (int e = 0; e < E; e++) {
            const int c = start[e];
            start[e] = at;
            offsets[e] = at;
            at += (c + align - 1) / align * align;
        }
        start[E] = at;
        offsets[E] = at;
    }
    for (long long r = threadIdx.x; r < cap; r += kOrderThreads) rows[r] = -1;
    __syncthreads();
    for (long long p = p0; p < p1; p += 32) {
        const bool in = p + lane < p1;
        int e = in ? idx[p + lane] : -1;
        if (e >= E) e = -1;
        const unsigned peers = __match_any_sync(kAll, e);
        const int rank = __popc(peers & ((1u << lane) - 1u));
        int at = -1;
        if (e >= 0) at = start[e] + mine[e] + rank;
        __syncwarp();
        if (e >= 0 && rank == 0) mine[e] += __popc(peers);
        __syncwarp();
        if (in) pos[p + lane] = at;
        if (at >= 0) rows[at] = (int)(p + lane);
    }
}

// ---------------------------------------------------------------------------
// Weighted sum of the experts' outputs
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(256)
    combine_kernel(const void* o, int dtype, long long ld_o, const int* __restrict__ pos, const float* __restrict__ w,
                   int k, int D, void* y, long long ld_y) {
    const size_t t = blockIdx.x;
    for (int c = blockIdx.y * blockDim.x + threadIdx.x; c < D; c += gridDim.y * blockDim.x) {
        float acc = 0.f;
        for (int j = 0; j < k; j++) {
            const int p = pos[t * k + j];
            if (p >= 0) acc = fmaf(w ? w[t * k + j] : 1.f, ld_any(o, dtype, (size_t)p * ld_o + c), acc);
        }
        st_any(y, dtype, t * ld_y + c, acc);
    }
}

// One warp a row of the ordered outputs.
__global__ void __launch_bounds__(256)
    combine_bwd_kernel(const void* dy, const void* o, int dtype, long long ld_dy, long long ld_o,
                       const int* __restrict__ rows, const int* __restrict__ pos, const float* __restrict__ w,
                       long long P, int k, int R, int D, void* d_o, long long ld_do, float* dw) {
    const long long gt = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    const long long step = (long long)gridDim.x * blockDim.x;
    if (dw)
        for (long long p = gt; p < P; p += step)
            if (pos[p] < 0) dw[p] = 0.f;
    const int lane = threadIdx.x & 31;
    for (long long r = gt >> 5; r < R; r += step >> 5) {
        const int pair = rows[r];
        const float wp = pair >= 0 && w ? w[pair] : 1.f;
        const size_t t = pair >= 0 ? pair / k : 0;
        float acc = 0.f;
        for (int c = lane; c < D; c += 32) {
            const float g = pair >= 0 ? ld_any(dy, dtype, t * ld_dy + c) : 0.f;
            if (pair >= 0 && dw) acc = fmaf(g, ld_any(o, dtype, (size_t)r * ld_o + c), acc);
            st_any(d_o, dtype, (size_t)r * ld_do + c, wp * g);
        }
        acc = warp_sum(acc);
        if (lane == 0 && pair >= 0 && dw) dw[pair] = acc;
    }
}

}  // namespace

int moe_topk_route(const RouteDesc& d, int* idx, float* w, cudaStream_t st) {
    if (!route_ok(d) || !idx || !w) return -1;
    if (d.M == 0) return 0;
    const unsigned grid = (unsigned)((d.M + 3) / 4);
    const int nv = (d.E + 31) / 32;
    if (nv <= 1) route_kernel<1><<<grid, 128, 0, st>>>(d, idx, w);
    else if (nv <= 2) route_kernel<2><<<grid, 128, 0, st>>>(d, idx, w);
    else if (nv <= 4) route_kernel<4><<<grid, 128, 0, st>>>(d, idx, w);
    else if (nv <= 8) route_kernel<8><<<grid, 128, 0, st>>>(d, idx, w);
    else if (nv <= 16) route_kernel<16><<<grid, 128, 0, st>>>(d, idx, w);
    else route_kernel<32><<<grid, 128, 0, st>>>(d, idx, w);
    return launched();
}

int moe_topk_route_bwd(const RouteDesc& d, const float* dw, const int* idx, void* dl, long long ld_d,
                       cudaStream_t st) {
    if (!route_ok(d) || !idx || !dw || !dl || ld_d < d.E) return -1;
    if (d.M == 0) return 0;
    const unsigned grid = (unsigned)((d.M + 3) / 4);
    const int nv = (d.E + 31) / 32;
    if (nv <= 1) route_bwd_kernel<1><<<grid, 128, 0, st>>>(d, dw, idx, dl, ld_d);
    else if (nv <= 2) route_bwd_kernel<2><<<grid, 128, 0, st>>>(d, dw, idx, dl, ld_d);
    else if (nv <= 4) route_bwd_kernel<4><<<grid, 128, 0, st>>>(d, dw, idx, dl, ld_d);
    else if (nv <= 8) route_bwd_kernel<8><<<grid, 128, 0, st>>>(d, dw, idx, dl, ld_d);
    else if (nv <= 16) route_bwd_kernel<16><<<grid, 128, 0, st>>>(d, dw, idx, dl, ld_d);
    else route_bwd_kernel<32><<<grid, 128, 0, st>>>(d, dw, idx, dl, ld_d);
    return launched();
}

size_t moe_dispatch_rows(long long M, int k, int E, int align) {
    if (M <= 0 || k <= 0 || E <= 0 || align <= 0) return 0;
    const long long P = M * k;
    const long long used = P < E ? P : E;
    return (size_t)((P + used * (align - 1) + align - 1) / align * align);
}

int moe_dispatch(const int* idx, int M, int k, int E, int align, int* offsets, int* counts, int* rows, int* pos,
                 cudaStream_t st) {
    if (M < 0 || k <= 0 || k > kTopkMaxK || E <= 0 || E > kTopkMaxE || align <= 0 || !offsets || !counts) return -1;
    if (M > 0 && (!idx || !rows || !pos)) return -1;
    const size_t cap = moe_dispatch_rows(M, k, E, align);
    if (cap > 0x7fffffffu) return -2;
    const int smem = (kOrderWarps * E + E + 1) * (int)sizeof(int);
    if (smem > 48 * 1024 &&
        cudaFuncSetAttribute(dispatch_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
        return -5;
    dispatch_kernel<<<1, kOrderThreads, smem, st>>>(idx, (long long)M * k, E, align, (long long)cap, offsets, counts,
                                                    rows, pos);
    return launched();
}

int moe_combine(const void* o, int dtype, long long ld_o, const int* pos, const float* w, int M, int k, int D,
                void* y, long long ld_y, cudaStream_t st) {
    if (M < 0 || k <= 0 || k > kTopkMaxK || D <= 0 || (dtype != kF32 && dtype != kBF16) || ld_o < D || ld_y < D)
        return -1;
    if (M == 0) return 0;
    if (!o || !pos || !y) return -1;
    combine_kernel<<<dim3((unsigned)M, (unsigned)((D + 1023) / 1024)), 256, 0, st>>>(o, dtype, ld_o, pos, w, k, D, y,
                                                                                 ld_y);
    return launched();
}

int moe_combine_bwd(const void* dy, const void* o, int dtype, long long ld_dy, long long ld_o, const int* rows,
                    const int* pos, const float* w, int M, int k, int R, int D, void* d_o, long long ld_do, float* dw,
                    cudaStream_t st) {
    if (M < 0 || R < 0 || k <= 0 || k > kTopkMaxK || D <= 0 || (dtype != kF32 && dtype != kBF16)) return -1;
    if (ld_dy < D || ld_do < D || (dw && ld_o < D)) return -1;
    if (M == 0 && R == 0) return 0;
    if (!dy || !rows || !pos || !d_o || (dw && !o)) return -1;
    const long long warps = R > 0 ? R : 1;
    const long long blocks = (warps + 7) / 8, most = (long long)num_sms() * 8;
    combine_bwd_kernel<<<(unsigned)(blocks < most ? blocks : most), 256, 0, st>>>(
        dy, o, dtype, ld_dy, ld_o, rows, pos, w, (long long)M * k, k, R, D, d_o, ld_do, dw);
    return launched();
}

}  // namespace nsb
