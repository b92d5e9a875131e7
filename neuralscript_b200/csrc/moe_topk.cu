// Mixture of experts with k experts a token (no counterpart in the
// reference, whose layer sends a token to one expert): routing, ordering of
// the pairs, weighted sum of the experts' outputs, and their gradients.
#include <cuda_bf16.h>
#include <math.h>

#include <type_traits>

#include "gemm.h"
#include "moe_topk.h"
#include "ptx.cuh"

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

// Logits of this lane's NV consecutive experts, from lane * NV on: 16-byte
// loads where the rows allow them.
template <int NV>
__device__ __forceinline__ void load_logits(const RouteDesc& d, int row, int lane, float* x) {
    const int e0 = lane * NV;
    if (d.vec && e0 + NV <= d.E) {
        if (d.dtype == kF32) {
            const float4* p = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(d.logits) + (size_t)row * d.ld + e0);
#pragma unroll
            for (int i = 0; i < NV / 4; i++) {
                const float4 t = p[i];
                x[4 * i] = t.x, x[4 * i + 1] = t.y, x[4 * i + 2] = t.z, x[4 * i + 3] = t.w;
            }
        } else {
            const uint2* p = reinterpret_cast<const uint2*>(reinterpret_cast<const __nv_bfloat16*>(d.logits) + (size_t)row * d.ld + e0);
#pragma unroll
            for (int i = 0; i < NV / 4; i++) {
                const uint2 t = p[i];
                const __nv_bfloat16* h = reinterpret_cast<const __nv_bfloat16*>(&t);
#pragma unroll
                for (int j = 0; j < 4; j++) x[4 * i + j] = bf2f(h[j]);
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < NV; i++) x[i] = e0 + i < d.E ? ld_any(d.logits, d.dtype, (size_t)row * d.ld + e0 + i) : 0.f;
}

// Which of them live, a bit each.
template <int NV>
__device__ __forceinline__ unsigned living(const RouteDesc& d, int lane) {
    const int e0 = lane * NV;
    const unsigned there = e0 >= d.E ? 0u : d.E - e0 >= NV ? (NV < 32 ? (1u << NV % 32) - 1 : ~0u) : (1u << (d.E - e0)) - 1;
    if (!d.active) return there;
    unsigned live = 0;
    if (NV % 4 == 0 && d.vec_e && e0 + NV <= d.E) {
#pragma unroll
        for (int i = 0; i < NV / 4; i++) {
            const unsigned t = reinterpret_cast<const unsigned*>(d.active + e0)[i];
#pragma unroll
            for (int j = 0; j < 4; j++) live |= t >> 8 * j & 0xff ? 1u << (4 * i + j) : 0u;
        }
        return live;
    }
#pragma unroll
    for (int i = 0; i < NV; i++) live |= (there >> i & 1) && d.active[e0 + i] ? 1u << i : 0u;
    return live;
}

// Scores: sigmoid(x), or exp(x - top) / total over the living. The softmax's
// sum is held in 64 bits and rounded once, so that the scores, and with them
// the choice, do not depend on the order of the sum.
struct Softmax {
    float top = 0.f, total = 1.f;
};
__device__ __forceinline__ float score(const RouteDesc& d, const Softmax& m, float x) {
    return d.sigmoid ? __frcp_rn(1.f + expf(-x)) : expf(x - m.top) / m.total;
}

// Those of this lane's experts; dead ones score 0.
template <int NV>
__device__ __forceinline__ Softmax scores(const RouteDesc& d, int row, int lane, unsigned live, float* s) {
    float x[NV];
    Softmax m;
    load_logits<NV>(d, row, lane, x);
    if (d.sigmoid) {
#pragma unroll
        for (int i = 0; i < NV; i++) s[i] = live >> i & 1 ? score(d, m, x[i]) : 0.f;
        return m;
    }
    m.top = -INFINITY;
#pragma unroll
    for (int i = 0; i < NV; i++)
        if (live >> i & 1) m.top = fmaxf(m.top, x[i]);
    m.top = warp_max(m.top);
    double sum = 0.;
#pragma unroll
    for (int i = 0; i < NV; i++) {
        s[i] = live >> i & 1 ? expf(x[i] - m.top) : 0.f;
        sum += s[i];
    }
    m.total = (float)warp_sum(sum);
#pragma unroll
    for (int i = 0; i < NV; i++) s[i] = s[i] / m.total;
    return m;
}

// A group's score is the sum of its two best keys b1 >= b2 (0: none there).
__device__ __forceinline__ unsigned group_score(unsigned b1, unsigned b2) {
    if (b1 == 0) return 0;
    return ordered(b2 ? unordered(b1) + unordered(b2) : unordered(b1));
}

// One warp a token; a lane holds NV consecutive experts. The k choices are k
// rounds of one warp maximum; only the lane that gave an expert away moves on
// to its next best. Instructions bound it (1075 a row of 256 logits at 60 % of
// the issue slots), not the 16.8 MB that it reads: 16384 x 256, 8 of 256 in 4
// of 8 groups: 20 us, without groups 17.
template <int NV>
__global__ void __launch_bounds__(128) route_kernel(const RouteDesc d, int* __restrict__ idx, float* __restrict__ w) {
    const int row = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (row >= d.M) return;
    const unsigned live = living<NV>(d, lane);
    float s[NV];
    unsigned key[NV];
    const Softmax m = scores<NV>(d, row, lane, live, s);
    if (d.bias) {
        if (NV % 4 == 0 && d.vec_e && lane * NV + NV <= d.E) {
#pragma unroll
            for (int i = 0; i < NV / 4; i++) {
                const float4 t = reinterpret_cast<const float4*>(d.bias + lane * NV)[i];
                s[4 * i] += t.x, s[4 * i + 1] += t.y, s[4 * i + 2] += t.z, s[4 * i + 3] += t.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < NV; i++)
                if (lane * NV + i < d.E) s[i] += d.bias[lane * NV + i];
        }
    }
#pragma unroll
    for (int i = 0; i < NV; i++) key[i] = (live >> i & 1) && s[i] > -INFINITY ? ordered(s[i]) : 0u;
    if (d.lanes > 0) {
        // a group is the experts of `lanes` neighbouring lanes, a power of 2
        unsigned b1 = 0, b2 = 0;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            b2 = max(b2, min(b1, key[i]));
            b1 = max(b1, key[i]);
        }
        for (int o = 1; o < d.lanes; o <<= 1) {
            const unsigned c1 = __shfl_xor_sync(kAll, b1, o), c2 = __shfl_xor_sync(kAll, b2, o);
            b2 = max(min(b1, c1), max(b2, c2));
            b1 = max(b1, c1);
        }
        const unsigned mine = group_score(b1, b2);
        const int g = lane / d.lanes;
        int better = 0;
        for (int o = 0; o < d.groups; o++) {
            const unsigned other = __shfl_sync(kAll, mine, o * d.lanes);
            better += other > mine || (other == mine && o < g);
        }
        if (better >= d.topk_groups) {
#pragma unroll
            for (int i = 0; i < NV; i++) key[i] = 0;
        }
    } else if (d.groups > 1) {
        // any other size: group by group, lane g (and g + 32, ...) keeps the
        // score of group g
        const int per = d.E / d.groups;
        int of[NV];
#pragma unroll
        for (int i = 0; i < NV; i++) of[i] = (lane * NV + i) / per;
        unsigned gs[(kTopkMaxE / 2) / 32];
#pragma unroll
        for (int q = 0; q < (kTopkMaxE / 2) / 32; q++) gs[q] = 0;
        for (int g = 0; g < d.groups; g++) {
            unsigned b1 = 0, b2 = 0;
#pragma unroll
            for (int i = 0; i < NV; i++) {
                const unsigned v = of[i] == g ? key[i] : 0u;
                b2 = max(b2, min(b1, v));
                b1 = max(b1, v);
            }
            const unsigned m1 = __reduce_max_sync(kAll, b1);
            const int owner = __ffs(__ballot_sync(kAll, b1 == m1)) - 1;
            const unsigned m2 = __reduce_max_sync(kAll, lane == owner ? b2 : b1);
            const unsigned v = group_score(m1, m2);
#pragma unroll
            for (int q = 0; q < (kTopkMaxE / 2) / 32; q++)
                if (q * 32 + lane == g) gs[q] = v;
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
                if (of[i] == g) key[i] = 0;
        }
    }
    // this lane's best key b1 of expert i1, and its second best while it is
    // known (two rounds of a lane to one search)
    unsigned b1 = 0, b2 = 0, gone = 0;
    int i1 = 0, i2 = 0;
    auto search = [&] {
        b1 = b2 = 0;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const unsigned v = gone >> i & 1 ? 0u : key[i];
            if (v > b1) {
                b2 = b1, i2 = i1;
                b1 = v, i1 = i;
            } else if (v > b2) {
                b2 = v, i2 = i;
            }
        }
    };
    search();
    bool second = true;
    int mine = -1;
    for (int j = 0; j < d.k; j++) {
        const unsigned top = __reduce_max_sync(kAll, b1);
        if (top == 0) break;
        const int owner = __ffs(__ballot_sync(kAll, b1 == top)) - 1;
        const int e = __shfl_sync(kAll, lane * NV + i1, owner);
        if (lane == j) mine = e;
        if (lane == owner) {
            gone |= 1u << i1;
            if (second) {
                b1 = b2, i1 = i2;
                second = false;
            } else {
                search();
                second = true;
            }
        }
    }
    float got = 0.f;  // the chosen one's score, once more from its logit
    if (mine >= 0) got = score(d, m, ld_any(d.logits, d.dtype, (size_t)row * d.ld + mine));
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

// One warp a token: the row's other experts first (zeros for sigmoid scores,
// which then need no more of the row than the chosen logits), then lane j
// the j-th chosen one. 16384 x 256 fp32: 6 us for sigmoid scores (the 16.8 MB
// written), 11 for softmax, which reads as much again (5.1 us) and is bound by
// instructions (84 % of the issue slots): every score is computed once more.
template <int NV>
__global__ void __launch_bounds__(128)
    route_bwd_kernel(const RouteDesc d, const float* __restrict__ dw, const int* __restrict__ idx, void* dlogits,
                     long long ld_d, int vec_d) {
    const int row = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (row >= d.M) return;
    int e = lane < d.k ? idx[(size_t)row * d.k + lane] : -1;
    if (e >= d.E) e = -1;
    const float g = e >= 0 ? dw[(size_t)row * d.k + lane] : 0.f;
    float s[NV];
    float sj = 0.f;
    if (d.sigmoid) {
        if (e >= 0) sj = score(d, Softmax(), ld_any(d.logits, d.dtype, (size_t)row * d.ld + e));
    } else {
        const Softmax m = scores<NV>(d, row, lane, living<NV>(d, lane), s);
        if (e >= 0) sj = score(d, m, ld_any(d.logits, d.dtype, (size_t)row * d.ld + e));
    }
    float ds = d.scale * g;
    if (d.renorm) {
        const float total = warp_sum(sj) + 1e-20f;
        ds = d.scale * (g - warp_sum(g * sj) / total) / total;
    }
    if (e < 0) ds = 0.f;
    const bool any = __any_sync(kAll, e >= 0);
    const float dot = d.sigmoid || !any ? 0.f : warp_sum(ds * sj);
    const size_t base = (size_t)row * ld_d;
    if (d.sigmoid || !any) {
        const size_t es = d.dtype == kBF16 ? 2 : 4;
        char* p = reinterpret_cast<char*>(dlogits) + base * es;
        if (vec_d) {
            for (int i = lane; i < (int)(d.E * es / 16); i += 32) reinterpret_cast<uint4*>(p)[i] = make_uint4(0, 0, 0, 0);
        } else {
            for (int i = lane; i < d.E; i += 32) st_any(dlogits, d.dtype, base + i, 0.f);
        }
    } else if (vec_d && d.dtype == kF32 && NV % 4 == 0 && lane * NV + NV <= d.E) {
#pragma unroll
        for (int i = 0; i < NV / 4; i++)
            reinterpret_cast<float4*>(reinterpret_cast<float*>(dlogits) + base + lane * NV)[i] =
                make_float4(-s[4 * i] * dot, -s[4 * i + 1] * dot, -s[4 * i + 2] * dot, -s[4 * i + 3] * dot);
    } else {
#pragma unroll
        for (int i = 0; i < NV; i++)
            if (lane * NV + i < d.E) st_any(dlogits, d.dtype, base + lane * NV + i, -s[i] * dot);
    }
    __syncwarp();
    if (e >= 0) st_any(dlogits, d.dtype, base + e, d.sigmoid ? ds * sj * (1.f - sj) : sj * (ds - dot));
}

bool route_ok(const RouteDesc& d) {
    if (d.M < 0 || d.E <= 0 || d.E > kTopkMaxE || d.k <= 0 || d.k > kTopkMaxK || d.k > d.E) return false;
    if ((d.M && !d.logits) || d.ld < d.E || (d.dtype != kF32 && d.dtype != kBF16)) return false;
    if (d.groups < 1 || d.E % d.groups || d.topk_groups < 1 || d.topk_groups > d.groups) return false;
    return d.groups == 1 || d.E / d.groups >= 2;
}

// ---------------------------------------------------------------------------
// Order of the pairs by expert
// ---------------------------------------------------------------------------
constexpr int kOrderThreads = 1024;
constexpr int kOrderWarps = kOrderThreads / 32;
constexpr int kOrderAhead = 8;

// the same word of the shared memory of CTA `rank` of the cluster
__device__ __forceinline__ int cluster_load(const int* p, unsigned rank) {
    int v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(ptx::cluster_addr(p, rank)) : "memory");
    return v;
}

// Lanes whose expert is this lane's (none where that is negative): one ballot
// a bit of the experts' numbers. (__match_any_sync takes a round for every
// different value: 40 us against 27 for 16384 x 8 pairs of 256 experts on 8
// blocks.)
__device__ __forceinline__ unsigned same_expert(int x, int bits) {
    const unsigned there = __ballot_sync(kAll, x >= 0);
    unsigned peers = there;
    for (int b = 0; b < bits; b++) {
        const bool one = x >> b & 1;
        const unsigned m = __ballot_sync(kAll, one);
        peers &= one ? m : ~m;
    }
    return x >= 0 ? peers : 0u;
}

// One cluster of CTAS blocks, one launch: every warp counts a contiguous
// share of the pairs, the counts are summed over the warps of a block, the
// blocks of the cluster (through each other's shared memory) and the experts,
// and every warp places its share in the same order. A pair's rank among its
// 32 neighbours of the same expert comes from ballots, so nothing is
// counted by atomics and the order is the pairs' own.
template <int CTAS>
__global__ void __launch_bounds__(kOrderThreads)
    dispatch_kernel(const int* __restrict__ idx, long long P, int E, int align, long long cap, int* offsets, int* counts,
                    int* rows, int* pos) {
    extern __shared__ int sh[];       // [kOrderWarps][E] counts of the warps
    int* total = sh + kOrderWarps * E;  // [E] of the block
    int* start = total + E;             // [E + 1] first row of an expert
    int* base = start + E + 1;          // [E] this block's first row of it
    int* sums = base + E;               // [kOrderWarps] scan over experts
    int* ends = sums + kOrderWarps;     // [E] row behind an expert's last pair
    const unsigned rank = CTAS > 1 ? ptx::cluster_ctarank() : 0;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int i = threadIdx.x; i < kOrderWarps * E; i += kOrderThreads) sh[i] = 0;
    __syncthreads();
    const long long share = (P + CTAS * kOrderThreads - 1) / (CTAS * kOrderThreads) * 32;
    const long long p0 = share * (rank * kOrderWarps + warp), p1 = min(P, p0 + share);
    int* mine = sh + warp * E;
    const int bits = 32 - __clz(E - 1 | 1);
    int x[kOrderAhead];  // 32 pairs each, all loads in flight before the first is counted
    auto load = [&](long long p) {
#pragma unroll
        for (int i = 0; i < kOrderAhead; i++) {
            x[i] = p + 32 * i + lane < p1 ? idx[p + 32 * i + lane] : -1;
            if (x[i] >= E) x[i] = -1;
        }
    };
    for (long long p = p0; p < p1; p += 32 * kOrderAhead) {
        load(p);
#pragma unroll
        for (int i = 0; i < kOrderAhead; i++) {
            if (p + 32 * i >= p1) break;
            const unsigned peers = same_expert(x[i], bits);
            if (x[i] >= 0 && lane == __ffs(peers) - 1) mine[x[i]] += __popc(peers);
            __syncwarp();
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += kOrderThreads) {
        int run = 0;
#pragma unroll 8
        for (int q = 0; q < kOrderWarps; q++) {
            const int c = sh[q * E + e];
            sh[q * E + e] = run;
            run += c;
        }
        total[e] = run;
    }
    if (CTAS > 1) ptx::cluster_sync();
    else __syncthreads();
    // E <= 1024 threads: thread e sums expert e over the blocks, then the
    // padded counts are scanned over the experts
    const int e = threadIdx.x;
    int all = 0, before = 0;
    if (e < E) {
#pragma unroll
        for (int c = 0; c < CTAS; c++) {
            const int v = CTAS > 1 ? cluster_load(total + e, c) : total[e];
            if (c < (int)rank) before += v;
            all += v;
        }
    }
    const int padded = (all + align - 1) / align * align;
    int inc = padded;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int n = __shfl_up_sync(kAll, inc, o);
        if (lane >= o) inc += n;
    }
    if (lane == 31) sums[warp] = inc;
    __syncthreads();
    if (warp == 0) {
        int v = sums[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int n = __shfl_up_sync(kAll, v, o);
            if (lane >= o) v += n;
        }
        sums[lane] = v;
    }
    __syncthreads();
    if (e < E) {
        const int first = inc - padded + (warp ? sums[warp - 1] : 0);
        base[e] = first + before;
        start[e] = first;
        if (e == E - 1) start[E] = first + padded;
        if (rank == 0) {
            offsets[e] = first;
            counts[e] = all;
            if (e == E - 1) offsets[E] = first + padded;
        }
        ends[e] = first + all;
    }
    __syncthreads();
    for (long long r = start[E] + (long long)rank * kOrderThreads + threadIdx.x; r < cap; r += CTAS * kOrderThreads)
        rows[r] = -1;
    // rows of the padding behind an expert's last pair, a warp an expert
    if (align > 1)
        for (int g = rank * kOrderWarps + warp; g < E; g += CTAS * kOrderWarps)
            for (int r = ends[g] + lane; r < start[g + 1]; r += 32) rows[r] = -1;
    for (long long p = p0; p < p1; p += 32 * kOrderAhead) {
        if (share > 32 * kOrderAhead) load(p);  // (else they are still there)
#pragma unroll
        for (int i = 0; i < kOrderAhead; i++) {
            if (p + 32 * i >= p1) break;
            const unsigned peers = same_expert(x[i], bits);
            const int place = __popc(peers & ((1u << lane) - 1u));
            int at = -1;
            if (x[i] >= 0) at = base[x[i]] + mine[x[i]] + place;
            __syncwarp();
            if (x[i] >= 0 && place == 0) mine[x[i]] += __popc(peers);
            __syncwarp();
            const long long pair = p + 32 * i + lane;
            if (pair < p1) pos[pair] = at;
            if (at >= 0) rows[at] = (int)pair;
        }
    }
    if (CTAS > 1) ptx::cluster_sync();  // no block leaves while others read its counts
}

// ---------------------------------------------------------------------------
// Weighted sum of the experts' outputs
// ---------------------------------------------------------------------------
// 16 bytes of a row as floats and back
template <typename T>
struct Pack;
template <>
struct Pack<float> {
    __device__ static void get(uint4 v, float* f) {
        f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y), f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
    }
    __device__ static uint4 put(const float* f) {
        return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    }
};
template <>
struct Pack<__nv_bfloat16> {
    __device__ static void get(uint4 v, float* f) {
        const __nv_bfloat16* h = reinterpret_cast<const __nv_bfloat16*>(&v);
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] = bf2f(h[i]);
    }
    __device__ static uint4 put(const float* f) {
        uint4 v;
        __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&v);
#pragma unroll
        for (int i = 0; i < 4; i++) h[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        return v;
    }
};

// W columns of a row (16 bytes, or 1 column where rows do not start on 16-byte
// boundaries) as they are loaded, and as floats.
template <typename T, int W>
struct Cols {
    uint4 v;
    __device__ __forceinline__ void load(const T* p) { v = __ldg(reinterpret_cast<const uint4*>(p)); }
    __device__ __forceinline__ void get(float* f) const { Pack<T>::get(v, f); }
    __device__ static __forceinline__ void store(T* p, const float* f) { *reinterpret_cast<uint4*>(p) = Pack<T>::put(f); }
};
template <typename T>
struct Cols<T, 1> {
    float v;
    __device__ __forceinline__ void load(const T* p) { v = (float)*p; }
    __device__ __forceinline__ void get(float* f) const { f[0] = v; }
    __device__ static __forceinline__ void store(T* p, const float* f) {
        if constexpr (sizeof(T) == 2) *p = f2bf(f[0]);
        else *p = f[0];
    }
};

// A thread sums W columns of a token; the rows of four choices are in flight
// together. HBM bounds it: 8192 x 4 rows of 2048 bf16 in 29 us (5.8 TB/s).
template <typename T, int W>
__global__ void __launch_bounds__(128)
    combine_kernel(const T* __restrict__ o, long long ld_o, int R, const int* __restrict__ pos,
                   const float* __restrict__ w, int k, int D, T* __restrict__ y, long long ld_y, int* err) {
    const size_t t = blockIdx.x;
    const int c = (blockIdx.y * blockDim.x + threadIdx.x) * W;
    if (c >= D) return;
    bool past = false;
    float acc[W];
#pragma unroll
    for (int i = 0; i < W; i++) acc[i] = 0.f;
    for (int j0 = 0; j0 < k; j0 += 4) {
        Cols<T, W> in[4];
        float wj[4];
        int p[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            p[j] = j0 + j < k ? pos[t * k + j0 + j] : -1;
            past |= p[j] >= R;
            if (p[j] >= R) p[j] = -1;
            wj[j] = p[j] >= 0 && w ? w[t * k + j0 + j] : 1.f;
        }
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (p[j] >= 0) in[j].load(o + (size_t)p[j] * ld_o + c);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (p[j] < 0) continue;
            float f[W];
            in[j].get(f);
#pragma unroll
            for (int i = 0; i < W; i++) acc[i] = fmaf(wj[j], f[i], acc[i]);
        }
    }
    Cols<T, W>::store(y + t * ld_y + c, acc);
    if (past && err) atomicCAS(err, 0, kErrBadIndex);
}

// One warp a row of the ordered outputs: o and d_o stream, the tokens' dy,
// which k rows share, come out of L2. Four steps of the row are in flight, as
// loaded (16 registers an array, not 32 floats). HBM bounds it: 40960 rows of
// 2048 bf16 in 57 us (5.9 TB/s).
template <typename T, int W>
__global__ void __launch_bounds__(256)
    combine_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ o, long long ld_dy, long long ld_o,
                       const int* __restrict__ rows, const int* __restrict__ pos, const float* __restrict__ w,
                       long long P, int k, int R, int D, T* __restrict__ d_o, long long ld_do, float* __restrict__ dw,
                       int* err) {
    const long long gt = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    const long long step = (long long)gridDim.x * blockDim.x;
    if (dw)
        for (long long p = gt; p < P; p += step)
            if (pos[p] < 0) dw[p] = 0.f;
    const int lane = threadIdx.x & 31;
    int next = gt >> 5 < R ? rows[gt >> 5] : -1;
    for (long long r = gt >> 5; r < R; r += step >> 5) {
        int pair = next;
        if (pair >= P) {
            if (err && lane == 0) atomicCAS(err, 0, kErrBadIndex);
            pair = -1;
        }
        if (r + (step >> 5) < R) next = rows[r + (step >> 5)];
        T* to = d_o + (size_t)r * ld_do;
        if (pair < 0) {
            float zero[W];
#pragma unroll
            for (int i = 0; i < W; i++) zero[i] = 0.f;
            for (int c = lane * W; c < D; c += 32 * W) Cols<T, W>::store(to + c, zero);
            continue;
        }
        const float wp = w ? w[pair] : 1.f;
        const T* g = dy + (size_t)(pair / k) * ld_dy;
        const T* f = o + (size_t)r * ld_o;
        float acc = 0.f;
        for (int c0 = lane * W; c0 < D; c0 += 4 * 32 * W) {
            Cols<T, W> gv[4], fv[4];
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const int c = c0 + q * 32 * W;
                if (c >= D) continue;
                if (dw) fv[q].load(f + c);
                gv[q].load(g + c);
            }
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const int c = c0 + q * 32 * W;
                if (c >= D) continue;
                float gf[W], out[W];
                gv[q].get(gf);
                if (dw) {
                    float ff[W];
                    fv[q].get(ff);
#pragma unroll
                    for (int i = 0; i < W; i++) acc = fmaf(gf[i], ff[i], acc);
                }
#pragma unroll
                for (int i = 0; i < W; i++) out[i] = wp * gf[i];
                Cols<T, W>::store(to + c, out);
            }
        }
        if (dw) {
            acc = warp_sum(acc);
            if (lane == 0) dw[pair] = acc;
        }
    }
}

}  // namespace

namespace {
// f with the smallest of 1, 2, 4, ... experts a lane that holds them all
template <typename F>
void by_lane(int E, F f) {
    const int nv = (E + 31) / 32;
    if (nv <= 1) f(std::integral_constant<int, 1>());
    else if (nv <= 2) f(std::integral_constant<int, 2>());
    else if (nv <= 4) f(std::integral_constant<int, 4>());
    else if (nv <= 8) f(std::integral_constant<int, 8>());
    else if (nv <= 16) f(std::integral_constant<int, 16>());
    else f(std::integral_constant<int, 32>());
}

bool rows16(const void* p, long long ld, int dtype) {
    return !(reinterpret_cast<uintptr_t>(p) & 15) && ld * (dtype == kBF16 ? 2 : 4) % 16 == 0;
}
bool experts16(const RouteDesc& d) {
    return !((reinterpret_cast<uintptr_t>(d.bias) | reinterpret_cast<uintptr_t>(d.active)) & 15);
}
}  // namespace

int moe_topk_route(const RouteDesc& d0, int* idx, float* w, cudaStream_t st) {
    if (!route_ok(d0)) return -1;
    if (d0.M == 0) return 0;
    if (!idx || !w) return -1;
    RouteDesc d = d0;
    by_lane(d.E, [&](auto n) {
        constexpr int NV = decltype(n)::value;
        d.vec = NV >= 4 && rows16(d.logits, d.ld, d.dtype);
        d.vec_e = experts16(d);
        const int per = d.E / d.groups;
        if (d.groups > 1 && per % NV == 0 && (per / NV & (per / NV - 1)) == 0) d.lanes = per / NV;
        route_kernel<NV><<<(unsigned)((d.M + 3) / 4), 128, 0, st>>>(d, idx, w);
    });
    return launched();
}

int moe_topk_route_bwd(const RouteDesc& d0, const float* dw, const int* idx, void* dl, long long ld_d,
                       cudaStream_t st) {
    if (!route_ok(d0) || ld_d < d0.E) return -1;
    if (d0.M == 0) return 0;
    if (!idx || !dw || !dl) return -1;
    RouteDesc d = d0;
    by_lane(d.E, [&](auto n) {
        constexpr int NV = decltype(n)::value;
        d.vec = NV >= 4 && rows16(d.logits, d.ld, d.dtype);
        d.vec_e = experts16(d);
        const int vec_d = rows16(dl, ld_d, d.dtype) && d.E * (d.dtype == kBF16 ? 2 : 4) % 16 == 0;
        route_bwd_kernel<NV><<<(unsigned)((d.M + 3) / 4), 128, 0, st>>>(d, dw, idx, dl, ld_d, vec_d);
    });
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
    const long long P = (long long)M * k;
    auto bytes = [](int experts) { return (kOrderWarps * experts + 4 * experts + 1 + kOrderWarps) * (int)sizeof(int); };
    const int smem = bytes(E);
    auto go = [&](auto ctas) {
        constexpr int CTAS = decltype(ctas)::value;
        auto f = dispatch_kernel<CTAS>;
        // Once a device, to the most that any E takes: a limit set for this E
        // would be another thread's, which launches with more.
        static bool done[kMaxDevices] = {};
        int dev = 0;
        if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return false;
        if (!done[dev]) {
            if (cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes(kTopkMaxE)) != cudaSuccess ||
                (CTAS > 8 && cudaFuncSetAttribute(f, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess))
                return false;
            done[dev] = true;
        }
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(CTAS);
        cfg.blockDim = dim3(kOrderThreads);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = st;
        cudaLaunchAttribute at;
        at.id = cudaLaunchAttributeClusterDimension;
        at.val.clusterDim.x = CTAS;
        at.val.clusterDim.y = at.val.clusterDim.z = 1;
        cfg.attrs = &at;
        cfg.numAttrs = 1;
        return cudaLaunchKernelEx(&cfg, f, idx, P, E, align, (long long)cap, offsets, counts, rows, pos) == cudaSuccess;
    };
    // One block needs no cluster's barriers; 16 (where the device lets so many
    // meet) place the larger numbers faster: 8192 x 4 pairs 9.6 us on 8, 7.6 on
    // 16, 16384 x 8 pairs 27 and 16.
    if (P <= kOrderThreads) return go(std::integral_constant<int, 1>()) ? 0 : -5;
    if (P > 8 * kOrderThreads) {
        if (go(std::integral_constant<int, 16>())) return 0;
        cudaGetLastError();
    }
    return go(std::integral_constant<int, 8>()) ? 0 : -5;
}

int moe_combine(const void* o, int dtype, long long ld_o, int R, const int* pos, const float* w, int M, int k, int D,
                void* y, long long ld_y, int* err, cudaStream_t st) {
    if (M < 0 || R < 0 || k <= 0 || k > kTopkMaxK || D <= 0 || (dtype != kF32 && dtype != kBF16) || ld_o < D || ld_y < D)
        return -1;
    if (M == 0) return 0;
    if ((R && !o) || !pos || !y) return -1;
    const bool vec = rows16(o, ld_o, dtype) && rows16(y, ld_y, dtype) && D % (dtype == kBF16 ? 8 : 4) == 0;
    auto go = [&](auto zero, auto width) {
        using T = decltype(zero);
        constexpr int W = decltype(width)::value;
        const int cols = (D + W - 1) / W, threads = cols < 128 ? (cols + 31) / 32 * 32 : 128;
        combine_kernel<T, W><<<dim3((unsigned)M, (unsigned)((cols + threads - 1) / threads)), threads, 0, st>>>(
            (const T*)o, ld_o, R, pos, w, k, D, (T*)y, ld_y, err);
    };
    if (dtype == kBF16) {
        if (vec) go(__nv_bfloat16(), std::integral_constant<int, 8>());
        else go(__nv_bfloat16(), std::integral_constant<int, 1>());
    } else {
        if (vec) go(0.f, std::integral_constant<int, 4>());
        else go(0.f, std::integral_constant<int, 1>());
    }
    return launched();
}

int moe_combine_bwd(const void* dy, const void* o, int dtype, long long ld_dy, long long ld_o, const int* rows,
                    const int* pos, const float* w, int M, int k, int R, int D, void* d_o, long long ld_do, float* dw,
                    int* err, cudaStream_t st) {
    if (M < 0 || R < 0 || k <= 0 || k > kTopkMaxK || D <= 0 || (dtype != kF32 && dtype != kBF16)) return -1;
    if (ld_dy < D || ld_do < D || (dw && ld_o < D)) return -1;
    if (M == 0 && R == 0) return 0;
    if (!dy || !rows || !pos || !d_o || (dw && !o)) return -1;
    const long long warps = R > 0 ? R : 1;
    const long long blocks = (warps + 7) / 8, most = (long long)num_sms() * 8;
    const bool vec = rows16(dy, ld_dy, dtype) && (!o || rows16(o, ld_o, dtype)) && rows16(d_o, ld_do, dtype) &&
                     D % (dtype == kBF16 ? 8 : 4) == 0;
    auto go = [&](auto zero, auto width) {
        using T = decltype(zero);
        constexpr int W = decltype(width)::value;
        combine_bwd_kernel<T, W><<<(unsigned)(blocks < most ? blocks : most), 256, 0, st>>>(
            (const T*)dy, (const T*)o, ld_dy, ld_o, rows, pos, w, (long long)M * k, k, R, D, (T*)d_o, ld_do, dw,
            err);
    };
    if (dtype == kBF16) {
        if (vec) go(__nv_bfloat16(), std::integral_constant<int, 8>());
        else go(__nv_bfloat16(), std::integral_constant<int, 1>());
    } else {
        if (vec) go(0.f, std::integral_constant<int, 4>());
        else go(0.f, std::integral_constant<int, 1>());
    }
    return launched();
}

}  // namespace nsb
