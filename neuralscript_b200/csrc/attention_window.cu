// Attention of packed sequences with a sliding window and a few first tokens
// that stay visible, forward and backward:
//   query i of a sequence sees key j where j <= i and (no window, or
//   i - j < window, or j < sinks);
//   out_i = sum_j p_ij v_j,  p_ij = exp(scale q_i.k_j - lse_i).
// With D_i = dout_i . out_i, dS_ij = p_ij (dout_i . v_j - D_i):
//   dq_i = scale sum_j dS_ij k_j,  dk_j = scale sum_i dS_ij q_i,
//   dv_j = sum_i p_ij dout_i, the sums of dk and dv also over the query heads
//   that share the key head.
//
// This file has the form for any type, head size and alignment, on the fp32
// units: tiles of 64 x 64 in shared memory, 4 x 4 scores a thread, every sum
// in fp32 and in a fixed order. The backward pass is two kernels, one that
// keeps queries and walks the keys (dq; it computes D on the way), one that
// keeps keys and walks the queries of all heads that share them (dk, dv), so
// that no sum needs an atomic addition.
//
// Bound by shared memory: 4 x 4 scores a thread take eight 16-byte reads for 64
// FMAs, and 2 x 4 scores on 512 threads were slower (117 to 135 us below). fp32,
// 4096 rows of 8 heads of 64 columns, causal, forward and backward: 3.3 ms, 18
// TFLOP/s (of some 74); 700 rows in 6 sequences, window 100: 26 + 34 + 52 us, of
// which some 39 pass in loading the first tiles and starting.
#include <cuda_bf16.h>
#include <math.h>

#include <type_traits>

#include "attention_cache.h"
#include "attention_window.cuh"
#include "gemm.h"
#include "ptx.cuh"
#include "shared_memory.h"

namespace nsb {

namespace {

constexpr int kB = 64;          // rows of a tile
constexpr int kGroup = 256;     // threads of a product: 16 x 16, 4 x 4 scores each
constexpr int kTwoGroups = 2 * kGroup;
constexpr int kLdS = kB + 4;    // leading dimension of a tile of scores

__device__ __forceinline__ float ldf(const float* p) { return *p; }
__device__ __forceinline__ float ldf(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void stf(float* p, float v) { *p = v; }
__device__ __forceinline__ void stf(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

template <int DHP>
constexpr int ld_of() {
    return DHP + 4;
}

// Rows [first, first + kB) of a head, zeros behind `end` and behind dh. fp32
// rows on 16-byte boundaries are copied without passing through registers
// (`land` waits for them), so that a tile's copies run beside the arithmetic of
// the one before: 2 buffers, as far as shared memory reaches.
template <typename T, int DHP, int THREADS>
__device__ __forceinline__ void load_tile(float* s, const Heads& x, long long row0, int first, int end, int head, int dh) {
    const T* p = (const T*)x.p + head * x.head;
    if constexpr (std::is_same<T, float>::value) {
        if (((reinterpret_cast<uintptr_t>(x.p) >> 2 | x.row | x.head | dh) & 3) == 0) {
            for (int e = threadIdx.x; e < kB * (DHP / 4); e += THREADS) {
                const int r = e / (DHP / 4), c = e % (DHP / 4) * 4;
                const bool on = first + r < end && c < dh;
                ptx::cp_async16(s + r * ld_of<DHP>() + c, on ? p + (row0 + first + r) * x.row + c : (const float*)x.p, on ? 16 : 0);
            }
            return;
        }
    }
    for (int e = threadIdx.x; e < kB * DHP; e += THREADS) {
        const int r = e / DHP, c = e % DHP;
        s[r * ld_of<DHP>() + c] = first + r < end && c < dh ? ldf(p + (row0 + first + r) * x.row + c) : 0.f;
    }
}

__device__ __forceinline__ void land() {
    ptx::cp_async_wait_all();
    __syncthreads();
}
template <int DHP>
constexpr int buffers(int heads, int scores) {  // of `heads` tiles, two of them twice where they fit
    return ((heads + 2) * kB * ld_of<DHP>() + scores * kB * kLdS) * (int)sizeof(float) <= 227 * 1024 ? 2 : 1;
}

// acc[i][j] = sum over the head's columns of a[ty 4 + i] . b[tx + 16 j]
template <int DHP>
__device__ __forceinline__ void dot_tile(float (&acc)[4][4], const float* a, const float* b, int ty, int tx) {
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][j] = 0.f;
#pragma unroll 4
    for (int c = 0; c < DHP; c += 4) {
        float4 x[4], y[4];
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = *reinterpret_cast<const float4*>(a + (ty * 4 + i) * ld_of<DHP>() + c);
#pragma unroll
        for (int j = 0; j < 4; j++) y[j] = *reinterpret_cast<const float4*>(b + (tx + 16 * j) * ld_of<DHP>() + c);
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                acc[i][j] = fmaf(x[i].x, y[j].x, acc[i][j]);
                acc[i][j] = fmaf(x[i].y, y[j].y, acc[i][j]);
                acc[i][j] = fmaf(x[i].z, y[j].z, acc[i][j]);
                acc[i][j] = fmaf(x[i].w, y[j].w, acc[i][j]);
            }
    }
}

// o[i][4 n ..] += sum over r of s[ty 4 + i][r] x[r][64 n + tx 4 ..]
template <int DHP>
__device__ __forceinline__ void add_rows(float (&o)[4][DHP / 16], const float* s, const float* x, int ty, int tx) {
#pragma unroll 2
    for (int r = 0; r < kB; r += 4) {
        float w[4][4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float4 v = *reinterpret_cast<const float4*>(s + (ty * 4 + i) * kLdS + r);
            w[i][0] = v.x, w[i][1] = v.y, w[i][2] = v.z, w[i][3] = v.w;
        }
#pragma unroll
        for (int u = 0; u < 4; u++)
#pragma unroll
            for (int n = 0; n < DHP / 64; n++) {
                const float4 v = *reinterpret_cast<const float4*>(x + (r + u) * ld_of<DHP>() + 64 * n + tx * 4);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    o[i][4 * n] = fmaf(w[i][u], v.x, o[i][4 * n]);
                    o[i][4 * n + 1] = fmaf(w[i][u], v.y, o[i][4 * n + 1]);
                    o[i][4 * n + 2] = fmaf(w[i][u], v.z, o[i][4 * n + 2]);
                    o[i][4 * n + 3] = fmaf(w[i][u], v.w, o[i][4 * n + 3]);
                }
            }
    }
}
// o[i][4 n ..] += sum over r of s[r][ty 4 + i] x[r][64 n + tx 4 ..]
template <int DHP>
__device__ __forceinline__ void add_cols(float (&o)[4][DHP / 16], const float* s, const float* x, int ty, int tx) {
#pragma unroll 4
    for (int r = 0; r < kB; r++) {
        const float4 v4 = *reinterpret_cast<const float4*>(s + r * kLdS + ty * 4);
        const float w[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
        for (int n = 0; n < DHP / 64; n++) {
            const float4 v = *reinterpret_cast<const float4*>(x + r * ld_of<DHP>() + 64 * n + tx * 4);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                o[i][4 * n] = fmaf(w[i], v.x, o[i][4 * n]);
                o[i][4 * n + 1] = fmaf(w[i], v.y, o[i][4 * n + 1]);
                o[i][4 * n + 2] = fmaf(w[i], v.z, o[i][4 * n + 2]);
                o[i][4 * n + 3] = fmaf(w[i], v.w, o[i][4 * n + 3]);
            }
        }
    }
}

template <typename T, int DHP>
__device__ __forceinline__ void store_tile(const float (&o)[4][DHP / 16], const float (&mul)[4], const Heads& x, long long row0,
                                           int first, int end, int head, int dh, int ty, int tx) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int r = first + ty * 4 + i;
        if (r >= end) continue;
        T* p = (T*)x.p + (row0 + r) * x.row + head * x.head;
#pragma unroll
        for (int n = 0; n < DHP / 64; n++)
#pragma unroll
            for (int c = 0; c < 4; c++)
                if (64 * n + tx * 4 + c < dh) stf(p + 64 * n + tx * 4 + c, o[i][4 * n + c] * mul[i]);
    }
}

// Sum over the 16 threads that hold a row of scores (one half of a warp).
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float row_max(float v) {
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

}  // namespace

// grid (tiles, Hq)
template <typename T, int DHP>
__global__ void __launch_bounds__(kGroup) window_fwd_kernel(const __grid_constant__ WindowDesc d) {
    extern __shared__ float sm[];
    constexpr int TILE = kB * ld_of<DHP>(), BUFS = buffers<DHP>(3, 1);
    float *sQ = sm, *sP = sQ + TILE, *ring = sP + kB * kLdS;  // keys and values of each buffer
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const Rows w = find_rows(d, gridDim.x - 1 - blockIdx.x, kB);
    if (w.n <= 0) return;
    const int h = blockIdx.y, hk = h / (d.Hq / d.Hkv), q0 = w.first;
    load_tile<T, DHP, kGroup>(sQ, d.q, w.row0, q0, w.n, h, d.dh);
    float o[4][DHP / 16] = {}, m[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; i++) m[i] = -INFINITY, l[i] = 0.f;
    const KeyTiles kt(d, q0, min(q0 + kB, w.n), kB);
    auto fetch = [&](int x) {
        float* to = ring + x % BUFS * 2 * TILE;
        load_tile<T, DHP, kGroup>(to, d.k, w.row0, kt.at(x) * kB, w.n, hk, d.dh);
        load_tile<T, DHP, kGroup>(to + TILE, d.v, w.row0, kt.at(x) * kB, w.n, hk, d.dh);
    };
    if (BUFS == 2) fetch(0);
    for (int x = 0; x < kt.count; x++) {
        const int k0 = kt.at(x) * kB;
        const float *sK = ring + x % BUFS * 2 * TILE, *sV = sK + TILE;
        if (BUFS == 1) {
            __syncthreads();
            fetch(x);
        }
        land();
        if (BUFS == 2 && x + 1 < kt.count) fetch(x + 1);
        float s[4][4];
        dot_tile<DHP>(s, sQ, sK, ty, tx);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float top = m[i];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                s[i][j] = sees(d, q0 + ty * 4 + i, k0 + tx + 16 * j) ? s[i][j] * d.scale : -INFINITY;
                top = fmaxf(top, s[i][j]);
            }
            top = row_max(top);
            const float safe = top == -INFINITY ? 0.f : top, turn = expf(m[i] - safe);
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float p = expf(s[i][j] - safe);
                sum += p;
                sP[(ty * 4 + i) * kLdS + tx + 16 * j] = p;
            }
            m[i] = top;
            l[i] = l[i] * turn + row_sum(sum);
#pragma unroll
            for (int c = 0; c < DHP / 16; c++) o[i][c] *= turn;
        }
        __syncwarp();  // a row's weights are written and read by one warp
        add_rows<DHP>(o, sP, sV, ty, tx);
    }
    float mul[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        mul[i] = l[i] == 0.f ? 0.f : 1.f / l[i];
        const int r = q0 + ty * 4 + i;
        if (tx == 0 && r < w.n && d.lse) d.lse[h * d.ld_lse + w.row0 + r] = l[i] == 0.f ? -INFINITY : m[i] + logf(l[i]);
    }
    store_tile<T, DHP>(o, mul, d.out, w.row0, q0, w.n, h, d.dh, ty, tx);
}

// dq and D of 64 queries: grid (tiles, Hq). bf16: where few keys are seen, a pass
// before corrects D (few_keys).
template <typename T, int DHP>
__global__ void __launch_bounds__(kGroup) window_bwd_q_kernel(const __grid_constant__ WindowDesc d) {
    extern __shared__ float sm[];
    constexpr int TILE = kB * ld_of<DHP>(), BUFS = buffers<DHP>(4, 1);
    float *sQ = sm, *sG = sQ + TILE, *sS = sG + TILE, *ring = sS + kB * kLdS;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const Rows w = find_rows(d, gridDim.x - 1 - blockIdx.x, kB);
    if (w.n <= 0) return;
    const int h = blockIdx.y, hk = h / (d.Hq / d.Hkv), q0 = w.first;
    load_tile<T, DHP, kGroup>(sQ, d.q, w.row0, q0, w.n, h, d.dh);
    load_tile<T, DHP, kGroup>(sG, d.dout, w.row0, q0, w.n, h, d.dh);
    load_tile<T, DHP, kGroup>(ring, d.out, w.row0, q0, w.n, h, d.dh);
    land();
    float o[4][DHP / 16] = {}, lse[4], D[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int r = q0 + ty * 4 + i;
        float sum = 0.f;
#pragma unroll
        for (int c = 0; c < DHP; c += 16)
            sum = fmaf(sG[(ty * 4 + i) * ld_of<DHP>() + c + tx], ring[(ty * 4 + i) * ld_of<DHP>() + c + tx], sum);
        D[i] = row_sum(sum);
        lse[i] = r < w.n ? d.lse[h * d.ld_lse + w.row0 + r] : -INFINITY;
    }
    const KeyTiles kt(d, q0, min(q0 + kB, w.n), kB);
    // steps of the pass that only sums dS, for what D is short of
    const int first = !std::is_same<T, float>::value && few_keys(d, q0, min(q0 + kB, w.n)) ? kt.count : 0;
    const int steps = first + kt.count;
    float rest[4] = {};
    auto tile_of = [&](int x) { return kt.at(x < first ? x : x - first) * kB; };
    auto fetch = [&](int x) {
        float* to = ring + x % BUFS * 2 * TILE;
        load_tile<T, DHP, kGroup>(to, d.k, w.row0, tile_of(x), w.n, hk, d.dh);
        load_tile<T, DHP, kGroup>(to + TILE, d.v, w.row0, tile_of(x), w.n, hk, d.dh);
    };
    if (BUFS == 2) {
        __syncthreads();  // the outputs have been read
        fetch(0);
    }
    for (int x = 0; x < steps; x++) {
        const int k0 = tile_of(x);
        const float *sK = ring + x % BUFS * 2 * TILE, *sV = sK + TILE;
        if (BUFS == 1) {
            __syncthreads();
            fetch(x);
        }
        land();
        if (BUFS == 2 && x + 1 < steps) fetch(x + 1);
        float s[4][4], g[4][4];
        dot_tile<DHP>(s, sQ, sK, ty, tx);
        dot_tile<DHP>(g, sG, sV, ty, tx);
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const bool on = lse[i] != -INFINITY && sees(d, q0 + ty * 4 + i, k0 + tx + 16 * j);
                s[i][j] = on ? expf(s[i][j] * d.scale - lse[i]) * (g[i][j] - D[i]) : 0.f;
                sS[(ty * 4 + i) * kLdS + tx + 16 * j] = s[i][j];
            }
        if (x < first) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                rest[i] += (s[i][0] + s[i][1]) + (s[i][2] + s[i][3]);
                if (x == first - 1) D[i] += row_sum(rest[i]);
            }
            continue;
        }
        __syncwarp();
        add_rows<DHP>(o, sS, sK, ty, tx);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int r = q0 + ty * 4 + i;
        if (tx == 0 && r < w.n) d.dvec[(long long)h * d.T + w.row0 + r] = D[i];
    }
    const float mul[4] = {d.scale, d.scale, d.scale, d.scale};
    store_tile<T, DHP>(o, mul, d.dq, w.row0, q0, w.n, h, d.dh, ty, tx);
}

// dk and dv of 64 keys: grid (tiles, Hkv). The block has two groups of 256
// threads: the first forms scores and weights, the second dP beside it and dS
// from both, then the first adds to dv and the second to dk. (One group that did
// all four left the SM with eight warps: 700 rows 58 us in place of 52. The
// queries' gradient has three products and gains nothing: 35 us for 34.)
template <typename T, int DHP>
__global__ void __launch_bounds__(kTwoGroups) window_bwd_kv_kernel(const __grid_constant__ WindowDesc d) {
    extern __shared__ float sm[];
    constexpr int TILE = kB * ld_of<DHP>(), BUFS = buffers<DHP>(4, 2);
    float *sK = sm, *sV = sK + TILE, *sP = sV + TILE, *sS = sP + kB * kLdS, *ring = sS + kB * kLdS;
    const int half = threadIdx.x / kGroup, tx = threadIdx.x & 15, ty = threadIdx.x >> 4 & 15;
    const Rows w = find_rows(d, blockIdx.x, kB);
    if (w.n <= 0) return;
    const int hk = blockIdx.y, group = d.Hq / d.Hkv, k0 = w.first;
    load_tile<T, DHP, kTwoGroups>(sK, d.k, w.row0, k0, w.n, hk, d.dh);
    load_tile<T, DHP, kTwoGroups>(sV, d.v, w.row0, k0, w.n, hk, d.dh);
    float o[4][DHP / 16] = {};
    const int first = k0 / kB, each = query_tiles_end(d, k0, w.n, kB) - first, count = each * group;
    auto fetch = [&](int x) {
        float* to = ring + x % BUFS * 2 * TILE;
        const int h = hk * group + x / each, q0 = (first + x % each) * kB;
        load_tile<T, DHP, kTwoGroups>(to, d.q, w.row0, q0, w.n, h, d.dh);
        load_tile<T, DHP, kTwoGroups>(to + TILE, d.dout, w.row0, q0, w.n, h, d.dh);
    };
    if (BUFS == 2) fetch(0);
    for (int x = 0; x < count; x++) {
        const int h = hk * group + x / each, q0 = (first + x % each) * kB;
        const float *sQ = ring + x % BUFS * 2 * TILE, *sG = sQ + TILE;
        if (BUFS == 1) {
            __syncthreads();
            fetch(x);
        }
        float stat[4];  // lse in the first group, D in the second
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = q0 + ty * 4 + i;
            stat[i] = half == 0 ? -INFINITY : 0.f;
            if (r < w.n) stat[i] = half == 0 ? d.lse[h * d.ld_lse + w.row0 + r] : d.dvec[(long long)h * d.T + w.row0 + r];
        }
        land();
        if (BUFS == 2 && x + 1 < count) fetch(x + 1);
        float s[4][4];
        dot_tile<DHP>(s, half ? sG : sQ, half ? sV : sK, ty, tx);
        const int at = ty * 4 * kLdS + tx;
        if (half == 0) {
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const bool on = stat[i] != -INFINITY && sees(d, q0 + ty * 4 + i, k0 + tx + 16 * j);
                    sP[at + i * kLdS + 16 * j] = on ? expf(s[i][j] * d.scale - stat[i]) : 0.f;
                }
        }
        __syncthreads();
        if (half == 1) {
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float p = sP[at + i * kLdS + 16 * j];  // 0 where the key is hidden, whatever its dP is
                    sS[at + i * kLdS + 16 * j] = p == 0.f ? 0.f : p * (s[i][j] - stat[i]);
                }
            asm volatile("bar.sync 1, %0;" ::"n"(kGroup) : "memory");  // its group's dS
        }
        add_cols<DHP>(o, half ? sS : sP, half ? sQ : sG, ty, tx);
    }
    const float m = half ? d.scale : 1.f, mul[4] = {m, m, m, m};
    store_tile<T, DHP>(o, mul, half ? d.dk : d.dv, w.row0, k0, w.n, hk, d.dh, ty, tx);
}

namespace {

template <int DHP>
constexpr int smem_of(int heads, int scores) {
    return ((heads + (buffers<DHP>(heads, scores) - 1) * 2) * kB * ld_of<DHP>() + scores * kB * kLdS) * (int)sizeof(float);
}

int check(const WindowDesc& d) {
    if (d.T < 0 || d.Hkv <= 0 || d.Hq < d.Hkv || d.Hq % d.Hkv || d.dh <= 0 || d.dh > kAttnMaxHead ||
        (d.dtype != kF32 && d.dtype != kBF16) || d.B < 0 || d.window < 0 || d.sinks < 0 || !(d.scale > 0.f) ||
        !(d.scale < INFINITY))
        return -1;
    if (!d.offsets && d.B != 1) return -1;
    // rows are counted in 32 bits, with room for a window's, and so are the steps of one tile of keys
    if (d.Hq > 65535 || d.T > kWindowMaxRows || ((long long)d.T / kB + 1) * (d.Hq / d.Hkv) > 0x7fffffff) return -2;
    return 0;
}

long long tiles_of(const WindowDesc& d, int rows) {
    return d.offsets ? ((long long)d.T + rows - 1) / rows + d.B : ((long long)d.T + rows - 1) / rows;
}

template <typename F>
int by_type(const WindowDesc& d, F go) {
    using std::integral_constant;
    if (d.dtype == kBF16)
        return d.dh <= 64 ? go(__nv_bfloat16(), integral_constant<int, 64>()) : go(__nv_bfloat16(), integral_constant<int, 128>());
    return d.dh <= 64 ? go(0.f, integral_constant<int, 64>()) : go(0.f, integral_constant<int, 128>());
}

}  // namespace

int attention_window(const WindowDesc& d, cudaStream_t st) {
    if (const int bad = check(d)) return bad;
    if (d.T == 0 || d.B == 0) return 0;
    if (!d.q.p || !d.k.p || !d.v.p || !d.out.p || (d.lse && d.ld_lse < d.T)) return -1;
    if (!d.err) return -5;
    if (attention_window_tc_supported(d)) return attention_window_tc(d, st);
    return by_type(d, [&](auto zero, auto wide) {
        using T = decltype(zero);
        constexpr int DHP = decltype(wide)::value, bytes = smem_of<DHP>(3, 1);
        static size_t most[kMaxDevices];
        if (!allow_shared(window_fwd_kernel<T, DHP>, bytes, most)) return -5;
        window_fwd_kernel<T, DHP><<<dim3((unsigned)tiles_of(d, kB), d.Hq), kGroup, bytes, st>>>(d);
        return cudaGetLastError() == cudaSuccess ? 0 : -5;
    });
}

static size_t dvec_bytes(int T, int Hq) { return ((size_t)Hq * T * sizeof(float) + 15) / 16 * 16; }

size_t attention_window_bwd_workspace(int T, int Hq, int Hkv, int dh, int dtype) {
    if (T <= 0 || Hkv <= 0 || Hq < Hkv || Hq % Hkv || dh <= 0 || dh > kAttnMaxHead) return 0;
    return dvec_bytes(T, Hq) + (dtype == kBF16 && dh % 8 == 0 ? attention_window_bwd_tc_parts(dh) : 0);
}

int attention_window_bwd_launches(const WindowDesc& d) { return attention_window_bwd_tc_supported(d) ? 3 : 2; }

int attention_window_bwd(const WindowDesc& given, cudaStream_t st) {
    WindowDesc d = given;
    if (const int bad = check(d)) return bad;
    if (d.T == 0 || d.B == 0) return 0;
    if (!d.q.p || !d.k.p || !d.v.p || !d.out.p || !d.lse || d.ld_lse < d.T || !d.dout.p || !d.dq.p || !d.dk.p || !d.dv.p)
        return -1;
    if (!d.workspace || reinterpret_cast<uintptr_t>(d.workspace) % 16 ||
        d.workspace_bytes < attention_window_bwd_workspace(d.T, d.Hq, d.Hkv, d.dh, d.dtype))
        return -1;
    if (!d.err) return -5;
    d.dvec = reinterpret_cast<float*>(d.workspace);
    d.parts = reinterpret_cast<float*>(reinterpret_cast<char*>(d.workspace) + dvec_bytes(d.T, d.Hq));
    if (attention_window_bwd_tc_supported(d)) return attention_window_bwd_tc(d, st);
    return by_type(d, [&](auto zero, auto wide) {
        using T = decltype(zero);
        constexpr int DHP = decltype(wide)::value, bq = smem_of<DHP>(4, 1), bk = smem_of<DHP>(4, 2);
        static size_t most_q[kMaxDevices], most_kv[kMaxDevices];
        if (!allow_shared(window_bwd_q_kernel<T, DHP>, bq, most_q) || !allow_shared(window_bwd_kv_kernel<T, DHP>, bk, most_kv))
            return -5;
        window_bwd_q_kernel<T, DHP><<<dim3((unsigned)tiles_of(d, kB), d.Hq), kGroup, bq, st>>>(d);
        window_bwd_kv_kernel<T, DHP><<<dim3((unsigned)tiles_of(d, kB), d.Hkv), kTwoGroups, bk, st>>>(d);
        return cudaGetLastError() == cudaSuccess ? 0 : -5;
    });
}

}  // namespace nsb
