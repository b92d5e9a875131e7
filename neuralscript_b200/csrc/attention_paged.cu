// Attention of one new token a sequence over a paged cache:
//   out[b, h] = sum over visible j of p_j v_j,  p = softmax(scale * q[b, h] . k_j),
// j visible where j < len and (no window, or j >= len - window, or j < sinks).
//
// Memory-bound: every visible key and value is read once, for all query heads
// that share it. One pass with the running maximum and sum of the softmax.
//
// Work is cut without regard to where sequences end: the visible keys of every
// (sequence, key head), counted in tiles of 64, stand in one line, and every
// block takes the same number of neighbouring tiles of it. (A cut into equal
// parts a sequence leaves the blocks of short ones idle: the lengths of a
// batch differ by a factor of ten and more.) The lengths are on the device,
// so each block sums them up itself. A block writes what it covers whole; of
// a head that other blocks share it leaves maximum, sum and weighted values
// in the workspace, and a second kernel joins those in the order of the keys.
// Nothing depends on timing.
#include <cuda_bf16.h>
#include <math.h>

#include <type_traits>

#include "attention_cache.h"
#include "gemm.h"

namespace nsb {

namespace {

constexpr int kTile = 64;        // keys a tile
constexpr int kThreads = 128;
constexpr int kPerSm = 2;        // blocks an SM that the grid is made for
constexpr int kMinTiles = 2;     // least tiles a block: below, joining costs more than a block saves
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct PagedArgs {
    PagedDesc d;
    int group;   // query heads that share a key head
    int chunks;  // blocks' shares of a group
    int* plan;   // [0]: tiles a block, [1 + b]: tiles before sequence b
    float* part; // [grid][2] maxima, sums [HB] and values [HB][DHP]
};

// Visible keys of a sequence, numbered 0 .. n - 1: the first `front` are the
// sequence's first, the others lie side by side from `back` on.
struct Seen {
    int n, front, back;
};
__device__ __forceinline__ Seen seen_of(const PagedDesc& d, int b) {
    int len = d.lens[b];
    const long long room = min((long long)d.width * d.page, 0x7fffffffLL);
    if (len < 0 || len > room) {
        if (len > 0) atomicCAS(d.err, 0, kErrBadIndex);
        len = len < 0 ? 0 : (int)room;
    }
    Seen s{len, 0, 0};
    if (d.window > 0 && len > d.window) {
        s.back = len - d.window;
        s.front = min(d.sinks, s.back);
        s.n = d.window + s.front;
    }
    return s;
}
__device__ __forceinline__ int tiles_of(int n) { return n > 0 ? (n + kTile - 1) / kTile : 1; }

// pre[b] = tiles of the sequences before b, of one key head (pre: B + 1 ints).
__device__ __forceinline__ void sum_up(const PagedDesc& d, int* pre) {
    __shared__ int s_warp[kThreads / 32];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    int carry = 0;
    if (t == 0) pre[0] = 0;
    for (int b0 = 0; b0 < d.B; b0 += kThreads) {
        int v = b0 + t < d.B ? tiles_of(seen_of(d, b0 + t).n) : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += u;
        }
        if (lane == 31) s_warp[warp] = v;
        __syncthreads();
        int all = 0;
#pragma unroll
        for (int w = 0; w < kThreads / 32; w++) {
            if (w < warp) v += s_warp[w];
            all += s_warp[w];
        }
        if (b0 + t < d.B) pre[b0 + t + 1] = carry + v;
        carry += all;
        __syncthreads();
    }
}

// Output of one head from its maximum (in powers of two), sum and values.
template <typename T>
__device__ __forceinline__ void put(const PagedDesc& d, int b, int h, int c, float m, float l, float o) {
    if (c < d.dh) {
        T* to = (T*)d.out.p + b * d.out.row + h * d.out.head + c;
        const float v = l > 0.f ? o / l : l == 0.f ? 0.f : l;  // nothing seen: 0; NaN stays
        if constexpr (std::is_same<T, float>::value) *to = v;
        else *to = __float2bfloat16_rn(v);
    }
    if (c == 0 && d.lse) d.lse[(long long)b * d.Hq + h] = l > 0.f ? (m + log2f(l)) * kLn2 : l == 0.f ? -INFINITY : l;
}

__device__ __forceinline__ float ldf(const float* p) { return *p; }
__device__ __forceinline__ float ldf(const __nv_bfloat16* p) { return __bfloat162float(*p); }

// A lane's DIMS columns of one head: pieces of 16 bytes, eight lanes apart
// (VEC), or single columns eight apart.
template <typename T, int DIMS, bool VEC>
__device__ __forceinline__ void load_dims(float* r, const T* p, int sub, int dh) {
    if constexpr (VEC) {
        constexpr int W = 16 / sizeof(T);
#pragma unroll
        for (int j = 0; j < DIMS / W; j++) {
            const int c = (j * 8 + sub) * W;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (c < dh) v = *reinterpret_cast<const uint4*>(p + c);
            const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
            for (int i = 0; i < W; i++) r[j * W + i] = ldf(e + i);
        }
    } else {
#pragma unroll
        for (int j = 0; j < DIMS; j++) r[j] = j * 8 + sub < dh ? ldf(p + j * 8 + sub) : 0.f;
    }
}
template <typename T, int DIMS, bool VEC>
__device__ __forceinline__ int dim_of(int j, int sub) {
    constexpr int W = 16 / sizeof(T);
    return VEC ? ((j / W) * 8 + sub) * W + j % W : j * 8 + sub;
}

// Any type, head size and alignment, on the fp32 units: eight lanes hold a
// key, four keys a warp at a time, each with a softmax of its own over every
// sixteenth key of a tile; the sixteen of a block meet at its end. HB query
// heads share what is read.
template <typename T, int DHP, int HB, bool VEC>
__global__ void __launch_bounds__(kThreads) paged_kernel(const __grid_constant__ PagedArgs a) {
    constexpr int DIMS = DHP / 8;
    constexpr int STREAMS = kThreads / 8;
    extern __shared__ int pre[];
    __shared__ float s_m[STREAMS][HB], s_l[STREAMS][HB];
    __shared__ float s_o[STREAMS][DHP];
    const PagedDesc& d = a.d;
    const int t = threadIdx.x, sub = t & 7, stream = t >> 3;
    sum_up(d, pre);
    __syncthreads();
    const int Hc = d.Hkv * a.chunks;
    const long long W = (long long)pre[d.B] * Hc;
    const long long per = max((long long)kMinTiles, (W + gridDim.x - 1) / gridDim.x);
    if (blockIdx.x == 0) {
        for (int b = t; b <= d.B; b += kThreads) a.plan[1 + b] = pre[b];
        if (t == 0) a.plan[0] = (int)per;
    }
    const long long begin = blockIdx.x * per, end = min(W, begin + per);
    const float s2 = d.scale * kLog2e;

    for (long long at = begin; at < end;) {
        int b = 0;
        for (int step = 1 << 13; step; step >>= 1)
            if (b + step < d.B && (long long)pre[b + step] * Hc <= at) b += step;
        const int tiles = pre[b + 1] - pre[b];
        const long long in = at - (long long)pre[b] * Hc;
        const int hc = (int)(in / tiles), i0 = (int)(in - (long long)hc * tiles);
        const int i1 = (int)min((long long)tiles, i0 + (end - at));
        const int hk = hc / a.chunks, g0 = (hc - hk * a.chunks) * HB, h0 = hk * a.group + g0;
        const int heads = min(HB, a.group - g0);
        const Seen s = seen_of(d, b);

        float q[HB][DIMS], o[HB][DIMS], m[HB], l[HB];
#pragma unroll
        for (int g = 0; g < HB; g++) {
            if (g < heads) load_dims<T, DIMS, VEC>(q[g], (const T*)d.q.p + b * d.q.row + (h0 + g) * d.q.head, sub, d.dh);
            m[g] = -INFINITY;
            l[g] = 0.f;
#pragma unroll
            for (int j = 0; j < DIMS; j++) {
                if (g >= heads) q[g][j] = 0.f;
                o[g][j] = 0.f;
            }
        }
        const int last = min(s.n, i1 * kTile);
        for (int x = i0 * kTile + stream; x < last; x += STREAMS) {
            const int key = x < s.front ? x : x - s.front + s.back;
            const int pi = key / d.page;
            const int page = d.table[b * d.ld_table + pi];
            if (page < 0 || page >= d.pages) {  // no such page: its keys are left out
                atomicCAS(d.err, 0, kErrBadIndex);
                continue;
            }
            float k[DIMS], v[DIMS];
            load_dims<T, DIMS, VEC>(k, (const T*)d.kc.p + page * d.kc.page + (key - pi * d.page) * d.kc.slot + hk * d.kc.head,
                                    sub, d.dh);
            load_dims<T, DIMS, VEC>(v, (const T*)d.vc.p + page * d.vc.page + (key - pi * d.page) * d.vc.slot + hk * d.vc.head,
                                    sub, d.dh);
            const uint32_t mates = 0xffu << (threadIdx.x & 24);
#pragma unroll
            for (int g = 0; g < HB; g++) {
                float z = 0.f;
#pragma unroll
                for (int j = 0; j < DIMS; j++) z = fmaf(q[g][j], k[j], z);
                z += __shfl_xor_sync(mates, z, 1);
                z += __shfl_xor_sync(mates, z, 2);
                z += __shfl_xor_sync(mates, z, 4);
                z *= s2;
                const float top = fmaxf(m[g], z), safe = top == -INFINITY ? 0.f : top;
                const float turn = exp2f(m[g] - safe), p = exp2f(z - safe);
                m[g] = top;
                l[g] = l[g] * turn + p;
#pragma unroll
                for (int j = 0; j < DIMS; j++) o[g][j] = fmaf(p, v[j], o[g][j] * turn);
            }
        }
        // the block's streams meet, head by head
        const bool whole = i0 == 0 && i1 == tiles;
        float* part = a.part + ((long long)blockIdx.x * 2 + (at == begin ? 0 : 1)) * (HB * (DHP + 2));
        __syncthreads();
        if (sub == 0) {
#pragma unroll
            for (int g = 0; g < HB; g++) s_m[stream][g] = m[g], s_l[stream][g] = l[g];
        }
#pragma unroll
        for (int g = 0; g < HB; g++) {
            __syncthreads();
#pragma unroll
            for (int j = 0; j < DIMS; j++) s_o[stream][dim_of<T, DIMS, VEC>(j, sub)] = o[g][j];
            __syncthreads();
            if (t < DHP && g < heads) {
                float top = -INFINITY, sum = 0.f, val = 0.f;
                for (int i = 0; i < STREAMS; i++) top = fmaxf(top, s_m[i][g]);
                const float safe = top == -INFINITY ? 0.f : top;
                for (int i = 0; i < STREAMS; i++) {
                    const float w = exp2f(s_m[i][g] - safe);
                    sum = fmaf(s_l[i][g], w, sum);
                    val = fmaf(s_o[i][t], w, val);
                }
                if (whole) {
                    put<T>(d, b, h0 + g, t, top, sum, val);
                } else {
                    part[2 * HB + g * DHP + t] = val;
                    if (t == 0) part[g] = top, part[HB + g] = sum;
                }
            }
        }
        at += i1 - i0;
    }
}

// Joins what several blocks left of one head: eight warps take every eighth
// part, and meet at the end.
template <typename T, int DHP, int HB>
__global__ void __launch_bounds__(256) paged_join_kernel(const __grid_constant__ PagedArgs a) {
    constexpr int C = DHP / 32;
    __shared__ float s_m[8], s_l[8], s_o[8][DHP];
    const PagedDesc& d = a.d;
    cudaGridDependencySynchronize();
    const int Hc = d.Hkv * a.chunks;
    const int b = blockIdx.x / Hc, hc = blockIdx.x - b * Hc, g = blockIdx.y;
    const int hk = hc / a.chunks, g0 = (hc - hk * a.chunks) * HB;
    const long long per = a.plan[0];
    const int before = a.plan[1 + b], tiles = a.plan[2 + b] - before;
    const long long t0 = (long long)before * Hc + (long long)hc * tiles;
    const int c0 = (int)(t0 / per), c1 = (int)((t0 + tiles - 1) / per);
    if (c0 == c1 || g0 + g >= a.group) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float m = -INFINITY, l = 0.f, o[C] = {};
    for (int c = c0 + warp; c <= c1; c += 8) {
        // in the first block the head begins behind others, unless at its very start
        const float* part = a.part + ((long long)c * 2 + (c == c0 && t0 != c * per ? 1 : 0)) * (HB * (DHP + 2));
        const float mc = part[g], lc = part[HB + g];
        const float top = fmaxf(m, mc), safe = top == -INFINITY ? 0.f : top;
        const float turn = exp2f(m - safe), w = exp2f(mc - safe);
        m = top;
        l = fmaf(lc, w, l * turn);
#pragma unroll
        for (int j = 0; j < C; j++) o[j] = fmaf(part[2 * HB + g * DHP + lane + 32 * j], w, o[j] * turn);
    }
    if (lane == 0) s_m[warp] = m, s_l[warp] = l;
#pragma unroll
    for (int j = 0; j < C; j++) s_o[warp][lane + 32 * j] = o[j];
    __syncthreads();
    if (threadIdx.x < DHP) {
        float top = -INFINITY, sum = 0.f, val = 0.f;
        for (int i = 0; i < 8; i++) top = fmaxf(top, s_m[i]);
        const float safe = top == -INFINITY ? 0.f : top;
        for (int i = 0; i < 8; i++) {
            const float w = exp2f(s_m[i] - safe);
            sum = fmaf(s_l[i], w, sum);
            val = fmaf(s_o[i][threadIdx.x], w, val);
        }
        put<T>(d, b, hk * a.group + g0 + g, threadIdx.x, top, sum, val);
    }
}

int heads_a_block(int group) { return group == 1 ? 1 : 4; }
int padded(int dh) { return dh <= 64 ? 64 : 128; }
size_t round16(size_t n) { return (n + 15) / 16 * 16; }
size_t plan_bytes(int B) { return round16((size_t)(B + 2) * sizeof(int)); }

bool vectors(const void* p, long long a, long long b, long long c, int size) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && a * size % 16 == 0 && b * size % 16 == 0 && c * size % 16 == 0;
}

}  // namespace

size_t attention_paged_workspace(int B, int Hq, int Hkv, int dh) {
    if (B <= 0 || Hkv <= 0 || Hq < Hkv || Hq % Hkv || dh <= 0 || dh > kAttnMaxHead) return 0;
    return plan_bytes(B) + (size_t)num_sms() * kPerSm * 2 * heads_a_block(Hq / Hkv) * (padded(dh) + 2) * sizeof(float);
}

int attention_paged_launches() { return 2; }

int attention_paged(const PagedDesc& d, cudaStream_t st) {
    if (d.B < 0 || d.Hkv <= 0 || d.Hq < d.Hkv || d.Hq % d.Hkv || d.dh <= 0 || d.dh > kAttnMaxHead ||
        (d.dtype != kF32 && d.dtype != kBF16))
        return -1;
    if (d.pages < 0 || d.page <= 0 || d.width < 0 || d.ld_table < d.width || d.window < 0 || d.sinks < 0 ||
        !(d.scale > 0.f) || !(d.scale < INFINITY))
        return -1;
    if (d.B > kPagedMaxBatch) return -2;
    if (d.B == 0) return 0;
    // tiles are counted in 32 bits, those of one block too
    const long long room = (long long)d.width * d.page, seen = d.window ? (long long)d.window + d.sinks : room;
    if ((room < seen ? room : seen) / kTile * d.B >= (1LL << 31) - kPagedMaxBatch ||
        (room < seen ? room : seen) / kTile * d.B * d.Hq >= 1LL << 37)
        return -2;
    if (!d.q.p || !d.out.p || !d.lens || (d.width && !d.table) || (d.pages && (!d.kc.p || !d.vc.p))) return -1;
    if (!d.workspace || reinterpret_cast<uintptr_t>(d.workspace) % 16 ||
        d.workspace_bytes < attention_paged_workspace(d.B, d.Hq, d.Hkv, d.dh))
        return -1;
    if (!d.err) return -5;
    PagedArgs a;
    a.d = d;
    a.group = d.Hq / d.Hkv;
    a.plan = reinterpret_cast<int*>(d.workspace);
    a.part = reinterpret_cast<float*>(reinterpret_cast<char*>(d.workspace) + plan_bytes(d.B));
    const int size = d.dtype == kBF16 ? 2 : 4;
    const bool vec = vectors(d.q.p, d.q.row, d.q.head, 0, size) && d.dh * size % 16 == 0 &&
                     vectors(d.kc.p, d.kc.page, d.kc.slot, d.kc.head, size) &&
                     vectors(d.vc.p, d.vc.page, d.vc.slot, d.vc.head, size);
    auto go = [&](auto zero, auto wide, auto many, auto aligned) {
        using T = decltype(zero);
        constexpr int DHP = decltype(wide)::value, HB = decltype(many)::value;
        constexpr bool VEC = decltype(aligned)::value;
        a.chunks = (a.group + HB - 1) / HB;
        paged_kernel<T, DHP, HB, VEC><<<num_sms() * kPerSm, kThreads, (d.B + 1) * sizeof(int), st>>>(a);
        if (cudaGetLastError() != cudaSuccess) return -5;
        // the second kernel is launched while the first runs, and waits for it
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(d.B * d.Hkv * a.chunks), HB);
        cfg.blockDim = dim3(256);
        cfg.stream = st;
        cudaLaunchAttribute at;
        at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at.val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = &at;
        cfg.numAttrs = 1;
        return cudaLaunchKernelEx(&cfg, paged_join_kernel<T, DHP, HB>, a) == cudaSuccess ? 0 : -5;
    };
    using std::integral_constant;
    auto types = [&](auto wide, auto many, auto aligned) {
        return d.dtype == kBF16 ? go(__nv_bfloat16(), wide, many, aligned) : go(0.f, wide, many, aligned);
    };
    auto heads = [&](auto wide, auto aligned) {
        return heads_a_block(a.group) == 1 ? types(wide, integral_constant<int, 1>(), aligned)
                                           : types(wide, integral_constant<int, 4>(), aligned);
    };
    if (d.dh <= 64)
        return vec ? heads(integral_constant<int, 64>(), std::true_type()) : heads(integral_constant<int, 64>(), std::false_type());
    return vec ? heads(integral_constant<int, 128>(), std::true_type()) : heads(integral_constant<int, 128>(), std::false_type());
}

}  // namespace nsb
