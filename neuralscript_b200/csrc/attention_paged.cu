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
#include "ptx.cuh"

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

// A lane's DIMS columns of one head, eight apart.
template <typename T, int DIMS>
__device__ __forceinline__ void load_dims(float* r, const T* p, int sub, int dh) {
#pragma unroll
    for (int j = 0; j < DIMS; j++) r[j] = j * 8 + sub < dh ? ldf(p + j * 8 + sub) : 0.f;
}

// Any type, head size and alignment, on the fp32 units: eight lanes hold a
// key, four keys a warp at a time, each with a softmax of its own over every
// sixteenth key of a tile; the sixteen of a block meet at its end. HB query
// heads share what is read.
template <typename T, int DHP, int HB>
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
            if (g < heads) load_dims<T, DIMS>(q[g], (const T*)d.q.p + b * d.q.row + (h0 + g) * d.q.head, sub, d.dh);
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
            load_dims<T, DIMS>(k, (const T*)d.kc.p + page * d.kc.page + (key - pi * d.page) * d.kc.slot + hk * d.kc.head,
                                    sub, d.dh);
            load_dims<T, DIMS>(v, (const T*)d.vc.p + page * d.vc.page + (key - pi * d.page) * d.vc.slot + hk * d.vc.head,
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
            for (int j = 0; j < DIMS; j++) s_o[stream][j * 8 + sub] = o[g][j];
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

// ---------------------------------------------------------------------------
// The same from 16-byte pieces. Each of four warps takes 16 keys of every
// tile, through a ring of its own in shared memory that cp.async fills some
// tiles ahead, over the borders of heads and sequences too: no barrier of the
// block stands between two tiles. Pieces of a row are exchanged by the row's
// lowest three bits, so that neither reading rows nor columns meets a bank
// twice. What is behind a sequence's end, or on no page, arrives as zeros.
//
// bf16: on the tensor cores (m16n8k16), the keys as the product's rows and 8
// query heads its columns, S^T = K Q^T; the weights (rounded to bf16, half a
// step of 2^-9; their sum is taken before) turn into the second product's
// columns by a transpose in registers, O^T += V^T P^T. Groups of fewer heads
// leave columns empty, which costs nothing: the bytes take the time.
// fp32: on the fp32 units, two lanes a key for the scores, and four columns a
// lane for the values.
// ---------------------------------------------------------------------------
constexpr int kWarps = kThreads / 32;
constexpr int kKeys = kTile / kWarps;  // of a warp in a tile: 16

template <typename T, int DHP>
struct Ring {
    static constexpr int ROW = DHP * (int)sizeof(T);
    static constexpr int STAGE = 2 * kKeys * ROW;  // keys, values
    static constexpr int STAGES = ROW == 128 ? 6 : 3;
    static constexpr int MEET = 4;  // heads whose results meet at a time
    static constexpr int BYTES = kWarps * STAGES * STAGE + kWarps * MEET * (DHP + 2) * 4 + kWarps * STAGES * 4;
    static constexpr int PER_SM = BYTES <= 108 * 1024 ? 2 : 1;
};

// Where a warp's next tile is; `offset`: of this lane's row, -1 for none
// (lanes 0 .. 15 the keys', 16 .. 31 the values' rows).
struct Cursor {
    int b, hc, i, tiles;
    Seen s;
    int page;  // of the row, from the table; -1: no such key
    int place;
};

__device__ __forceinline__ void look_up(const PagedArgs& a, Cursor& c, bool real) {
    const int x = c.i * kTile + (threadIdx.x >> 5) * kKeys + (threadIdx.x & (kKeys - 1));
    c.page = -1;
    if (real && x < c.s.n) {
        const int key = x < c.s.front ? x : x - c.s.front + c.s.back;
        const int pi = key / a.d.page;
        c.place = key - pi * a.d.page;
        c.page = a.d.table[c.b * a.d.ld_table + pi];
        if (c.page < 0 || c.page >= a.d.pages) {
            c.page = -1;
            atomicCAS(a.d.err, 0, kErrBadIndex);
        }
    }
}

template <typename T, int DHP>
__device__ __forceinline__ void fetch(const PagedArgs& a, const Cursor& c, uint8_t* stage, uint32_t* mask) {
    constexpr int PIECES = DHP * (int)sizeof(T) / 16, ROWS = 32 / PIECES > 0 ? 32 / PIECES : 1;
    const int lane = threadIdx.x & 31;
    const int hk = c.hc / a.chunks;
    const Pages& mine = lane < kKeys ? a.d.kc : a.d.vc;
    const long long offset = c.page < 0 ? -1 : c.page * mine.page + c.place * mine.slot + hk * mine.head;
    const uint32_t there = __ballot_sync(0xffffffffu, c.page >= 0);
    if (lane == 0) *mask = there;
    const int piece = lane % PIECES;
    const bool inside = piece * 16 < a.d.dh * (int)sizeof(T);
#pragma unroll
    for (int r0 = 0; r0 < 2 * kKeys; r0 += ROWS) {  // rows of the keys, then of the values
        const int row = r0 + lane / PIECES;
        const long long at = __shfl_sync(0xffffffffu, offset, row);
        const T* base = (const T*)(r0 < kKeys ? a.d.kc.p : a.d.vc.p);
        const bool on = at >= 0 && inside;
        ptx::cp_async16(stage + row * (DHP * (int)sizeof(T)) + ((piece ^ (row & 7)) << 4),
                        on ? base + at + piece * (16 / (int)sizeof(T)) : (const T*)a.d.q.p, on ? 16 : 0);
    }
}

__device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void wait_but() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t* r, uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at));
}
__device__ __forceinline__ void ldsm4_t(uint32_t* r, uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at));
}
__device__ __forceinline__ uint32_t turned(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// What a warp keeps of its keys for HB heads: bf16.
template <typename T, int DHP, int HB>
struct State {
    static constexpr int NT = HB / 8, KS = DHP / 16;
    uint32_t q[NT][KS][2];
    float o[KS][NT][4];  // columns of the head 16 k + lane / 4 (+ 8), heads 2 (lane % 4) (+ 1)
    float m[NT][2], l[NT][2];

    __device__ __forceinline__ void start(const PagedDesc& d, int b, int h0, int heads, float*) {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const int h = n * 8 + lane / 4;
            const __nv_bfloat16* p = (const __nv_bfloat16*)d.q.p + b * d.q.row + (h0 + h) * d.q.head;
#pragma unroll
            for (int k = 0; k < KS; k++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int c = 16 * k + 8 * e + 2 * (lane & 3);
                    q[n][k][e] = h < heads && c < d.dh ? *reinterpret_cast<const uint32_t*>(p + c) : 0u;
                }
            m[n][0] = m[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.f;
#pragma unroll
            for (int k = 0; k < KS; k++) o[k][n][0] = o[k][n][1] = o[k][n][2] = o[k][n][3] = 0.f;
        }
    }
    __device__ __forceinline__ void add(uint32_t stage, uint32_t mask, float s2, const float*) {
        const int lane = threadIdx.x & 31;
        constexpr int ROW = DHP * 2;
        float s[NT][4] = {};
        {
            const int row = lane & 15;
            const uint32_t at = stage + row * ROW;
#pragma unroll
            for (int k = 0; k < KS; k++) {
                uint32_t a[4];
                ldsm4(a, at + (((2 * k + (lane >> 4)) ^ (row & 7)) << 4));
#pragma unroll
                for (int n = 0; n < NT; n++) mma16816(s[n], a, q[n][k][0], q[n][k][1]);
            }
        }
        const bool on0 = mask >> (lane >> 2) & 1, on1 = mask >> ((lane >> 2) + 8) & 1;
        uint32_t p[NT][2];
        bool rise = false;
        float turn[NT][2];
#pragma unroll
        for (int n = 0; n < NT; n++) {
#pragma unroll
            for (int e = 0; e < 2; e++) {
                s[n][e] = on0 ? s[n][e] * s2 : -INFINITY;
                s[n][2 + e] = on1 ? s[n][2 + e] * s2 : -INFINITY;
                float top = fmaxf(s[n][e], s[n][2 + e]);
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                top = fmaxf(top, m[n][e]);
                const float safe = top == -INFINITY ? 0.f : top;
                turn[n][e] = exp2f(m[n][e] - safe);
                rise |= top != m[n][e];
                m[n][e] = top;
                s[n][e] = exp2f(s[n][e] - safe);
                s[n][2 + e] = exp2f(s[n][2 + e] - safe);
                l[n][e] = fmaf(l[n][e], turn[n][e], s[n][e] + s[n][2 + e]);
            }
            const __nv_bfloat162 lo = __floats2bfloat162_rn(s[n][0], s[n][1]), hi = __floats2bfloat162_rn(s[n][2], s[n][3]);
            p[n][0] = turned(*reinterpret_cast<const uint32_t*>(&lo));
            p[n][1] = turned(*reinterpret_cast<const uint32_t*>(&hi));
        }
        if (__any_sync(0xffffffffu, rise)) {
#pragma unroll
            for (int k = 0; k < KS; k++)
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int e = 0; e < 4; e++) o[k][n][e] *= turn[n][e & 1];
        }
        const int row = (lane & 7) + ((lane >> 4) << 3);
        const uint32_t at = stage + kKeys * ROW + row * ROW;
#pragma unroll
        for (int k = 0; k < KS; k++) {
            uint32_t a[4];
            ldsm4_t(a, at + (((2 * k + (lane >> 3 & 1)) ^ (row & 7)) << 4));
#pragma unroll
            for (int n = 0; n < NT; n++) mma16816(o[k][n], a, p[n][0], p[n][1]);
        }
    }
    // maxima [4], sums [4] and values [4][DHP] of heads 4 round .. + 3
    __device__ __forceinline__ void leave(float* to, int round) {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int n = 0; n < NT; n++) {
            if (n != round >> 1) continue;
#pragma unroll
            for (int e = 0; e < 2; e++) {
                float sum = l[n][e];
                sum += __shfl_xor_sync(0xffffffffu, sum, 4);
                sum += __shfl_xor_sync(0xffffffffu, sum, 8);
                sum += __shfl_xor_sync(0xffffffffu, sum, 16);
                const int h = 2 * (lane & 1) + e;
                if ((lane >> 1 & 1) != (round & 1)) continue;
                if (lane < 4) to[h] = m[n][e], to[4 + h] = sum;
#pragma unroll
                for (int k = 0; k < KS; k++) {
                    to[8 + h * DHP + 16 * k + (lane >> 2)] = o[k][n][e];
                    to[8 + h * DHP + 16 * k + (lane >> 2) + 8] = o[k][n][2 + e];
                }
            }
        }
    }
};

// fp32; the queries lie in shared memory.
template <int DHP, int HB>
struct State<float, DHP, HB> {
    static constexpr int COLS = DHP / 4, SHARE = 32 / COLS;  // lanes of 4 columns; how many share 16 keys
    float o[HB][4], m[HB], l[HB];

    __device__ __forceinline__ void start(const PagedDesc& d, int b, int h0, int heads, float* q) {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int g = 0; g < HB; g++) {
            const float* p = (const float*)d.q.p + b * d.q.row + (h0 + g) * d.q.head;
            for (int c = lane; c < DHP; c += 32) q[g * DHP + c] = g < heads && c < d.dh ? p[c] : 0.f;
            m[g] = -INFINITY;
            l[g] = 0.f;
            o[g][0] = o[g][1] = o[g][2] = o[g][3] = 0.f;
        }
        __syncwarp();
    }
    __device__ __forceinline__ void add(const uint8_t* stage, uint32_t mask, float s2, const float* q) {
        const int lane = threadIdx.x & 31, key = lane & 15, half = lane >> 4;
        constexpr int ROW = DHP * 4;
        float z[HB] = {};
#pragma unroll
        for (int c = 0; c < DHP / 8; c++) {
            const int at = half * (DHP / 8) + c;
            const float4 k = *reinterpret_cast<const float4*>(stage + key * ROW + ((at ^ (key & 7)) << 4));
#pragma unroll
            for (int g = 0; g < HB; g++) {
                const float4 x = *reinterpret_cast<const float4*>(q + g * DHP + at * 4);
                z[g] = fmaf(x.x, k.x, z[g]);
                z[g] = fmaf(x.y, k.y, z[g]);
                z[g] = fmaf(x.z, k.z, z[g]);
                z[g] = fmaf(x.w, k.w, z[g]);
            }
        }
        float p[HB];
#pragma unroll
        for (int g = 0; g < HB; g++) {
            z[g] += __shfl_xor_sync(0xffffffffu, z[g], 16);
            z[g] = mask >> key & 1 ? z[g] * s2 : -INFINITY;
            float top = z[g];
#pragma unroll
            for (int x = 1; x < 16; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
            top = fmaxf(top, m[g]);
            const float safe = top == -INFINITY ? 0.f : top, turn = exp2f(m[g] - safe);
            p[g] = exp2f(z[g] - safe);
            m[g] = top;
            l[g] = fmaf(l[g], turn, p[g]);
#pragma unroll
            for (int e = 0; e < 4; e++) o[g][e] *= turn;
        }
        const int col = lane % COLS, first = lane / COLS * (kKeys / SHARE);
#pragma unroll
        for (int j = 0; j < kKeys / SHARE; j++) {
            const int row = first + j;
            const float4 v =
                *reinterpret_cast<const float4*>(stage + kKeys * ROW + row * ROW + ((col ^ (row & 7)) << 4));
#pragma unroll
            for (int g = 0; g < HB; g++) {
                const float w = __shfl_sync(0xffffffffu, p[g], row);
                o[g][0] = fmaf(w, v.x, o[g][0]);
                o[g][1] = fmaf(w, v.y, o[g][1]);
                o[g][2] = fmaf(w, v.z, o[g][2]);
                o[g][3] = fmaf(w, v.w, o[g][3]);
            }
        }
    }
    __device__ __forceinline__ void leave(float* to, int) {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int g = 0; g < HB; g++) {
            float sum = l[g];
#pragma unroll
            for (int x = 1; x < 16; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
            if (lane == 0) to[g] = m[g], to[4 + g] = sum;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (SHARE == 2) o[g][e] += __shfl_xor_sync(0xffffffffu, o[g][e], 16);
                if (lane < COLS) to[8 + g * DHP + lane * 4 + e] = o[g][e];
            }
        }
    }
};

template <typename T, int DHP, int HB>
__global__ void __launch_bounds__(kThreads, Ring<T, DHP>::PER_SM) paged_ring_kernel(const __grid_constant__ PagedArgs a) {
    using R = Ring<T, DHP>;
    constexpr int ROUNDS = HB > R::MEET ? HB / R::MEET : 1, MEET = HB < R::MEET ? HB : R::MEET;
    extern __shared__ __align__(128) uint8_t smem[];
    float* meet = reinterpret_cast<float*>(smem + kWarps * R::STAGES * R::STAGE);
    uint32_t* masks = reinterpret_cast<uint32_t*>(meet + kWarps * R::MEET * (DHP + 2));
    int* pre = reinterpret_cast<int*>(masks + kWarps * R::STAGES);
    const PagedDesc& d = a.d;
    const int t = threadIdx.x, warp = t >> 5;
    float* mine = meet + warp * R::MEET * (DHP + 2);
    float* queries = reinterpret_cast<float*>(pre + ((d.B + 4) & ~3)) + warp * HB * DHP;  // (fp32)
    uint8_t* ring = smem + warp * R::STAGES * R::STAGE;
    uint32_t* mask = masks + warp * R::STAGES;
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
    if (begin >= end) return;

    Cursor c;  // of the tile to fetch
    c.b = 0;
    for (int step = 1 << 13; step; step >>= 1)
        if (c.b + step < d.B && (long long)pre[c.b + step] * Hc <= begin) c.b += step;
    c.tiles = pre[c.b + 1] - pre[c.b];
    c.hc = (int)((begin - (long long)pre[c.b] * Hc) / c.tiles);
    c.i = (int)(begin - (long long)pre[c.b] * Hc - (long long)c.hc * c.tiles);
    c.s = seen_of(d, c.b);
    int b = c.b, hc = c.hc, i = c.i, tiles = c.tiles;  // of the tile to add
    long long ahead = begin;
    look_up(a, c, true);
    auto fetch_next = [&](int slot) {
        if (ahead < end) {
            fetch<T, DHP>(a, c, ring + slot * R::STAGE, mask + slot);
            ahead++;
            if (++c.i == c.tiles) {
                c.i = 0;
                if (++c.hc == Hc) {
                    c.hc = 0;
                    if (++c.b < d.B) {
                        c.tiles = pre[c.b + 1] - pre[c.b];
                        c.s = seen_of(d, c.b);
                    }
                }
            }
            look_up(a, c, ahead < end);  // a tile before it is wanted
        }
        commit();
    };
    for (int s = 0; s < R::STAGES - 1; s++) fetch_next(s);

    State<T, DHP, HB> state;
    int slot = 0;
    for (long long at = begin; at < end;) {
        const int hk = hc / a.chunks, g0 = (hc - hk * a.chunks) * HB, h0 = hk * a.group + g0;
        const int heads = min(HB, a.group - g0);
        const int i1 = (int)min((long long)tiles, i + (end - at));
        const bool whole = i == 0 && i1 == tiles;
        float* part = a.part + ((long long)blockIdx.x * 2 + (at == begin ? 0 : 1)) * (HB * (DHP + 2));
        at += i1 - i;
        state.start(d, b, h0, heads, queries);
        for (; i < i1; i++) {
            wait_but<R::STAGES - 2>();
            __syncwarp();  // every lane's pieces are there, and the slot before has been read
            fetch_next(slot == 0 ? R::STAGES - 1 : slot - 1);
            if constexpr (std::is_same<T, float>::value) state.add(ring + slot * R::STAGE, mask[slot], s2, queries);
            else state.add(ptx::smem_u32(ring + slot * R::STAGE), mask[slot], s2, nullptr);
            slot = slot + 1 == R::STAGES ? 0 : slot + 1;
        }
        // the warps meet, four heads at a time
        for (int round = 0; round < ROUNDS; round++) {
            __syncthreads();
            state.leave(mine, round);
            __syncthreads();
            for (int e = t; e < MEET * DHP; e += kThreads) {
                const int g = e / DHP, col = e % DHP, head = round * MEET + g;
                float top = -INFINITY, sum = 0.f, val = 0.f;
#pragma unroll
                for (int w = 0; w < kWarps; w++) top = fmaxf(top, meet[w * R::MEET * (DHP + 2) + g]);
                const float safe = top == -INFINITY ? 0.f : top;
#pragma unroll
                for (int w = 0; w < kWarps; w++) {
                    const float* x = meet + w * R::MEET * (DHP + 2);
                    const float f = exp2f(x[g] - safe);
                    sum = fmaf(x[4 + g], f, sum);
                    val = fmaf(x[8 + g * DHP + col], f, val);
                }
                if (head >= heads) continue;
                if (whole) {
                    put<T>(d, b, h0 + head, col, top, sum, val);
                } else {
                    part[2 * HB + head * DHP + col] = val;
                    if (col == 0) part[head] = top, part[HB + head] = sum;
                }
            }
        }
        if (i == tiles) {
            i = 0;
            if (++hc == Hc) {
                hc = 0;
                if (++b < d.B) tiles = pre[b + 1] - pre[b];
            }
        }
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

// Query heads that share what a block reads: as the kernels are made.
int heads_a_block(int group, bool tensor) { return tensor ? (group <= 8 ? 8 : 16) : group == 1 ? 1 : 4; }
int padded(int dh) { return dh <= 64 ? 64 : 128; }
size_t round16(size_t n) { return (n + 15) / 16 * 16; }
size_t plan_bytes(int B) { return round16((size_t)(B + 2) * sizeof(int)); }

bool vectors(const void* p, long long a, long long b, long long c, int size) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && a * size % 16 == 0 && b * size % 16 == 0 && c * size % 16 == 0;
}

}  // namespace

size_t attention_paged_workspace(int B, int Hq, int Hkv, int dh) {
    if (B <= 0 || Hkv <= 0 || Hq < Hkv || Hq % Hkv || dh <= 0 || dh > kAttnMaxHead) return 0;
    return plan_bytes(B) + (size_t)num_sms() * kPerSm * 2 * heads_a_block(Hq / Hkv, true) * (padded(dh) + 2) * sizeof(float);
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
        a.chunks = (a.group + HB - 1) / HB;
        if constexpr (decltype(aligned)::value) {
            using R = Ring<T, DHP>;
            auto f = paged_ring_kernel<T, DHP, HB>;
            const size_t queries = std::is_same<T, float>::value ? (size_t)kWarps * HB * DHP * sizeof(float) : 0;
            const size_t bytes = R::BYTES + (size_t)((d.B + 4) & ~3) * sizeof(int) + queries;
            if (cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != cudaSuccess) return -5;
            f<<<num_sms() * R::PER_SM, kThreads, bytes, st>>>(a);
        } else {
            paged_kernel<T, DHP, HB><<<num_sms() * kPerSm, kThreads, (d.B + 1) * sizeof(int), st>>>(a);
        }
        if (cudaGetLastError() != cudaSuccess) return -5;
        // the second kernel is launched while the first runs, and waits for it
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(d.B * d.Hkv * a.chunks), HB < a.group ? HB : a.group);
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
    auto by_heads = [&](auto zero, auto wide) {
        const bool tensor = vec && d.dtype == kBF16;
        switch (heads_a_block(a.group, tensor)) {
            case 1:
                if constexpr (std::is_same<decltype(zero), float>::value)
                    if (vec) return go(zero, wide, integral_constant<int, 1>(), std::true_type());
                return go(zero, wide, integral_constant<int, 1>(), std::false_type());
            case 4:
                if constexpr (std::is_same<decltype(zero), float>::value)
                    if (vec) return go(zero, wide, integral_constant<int, 4>(), std::true_type());
                return go(zero, wide, integral_constant<int, 4>(), std::false_type());
            default:
                if constexpr (std::is_same<decltype(zero), __nv_bfloat16>::value)
                    return a.group <= 8 ? go(zero, wide, integral_constant<int, 8>(), std::true_type())
                                        : go(zero, wide, integral_constant<int, 16>(), std::true_type());
                return -1;
        }
    };
    if (d.dtype == kBF16)
        return d.dh <= 64 ? by_heads(__nv_bfloat16(), integral_constant<int, 64>()) : by_heads(__nv_bfloat16(), integral_constant<int, 128>());
    return d.dh <= 64 ? by_heads(0.f, integral_constant<int, 64>()) : by_heads(0.f, integral_constant<int, 128>());
}

}  // namespace nsb
