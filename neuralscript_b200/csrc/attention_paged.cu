// Attention of one new token a sequence over a paged cache:
//   out[b, h] = sum over visible j of p_j v_j,  p = softmax(scale * q[b, h] . k_j),
// j visible where j < len and (no window, or j >= len - window, or j < sinks).
//
// Memory-bound: every visible key and value is read once for up to 16 query heads
// that share it in bf16, and for up to 4 in fp32 (a warp's registers hold no more;
// larger groups are cut into shares that each read it). One pass with the running
// maximum and sum of the softmax.
//
// Work is cut without regard to where sequences end: the visible keys of every
// (sequence, key head), counted in units of 16, stand in one line, and every
// warp takes the same number of neighbouring units of it. (A cut into equal
// parts a sequence leaves the blocks of short ones idle: the lengths of a
// batch differ by a factor of ten and more.) The lengths are on the device,
// so each block sums them up itself. A warp writes what it covers whole; of a
// head that others share it leaves maximum, sum and weighted values in the
// workspace (a block all of whose warps are in one head leaves one for all),
// and a second kernel joins those in the order of the keys. Nothing depends
// on timing.
//
// Bound by HBM while it streams; the sum of lengths before it takes some 5 us,
// the join behind it 2 to 9. 64 sequences of up to 4096 keys, 24 heads on 4 of
// 128 columns, bf16: 46.9 us, 4.5 TB/s; two of 120000, 16 heads on 2: 41.9 us,
// 4.8 TB/s; fp32, 96 behind a window of 1024, 8 heads of 64: 62.4 us, 5.7 TB/s;
// one sequence of 900 keys, 8 heads of 64: 9.7 us, all of it latency. What the
// forms cost that it suits less, 64 sequences of up to 4096 keys on 4 key heads:
// fp32 of 64 columns, 4 query heads a key head 56 us (3.8 TB/s), 8 105, 16 196;
// fp32 of 128 columns, whose ring leaves room for one block an SM, one query head
// 84 us (5.0 TB/s), 6 223; bf16 of 128, 16 query heads 113, 24 188. Every block
// holds a number for each sequence and sums all lengths up, and shares are cut for
// as many blocks as a small batch's SMs hold: 512 sequences of up to 2048 keys,
// 24 heads on 4 of 128, bf16, 182 us (5.0 TB/s), 1024 of up to 1024 251 us (3.5),
// 4096 of up to 256 387 us (2.3).
#include <cuda_bf16.h>
#include <math.h>

#include <type_traits>

#include "attention_cache.h"
#include "gemm.h"
#include "ptx.cuh"
#include "shared_memory.h"

namespace nsb {

namespace {

constexpr int kKeys = 16;        // a unit
constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kPerSm = 3;        // most blocks an SM that the grid is made for (fewer fit beside some 700 sequences' sums)
constexpr long long kMaxKeys = (1LL << 31) - kKeys;  // of a sequence: whole units of them are counted in 32 bits
constexpr int kMinUnits = 2;     // least units a warp: below, joining costs more than a warp saves
constexpr int kSlots = 2 * kWarps + 1;  // parts that a block may leave: two a warp, or one
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct PagedArgs {
    PagedDesc d;
    int group;   // query heads that share a key head
    int chunks;  // shares of a group
    int blocks;
    bool same;   // keys and values have the same strides
    int shift;   // log2 of a page's places, -1: no power of two
    int* plan;   // [0]: units a warp, [1 + b]: units before sequence b
    float* part; // [blocks][kSlots] maxima, sums [HB] and values [HB][DHP]
};

// Visible keys of a sequence, numbered 0 .. n - 1: the first `front` are the
// sequence's first, the others lie side by side from `back` on.
struct Seen {
    int n, front, back;
};
__device__ __forceinline__ Seen seen_of(const PagedDesc& d, int b) {
    int len = d.lens[b];
    const long long room = min((long long)d.width * d.page, kMaxKeys);
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
__device__ __forceinline__ int units_of(int n) { return n > 0 ? (n + kKeys - 1) / kKeys : 1; }

// pre[b] = units of the sequences before b, of one key head (pre: B + 1 ints).
__device__ __forceinline__ void sum_up(const PagedDesc& d, int* pre) {
    __shared__ int s_warp[kThreads / 32];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    int carry = 0;
    if (t == 0) pre[0] = 0;
    for (int b0 = 0; b0 < d.B; b0 += kThreads) {
        int v = b0 + t < d.B ? units_of(seen_of(d, b0 + t).n) : 0;
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

// Units a warp, and where the line's unit `at` is: in sequence b, share hc of
// its heads, unit i of `units`.
__device__ __forceinline__ long long share(long long all, int warps) {
    const long long each = all < 0x7fffffff - warps ? ((int)all + warps - 1) / warps : (all + warps - 1) / warps;
    return max((long long)kMinUnits, each);
}
struct Place {
    int b, hc, i, units;
};
__device__ __forceinline__ Place locate(const int* pre, int B, int Hc, long long at) {
    Place p;
    p.b = 0;
    for (int step = 1 << (31 - __clz(B)); step; step >>= 1)
        if (p.b + step < B && (long long)pre[p.b + step] * Hc <= at) p.b += step;
    p.units = pre[p.b + 1] - pre[p.b];
    const long long in = at - (long long)pre[p.b] * Hc;
    p.hc = in < 0x7fffffff ? (int)in / p.units : (int)(in / p.units);
    p.i = (int)(in - (long long)p.hc * p.units);
    return p;
}

__device__ __forceinline__ void put_lse(const PagedDesc& d, int b, int h, float m, float l) {
    if (d.lse) d.lse[(long long)b * d.Hq + h] = l > 0.f ? (m + log2f(l)) * kLn2 : l == 0.f ? -INFINITY : l;
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
    if (c == 0) put_lse(d, b, h, m, l);
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
// fourth key of the warp's; the four meet where its keys of a head end. HB
// query heads share what is read.
template <typename T, int DHP, int HB>
__global__ void __launch_bounds__(kThreads) paged_kernel(const __grid_constant__ PagedArgs a) {
    constexpr int DIMS = DHP / 8;
    extern __shared__ int pre[];
    const PagedDesc& d = a.d;
    const int t = threadIdx.x, sub = t & 7, warp = t >> 5;
    cudaTriggerProgrammaticLaunchCompletion();  // the join's blocks take the places of those that end
    sum_up(d, pre);
    __syncthreads();
    const int Hc = d.Hkv * a.chunks;
    const long long W = (long long)pre[d.B] * Hc, per = share(W, a.blocks * kWarps);
    if (blockIdx.x == 0) {
        for (int b = t; b <= d.B; b += kThreads) a.plan[1 + b] = pre[b];
        if (t == 0) a.plan[0] = (int)per;
    }
    const long long begin = ((long long)blockIdx.x * kWarps + warp) * per, end = min(W, begin + per);
    const float s2 = d.scale * kLog2e;

    for (long long at = begin; at < end;) {
        const Place w = locate(pre, d.B, Hc, at);
        const int i1 = (int)min((long long)w.units, w.i + (end - at));
        const int hk = w.hc / a.chunks, g0 = (w.hc - hk * a.chunks) * HB, h0 = hk * a.group + g0;
        const int heads = min(HB, a.group - g0);
        const Seen s = seen_of(d, w.b);

        float q[HB][DIMS], o[HB][DIMS], m[HB], l[HB];
#pragma unroll
        for (int g = 0; g < HB; g++) {
            if (g < heads) load_dims<T, DIMS>(q[g], (const T*)d.q.p + w.b * d.q.row + (h0 + g) * d.q.head, sub, d.dh);
            m[g] = -INFINITY;
            l[g] = 0.f;
#pragma unroll
            for (int j = 0; j < DIMS; j++) {
                if (g >= heads) q[g][j] = 0.f;
                o[g][j] = 0.f;
            }
        }
        const int last = min(s.n, i1 * kKeys);
        for (int x = w.i * kKeys + (t >> 3 & 3); x < last; x += 4) {
            const int key = x < s.front ? x : x - s.front + s.back;
            const int pi = key / d.page;
            const int page = d.table[w.b * d.ld_table + pi];
            if (page < 0 || page >= d.pages) {  // no such page: its keys are left out
                atomicCAS(d.err, 0, kErrBadIndex);
                continue;
            }
            float k[DIMS], v[DIMS];
            load_dims<T, DIMS>(k, (const T*)d.kc.p + page * d.kc.page + (key - pi * d.page) * d.kc.slot + hk * d.kc.head, sub,
                               d.dh);
            load_dims<T, DIMS>(v, (const T*)d.vc.p + page * d.vc.page + (key - pi * d.page) * d.vc.slot + hk * d.vc.head, sub,
                               d.dh);
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
        __syncwarp();
        const bool whole = w.i == 0 && i1 == w.units;
        float* part = a.part + ((long long)blockIdx.x * kSlots + 2 * warp + (at == begin ? 0 : 1)) * (HB * (DHP + 2));
#pragma unroll
        for (int g = 0; g < HB; g++) {
            float top = m[g];
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
            const float f = exp2f(m[g] - (top == -INFINITY ? 0.f : top));
            float sum = l[g] * f;
            sum += __shfl_xor_sync(0xffffffffu, sum, 8);
            sum += __shfl_xor_sync(0xffffffffu, sum, 16);
#pragma unroll
            for (int j = 0; j < DIMS; j++) {
                float val = o[g][j] * f;
                val += __shfl_xor_sync(0xffffffffu, val, 8);
                val += __shfl_xor_sync(0xffffffffu, val, 16);
                const int col = j * 8 + sub;
                if (g >= heads || (t & 31) >= 8) continue;
                if (whole) put<T>(d, w.b, h0 + g, col, top, sum, val);
                else part[2 * HB + g * DHP + col] = val;
            }
            if (!whole && g < heads && (t & 31) == 0) part[g] = top, part[HB + g] = sum;
        }
        at += i1 - w.i;
    }
}

// ---------------------------------------------------------------------------
// The same from 16-byte pieces. Each warp has a ring of its own in shared
// memory that cp.async fills some units ahead, over the borders of heads and
// sequences too; no barrier of the block stands between two units. Pieces of a
// row are exchanged by the row's lowest three bits, so that neither reading rows
// nor columns meets a bank twice. What is behind a sequence's end, or on no
// page, arrives as zeros.
//
// bf16: on the tensor cores (m16n8k16: a unit is too small for the large
// products, and the bytes take the time), the keys as the product's rows and 8
// query heads its columns, S^T = K Q^T; the weights turn into the second
// product's columns by a transpose in registers, O^T += V^T P^T. A weight goes in
// as two bf16, its first eight digits and the next (2^-16 of it is lost; its sum
// is taken before): the tensor pipe has room beside the bytes. 64 sequences
// take 46.9 us for 45.7 with a rounded weight, and the result differs from one
// of fp32 weights by 8e-5 for 1.7e-3. Groups of fewer heads leave columns
// empty, which costs nothing.
// fp32: on the fp32 units, two lanes a key for the scores, and four columns a
// lane for the values.
//
// One unit ahead is enough (a unit's arithmetic takes longer than memory's
// answer), and twelve warps an SM hide each other's latencies: with eight and
// two units ahead 64 sequences took 60 us in place of 48.
// ---------------------------------------------------------------------------
template <typename T, int DHP, int HB>
struct Ring {
    static constexpr int ROW = DHP * (int)sizeof(T);
    static constexpr int STAGE = 2 * kKeys * ROW;  // keys, values
    static constexpr int STAGES = ROW == 128 ? 4 : 2;
    static constexpr int MEET = 4;  // heads whose results meet at a time
    static constexpr int BYTES = kWarps * STAGES * STAGE + kWarps * MEET * (DHP + 2) * 4 + kWarps * STAGES * 4;
    static constexpr int PER_SM = ROW == 512 ? 1 : HB * DHP > 1024 ? 2 : 3;  // by shared memory, and registers
};

// Of a unit to fetch, the page (from the table; -1: no such key) and the place
// of this lane's row (lanes 0 .. 15 the keys', 16 .. 31 the values').
struct Row {
    int page, place, hk;
    bool real;
};
// Where a warp's next unit is.
struct Cursor {
    Place w;
    Seen s;
    __device__ __forceinline__ void next(const PagedArgs& a, const int* pre, int Hc) {
        if (++w.i < w.units) return;
        w.i = 0;
        if (++w.hc < Hc) return;
        w.hc = 0;
        if (++w.b < a.d.B) {
            w.units = pre[w.b + 1] - pre[w.b];
            s = seen_of(a.d, w.b);
        }
    }
    __device__ __forceinline__ Row look_up(const PagedArgs& a) const {
        Row r{-1, 0, w.hc / a.chunks, false};
        const int x = w.i * kKeys + (threadIdx.x & (kKeys - 1));
        if (x < s.n) {
            const int key = x < s.front ? x : x - s.front + s.back;
            const int pi = a.shift >= 0 ? key >> a.shift : key / a.d.page;
            r.place = key - pi * a.d.page;
            r.page = a.d.table[w.b * a.d.ld_table + pi];
            r.real = true;
        }
        return r;
    }
};

// 16 bytes, zeros where `on` does not hold.
// The cache is read once: it leaves L2 first, so that what is read again
// (parts, tables, and the kernels' own code) stays.
__device__ __forceinline__ uint64_t once() {
    uint64_t p;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
    return p;
}
__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool on, uint64_t policy) {
    asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(to), "l"(from), "r"(on ? 16 : 0),
                 "l"(policy)
                 : "memory");
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Offsets are counted in pieces of 16 bytes: 32 bits reach 64 GB.
constexpr uint32_t kNone = 0xffffffffu;

template <typename T, int DHP>
__device__ __forceinline__ void fetch(const PagedArgs& a, Row c, uint32_t stage, uint32_t* mask, uint64_t policy) {
    constexpr int ROW = DHP * (int)sizeof(T), PIECES = ROW / 16, ROWS = 32 / PIECES;
    const int lane = threadIdx.x & 31;
    const bool there_is = c.page >= 0 && c.page < a.d.pages;
    const uint32_t there = __ballot_sync(0xffffffffu, there_is);
    if (c.real && !there_is) atomicCAS(a.d.err, 0, kErrBadIndex);  // no such page: its keys are left out
    if (lane == 0) *mask = there;
    const int piece = lane % PIECES;
    const bool inside = piece * 16 < a.d.dh * (int)sizeof(T);
    const char* nothing = (const char*)a.d.q.p;  // an address for copies of no bytes
    const char *k = (const char*)a.d.kc.p + piece * 16, *v = (const char*)a.d.vc.p + piece * 16;
    if (a.same) {  // keys and values lie alike
        const uint32_t offset =
            there_is ? (uint32_t)((c.page * a.d.kc.page + c.place * a.d.kc.slot + c.hk * a.d.kc.head) / (16 / (int)sizeof(T))) : kNone;
#pragma unroll
        for (int r0 = 0; r0 < kKeys; r0 += ROWS) {
            const int row = r0 + lane / PIECES;
            const uint32_t at = __shfl_sync(0xffffffffu, offset, row);
            const bool on = at != kNone && inside;
            const uint32_t to = stage + row * ROW + ((piece ^ (row & 7)) << 4);
            copy16(to, on ? k + (size_t)at * 16 : nothing, on, policy);
            copy16(to + kKeys * ROW, on ? v + (size_t)at * 16 : nothing, on, policy);
        }
        return;
    }
    const Pages& mine = lane < kKeys ? a.d.kc : a.d.vc;
    const uint32_t offset =
        there_is ? (uint32_t)((c.page * mine.page + c.place * mine.slot + c.hk * mine.head) / (16 / (int)sizeof(T))) : kNone;
#pragma unroll
    for (int r0 = 0; r0 < 2 * kKeys; r0 += ROWS) {  // rows of the keys, then of the values
        const int row = r0 + lane / PIECES;
        const uint32_t at = __shfl_sync(0xffffffffu, offset, row);
        const bool on = at != kNone && inside;
        copy16(stage + row * ROW + ((piece ^ (row & 7)) << 4), on ? (r0 < kKeys ? k : v) + (size_t)at * 16 : nothing, on,
               policy);
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

// What a weight has behind its first eight digits (its upper half, a bf16). Of a
// weight above 0 it is above 0 too, and never below: both times an infinite value
// are that infinity.
__device__ __forceinline__ float behind(float w) {
    return fmaxf(w - __uint_as_float(__float_as_uint(w) & 0xffff0000u), fminf(w, 0x1p-126f));
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
        uint32_t p[NT][2], rest[NT][2];
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
                turn[n][e] = ex2(m[n][e] - safe);
                rise |= top != m[n][e];
                m[n][e] = top;
                s[n][e] = ex2(s[n][e] - safe);
                s[n][2 + e] = ex2(s[n][2 + e] - safe);
                l[n][e] = fmaf(l[n][e], turn[n][e], s[n][e] + s[n][2 + e]);
            }
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const __nv_bfloat162 r = __floats2bfloat162_rn(behind(s[n][2 * e]), behind(s[n][2 * e + 1]));
                p[n][e] = turned(__byte_perm(__float_as_uint(s[n][2 * e]), __float_as_uint(s[n][2 * e + 1]), 0x7632));
                rest[n][e] = turned(*reinterpret_cast<const uint32_t*>(&r));
            }
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
            for (int n = 0; n < NT; n++) {
                mma16816(o[k][n], a, p[n][0], p[n][1]);
                mma16816(o[k][n], a, rest[n][0], rest[n][1]);
            }
        }
    }
    __device__ __forceinline__ float total(int n, int e) const {
        float sum = l[n][e];
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        return sum + __shfl_xor_sync(0xffffffffu, sum, 16);
    }
    // the heads' outputs
    __device__ __forceinline__ void finish(const PagedDesc& d, int b, int h0, int heads) const {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int n = 0; n < NT; n++) {
            float mul[2];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const float sum = total(n, e);
                mul[e] = sum == 0.f ? 0.f : 1.f / sum;
                const int h = n * 8 + 2 * (lane & 3) + e;
                if (lane < 4 && h < heads) put_lse(d, b, h0 + h, m[n][e], sum);
            }
            const int h = n * 8 + (lane >> 2);  // behind the transpose
            __nv_bfloat16* to = (__nv_bfloat16*)d.out.p + b * d.out.row + (h0 + h) * d.out.head + 2 * (lane & 3);
            const bool pairs = (reinterpret_cast<uintptr_t>(to) & 3) == 0;
#pragma unroll
            for (int k = 0; k < KS; k++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const __nv_bfloat162 v = __floats2bfloat162_rn(mul[0] == 0.f ? 0.f : o[k][n][2 * e] * mul[0],  // (0 times an infinity)
                                                                   mul[1] == 0.f ? 0.f : o[k][n][2 * e + 1] * mul[1]);
                    const uint32_t w = turned(*reinterpret_cast<const uint32_t*>(&v));
                    const int c = 16 * k + 8 * e;
                    if (h >= heads || c + 2 * (lane & 3) >= d.dh) continue;
                    if (pairs) {
                        *reinterpret_cast<uint32_t*>(to + c) = w;
                    } else {
                        const __nv_bfloat162 x = *reinterpret_cast<const __nv_bfloat162*>(&w);
                        to[c] = x.x;
                        to[c + 1] = x.y;
                    }
                }
        }
    }
    // what others join
    __device__ __forceinline__ void part(float* to) const {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const float sum = total(n, e);
                const int h = n * 8 + 2 * (lane & 3) + e;
                if (lane < 4) to[h] = m[n][e], to[HB + h] = sum;
#pragma unroll
                for (int k = 0; k < KS; k++) {
                    to[2 * HB + h * DHP + 16 * k + (lane >> 2)] = o[k][n][e];
                    to[2 * HB + h * DHP + 16 * k + (lane >> 2) + 8] = o[k][n][2 + e];
                }
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
                const float sum = total(n, e);
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
            const float safe = top == -INFINITY ? 0.f : top, turn = ex2(m[g] - safe);
            p[g] = ex2(z[g] - safe);
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
    template <typename F>
    __device__ __forceinline__ void each_head(F use) const {  // use(head, sum, value e of this lane's columns ..)
#pragma unroll
        for (int g = 0; g < HB; g++) {
            float sum = l[g], v[4];
#pragma unroll
            for (int x = 1; x < 16; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = SHARE == 2 ? o[g][e] + __shfl_xor_sync(0xffffffffu, o[g][e], 16) : o[g][e];
            use(g, sum, v);
        }
    }
    __device__ __forceinline__ void finish(const PagedDesc& d, int b, int h0, int heads) const {
        const int lane = threadIdx.x & 31;
        each_head([&](int g, float sum, const float* v) {
            if (g >= heads || lane >= COLS) return;
#pragma unroll
            for (int e = 0; e < 4; e++) put<float>(d, b, h0 + g, lane * 4 + e, m[g], sum, v[e]);
        });
    }
    __device__ __forceinline__ void part(float* to) const {
        const int lane = threadIdx.x & 31;
        each_head([&](int g, float sum, const float* v) {
            if (lane == 0) to[g] = m[g], to[HB + g] = sum;
            if (lane >= COLS) return;
#pragma unroll
            for (int e = 0; e < 4; e++) to[2 * HB + g * DHP + lane * 4 + e] = v[e];
        });
    }
    __device__ __forceinline__ void leave(float* to, int) const {
        const int lane = threadIdx.x & 31;
        each_head([&](int g, float sum, const float* v) {
            if (lane == 0) to[g] = m[g], to[4 + g] = sum;
            if (lane >= COLS) return;
#pragma unroll
            for (int e = 0; e < 4; e++) to[8 + g * DHP + lane * 4 + e] = v[e];
        });
    }
};

template <typename T, int DHP, int HB>
__global__ void __launch_bounds__(kThreads, Ring<T, DHP, HB>::PER_SM) paged_ring_kernel(const __grid_constant__ PagedArgs a) {
    using R = Ring<T, DHP, HB>;
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
    const uint32_t ring_at = ptx::smem_u32(ring);
    uint32_t* mask = masks + warp * R::STAGES;
    cudaTriggerProgrammaticLaunchCompletion();  // the join's blocks take the places of those that end
    sum_up(d, pre);
    __syncthreads();
    const int Hc = d.Hkv * a.chunks;
    const long long W = (long long)pre[d.B] * Hc, per = share(W, a.blocks * kWarps);
    if (blockIdx.x == 0) {
        for (int b = t; b <= d.B; b += kThreads) a.plan[1 + b] = pre[b];
        if (t == 0) a.plan[0] = (int)per;
    }
    const long long first = (long long)blockIdx.x * kWarps * per;
    if (first >= W) return;
    const long long begin = min(W, first + warp * per), end = min(W, begin + per);
    const float s2 = d.scale * kLog2e;
    // whether all of the block's units are in one head's line
    const Place f = locate(pre, d.B, Hc, first);
    const bool together = f.i + (min(W, first + kWarps * per) - first) <= f.units;

    Cursor c;  // of the next unit to look up
    c.w = f;
    if (f.i + (begin - first) < f.units) c.w.i += (int)(begin - first);
    else if (begin < W) c.w = locate(pre, d.B, Hc, begin);
    c.s = seen_of(d, c.w.b);
    Place w = c.w;  // of the next unit to add
    const uint64_t policy = once();
    Row ahead[R::STAGES - 1];
    long long looked = begin, fetched = begin;
#pragma unroll
    for (int s = 0; s < R::STAGES - 1; s++)
        if (looked < end) {
            ahead[s] = c.look_up(a);
            c.next(a, pre, Hc);
            looked++;
        }
#pragma unroll
    for (int s = 0; s < R::STAGES - 1; s++) {
        if (fetched < end) {
            fetch<T, DHP>(a, ahead[s], ring_at + s * R::STAGE, mask + s, policy);
            fetched++;
        }
        commit();
    }
    Row row = {};
    if (looked < end) row = c.look_up(a);

    State<T, DHP, HB> state;
    int slot = 0;
    for (long long at = begin; at < end;) {
        const int hk = w.hc / a.chunks, g0 = (w.hc - hk * a.chunks) * HB, h0 = hk * a.group + g0;
        const int heads = min(HB, a.group - g0);
        const int i1 = (int)min((long long)w.units, w.i + (end - at));
        const bool whole = w.i == 0 && i1 == w.units;
        const int which = 2 * warp + (at == begin ? 0 : 1);
        at += i1 - w.i;
        state.start(d, w.b, h0, heads, queries);
        for (; w.i < i1; w.i++) {
            wait_but<R::STAGES - 2>();
            __syncwarp();  // every lane's pieces are there, and the slot before has been read
            if (looked < end) {
                const int to = slot == 0 ? R::STAGES - 1 : slot - 1;
                fetch<T, DHP>(a, row, ring_at + to * R::STAGE, mask + to, policy);
                c.next(a, pre, Hc);
                if (++looked < end) row = c.look_up(a);  // a unit before it is wanted
            }
            commit();
            if constexpr (std::is_same<T, float>::value) state.add(ring + slot * R::STAGE, mask[slot], s2, queries);
            else state.add(ring_at + slot * R::STAGE, mask[slot], s2, nullptr);
            slot = slot + 1 == R::STAGES ? 0 : slot + 1;
        }
        if (together) break;
        if (whole) state.finish(d, w.b, h0, heads);
        else state.part(a.part + ((long long)blockIdx.x * kSlots + which) * (HB * (DHP + 2)));
        if (w.i == w.units) {
            w.i = 0;
            if (++w.hc == Hc) {
                w.hc = 0;
                if (++w.b < d.B) w.units = pre[w.b + 1] - pre[w.b];
            }
        }
    }
    if (!together) return;
    // the warps meet, four heads at a time
    const int hk = f.hc / a.chunks, g0 = (f.hc - hk * a.chunks) * HB, h0 = hk * a.group + g0, heads = min(HB, a.group - g0);
    const bool whole = f.i == 0 && min(W, first + kWarps * per) - first == f.units;
    float* part = a.part + ((long long)blockIdx.x * kSlots + 2 * kWarps) * (HB * (DHP + 2));
    if (begin >= end) state.start(d, f.b, h0, 0, queries);  // nothing of it
    for (int round = 0; round < ROUNDS; round++) {
        if (round) __syncthreads();
        state.leave(mine, round);
        __syncthreads();
        for (int e = t; e < MEET * DHP; e += kThreads) {
            const int g = e / DHP, col = e % DHP, head = round * MEET + g;
            float top = -INFINITY, sum = 0.f, val = 0.f;
#pragma unroll
            for (int x = 0; x < kWarps; x++) top = fmaxf(top, meet[x * R::MEET * (DHP + 2) + g]);
            const float safe = top == -INFINITY ? 0.f : top;
#pragma unroll
            for (int x = 0; x < kWarps; x++) {
                const float* from = meet + x * R::MEET * (DHP + 2);
                const float share = exp2f(from[g] - safe);
                sum = fmaf(from[4 + g], share, sum);
                val = fmaf(from[8 + g * DHP + col], share, val);
            }
            if (head >= heads) continue;
            if (whole) {
                put<T>(d, f.b, h0 + head, col, top, sum, val);
            } else {
                part[2 * HB + head * DHP + col] = val;
                if (col == 0) part[head] = top, part[HB + head] = sum;
            }
        }
    }
}

// Joins what several warps left of one head. Parts are numbered through the
// blocks: one of a block that is in the head's line with all of its units
// (where the blocks meet, `together`), else its warps'. 256 parts at a time:
// a thread each for maxima and sums, which gives every part its weight, then
// eight warps add up every eighth part's values, whose loads wait for nothing.
// AHEAD: the first values are loaded while the weights are formed. That takes 76
// registers for 44, so it is for grids that leave SMs room anyway (two sequences
// of 120000 keys, 32 blocks: 44.2 to 42.4 us; 64 sequences, 1536 blocks: 46.2 to
// 48.1).
template <typename T, int DHP, int HB, bool AHEAD>
__global__ void __launch_bounds__(256) paged_join_kernel(const __grid_constant__ PagedArgs a, bool merges) {
    constexpr int C = DHP / 32;
    __shared__ float s_top[8], s_sum[8], s_w[256], s_o[8][DHP];
    __shared__ int s_at[256];
    const PagedDesc& d = a.d;
    cudaGridDependencySynchronize();
    const int Hc = d.Hkv * a.chunks;
    const int b = blockIdx.x / Hc, hc = blockIdx.x - b * Hc, g = blockIdx.y;
    const int hk = hc / a.chunks, g0 = (hc - hk * a.chunks) * HB;
    if (g0 + g >= a.group) return;
    const int before = a.plan[1 + b], units = a.plan[2 + b] - before;
    const long long per = a.plan[0], W = (long long)a.plan[1 + d.B] * Hc;
    const long long t0 = (long long)before * Hc + (long long)hc * units, t1 = t0 + units;
    const bool small = W < 0x7fffffff;  // (a division of 64 bits takes a hundred instructions)
    const long long w0 = small ? (int)t0 / (int)per : t0 / per, w1 = small ? (int)(t1 - 1) / (int)per : (t1 - 1) / per;
    if (w0 == w1) return;  // one warp had it all
    const long long block = per * kWarps;
    const int c0 = (int)(w0 / kWarps), c1 = (int)(w1 / kWarps);
    auto inside = [&](int c) { return merges && t0 <= c * block && min(W, (c + 1) * block) <= t1; };
    const bool in0 = inside(c0), in1 = inside(c1);
    if (c0 == c1 && in0) return;  // or one block
    // parts of the first block, of those between, and of the last
    const int n0 = in0 ? 1 : kWarps, each = merges ? 1 : kWarps, n1 = c0 == c1 ? n0 : n0 + (c1 - c0 - 1) * each;
    const int n = c0 == c1 ? n0 : n1 + (in1 ? 1 : kWarps);
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
    float m = -INFINITY, l = 0.f, o[C] = {};
    for (int x0 = 0; x0 < n; x0 += 256) {
        const int x = x0 + t;
        int at = -1;
        float mc = -INFINITY, lc = 0.f;
        if (x < n) {
            const int c = x < n0 ? c0 : x < n1 ? c0 + 1 + (x - n0) / each : c1;
            const int w = x < n0 ? (in0 ? -1 : x) : x < n1 ? (merges ? -1 : (x - n0) % kWarps) : in1 ? -1 : x - n1;
            const long long from = c * block + w * per;
            if (w < 0) at = c * kSlots + 2 * kWarps;
            else if (from < t1 && from + per > t0) at = c * kSlots + 2 * w + (from < t0 ? 1 : 0);  // else in another head
            if (at >= 0) {
                mc = a.part[(long long)at * (HB * (DHP + 2)) + g];
                lc = a.part[(long long)at * (HB * (DHP + 2)) + HB + g];
            }
        }
        s_at[t] = at;
        const float* values = a.part + 2 * HB + g * DHP + lane;
        float v[8][C];
        auto load = [&](int y0) {  // eight parts' at once
#pragma unroll
            for (int u = 0; u < 8; u++) {
                const int from = y0 + 8 * u < 256 ? s_at[y0 + 8 * u] : -1;
#pragma unroll
                for (int j = 0; j < C; j++) v[u][j] = from >= 0 ? values[(long long)from * (HB * (DHP + 2)) + 32 * j] : 0.f;
            }
        };
        if (AHEAD) {
            __syncthreads();
            load(warp);
        }
        float top = mc;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
        if (lane == 0) s_top[warp] = top;
        __syncthreads();
        top = m;
#pragma unroll
        for (int w = 0; w < 8; w++) top = fmaxf(top, s_top[w]);
        const float safe = top == -INFINITY ? 0.f : top, turn = exp2f(m - safe), share = exp2f(mc - safe);
        s_w[t] = share;
        float sum = lc * share;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
        if (lane == 0) s_sum[warp] = sum;
        __syncthreads();
        m = top;
        l *= turn;
#pragma unroll
        for (int w = 0; w < 8; w++) l += s_sum[w];
#pragma unroll
        for (int j = 0; j < C; j++) o[j] *= turn;
        for (int y0 = warp; y0 < min(256, n - x0); y0 += 64) {
            if (!AHEAD || y0 != warp) load(y0);
#pragma unroll
            for (int u = 0; u < 8; u++)
#pragma unroll
                for (int j = 0; j < C; j++) o[j] = fmaf(v[u][j], y0 + 8 * u < 256 ? s_w[y0 + 8 * u] : 0.f, o[j]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < C; j++) s_o[warp][lane + 32 * j] = o[j];
    __syncthreads();
    if (t < DHP) {
        float val = 0.f;
#pragma unroll
        for (int w = 0; w < 8; w++) val += s_o[w][t];
        put<T>(d, b, hk * a.group + g0 + g, t, m, l, val);
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
    return plan_bytes(B) + (size_t)num_sms() * kPerSm * kSlots * heads_a_block(Hq / Hkv, true) * (padded(dh) + 2) * sizeof(float);
}

int attention_paged_launches() { return 2; }

int attention_paged(const PagedDesc& d, cudaStream_t st) {
    if (d.B < 0 || d.Hkv <= 0 || d.Hq < d.Hkv || d.Hq % d.Hkv || d.dh <= 0 || d.dh > kAttnMaxHead ||
        (d.dtype != kF32 && d.dtype != kBF16))
        return -1;
    if (d.pages < 0 || d.page <= 0 || d.width < 0 || d.ld_table < d.width || d.window < 0 || d.sinks < 0 ||
        !(d.scale > 0.f) || !(d.scale < INFINITY))
        return -1;
    if (d.B > kPagedMaxBatch || (long long)d.B * d.Hq > 0x7fffffff) return -2;
    if (d.B == 0) return 0;
    // units are counted in 32 bits, those of one warp too
    const long long places = (long long)d.width * d.page, room = places < kMaxKeys ? places : kMaxKeys;
    const long long seen = d.window ? (long long)d.window + d.sinks : room;
    if ((room < seen ? room : seen) / kKeys * d.B >= (1LL << 31) - kPagedMaxBatch ||
        (room < seen ? room : seen) / kKeys * d.B * d.Hq >= 1LL << 39)
        return -2;
    if (!d.q.p || !d.out.p || !d.lens || (d.width && !d.table) || (d.pages && (!d.kc.p || !d.vc.p))) return -1;
    if (!d.workspace || reinterpret_cast<uintptr_t>(d.workspace) % 16 ||
        d.workspace_bytes < attention_paged_workspace(d.B, d.Hq, d.Hkv, d.dh))
        return -1;
    if (!d.err) return -5;
    PagedArgs a;
    a.d = d;
    a.group = d.Hq / d.Hkv;
    a.shift = -1;
    for (int i = 0; i < 31; i++)
        if (d.page == 1 << i) a.shift = i;
    a.plan = reinterpret_cast<int*>(d.workspace);
    a.part = reinterpret_cast<float*>(reinterpret_cast<char*>(d.workspace) + plan_bytes(d.B));
    const int size = d.dtype == kBF16 ? 2 : 4;
    a.same = d.kc.page == d.vc.page && d.kc.slot == d.vc.slot && d.kc.head == d.vc.head;
    auto near = [&](const Pages& x) {  // offsets in pieces of 16 bytes fit 32 bits
        return x.page >= 0 && x.slot >= 0 && x.head >= 0 &&
               ((double)x.page * d.pages + (double)x.slot * d.page + (double)x.head * d.Hkv) * size / 16 < 4294967000.0;
    };
    const bool vec = near(d.kc) && near(d.vc) && vectors(d.q.p, d.q.row, d.q.head, 0, size) && d.dh * size % 16 == 0 &&
                     vectors(d.kc.p, d.kc.page, d.kc.slot, d.kc.head, size) &&
                     vectors(d.vc.p, d.vc.page, d.vc.slot, d.vc.head, size);
    auto go = [&](auto zero, auto wide, auto many, auto aligned) {
        using T = decltype(zero);
        constexpr int DHP = decltype(wide)::value, HB = decltype(many)::value;
        a.chunks = (a.group + HB - 1) / HB;
        if constexpr (decltype(aligned)::value) {
            using R = Ring<T, DHP, HB>;
            auto f = paged_ring_kernel<T, DHP, HB>;
            const size_t queries = std::is_same<T, float>::value ? (size_t)kWarps * HB * DHP * sizeof(float) : 0;
            const size_t bytes = R::BYTES + (size_t)((d.B + 4) & ~3) * sizeof(int) + queries;
            static size_t most[kMaxDevices];
            if (!allow_shared(f, bytes, most)) return -5;
            a.blocks = num_sms() * R::PER_SM;
            f<<<a.blocks, kThreads, bytes, st>>>(a);
        } else {
            a.blocks = num_sms() * kPerSm;
            paged_kernel<T, DHP, HB><<<a.blocks, kThreads, (d.B + 1) * sizeof(int), st>>>(a);
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
        const bool few = (long long)cfg.gridDim.x * cfg.gridDim.y <= 2 * num_sms();
        return cudaLaunchKernelEx(&cfg, few ? paged_join_kernel<T, DHP, HB, true> : paged_join_kernel<T, DHP, HB, false>, a,
                                  (bool)decltype(aligned)::value) == cudaSuccess
                   ? 0
                   : -5;
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
