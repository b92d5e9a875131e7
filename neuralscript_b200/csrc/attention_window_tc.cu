// Attention with a window on the tensor cores (tcgen05, TMEM, TMA), bf16,
// heads of up to 128 columns (a multiple of 8; padded with zeros to 64 or
// 128 on the way in). Definitions in attention_window.cu.
//
// All waits are bounded: a role whose wait runs out tells the others of its
// block through a flag in shared memory and the host through the error word,
// and every role waits for its own copies and products before it leaves.
#include <cuda.h>
#include <cuda_bf16.h>
#include <math.h>

#include <mutex>

#include "attention_window.cuh"
#include "common.cuh"
#include "gemm.h"
#include "ptx.cuh"

namespace nsb {

namespace {

constexpr int kT = 128;                // rows of a tile
constexpr int kChunk = kT * 128;       // 128 rows x 64 columns of bf16
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Waits of one block. `lane` is one thread's; the other is a whole warp's,
// all of whose lanes go on or none.
struct Waits {
    volatile int* failed;  // shared memory
    int* err;
    __device__ __forceinline__ bool operator()(uint64_t* bar, uint32_t phase) const {
        return __all_sync(0xffffffffu, lane(bar, phase));
    }
    __device__ __forceinline__ bool lane(uint64_t* bar, uint32_t phase) const {
        if (ptx::mbar_try_wait(bar, phase & 1)) return true;
        const long long t0 = clock64();
        while (!ptx::mbar_try_wait(bar, phase & 1)) {
            if (*failed) return false;
            if (clock64() - t0 > ptx::kWaitCycles) {
                *failed = 1;
                atomicCAS(err, 0, kErrTimeoutAttn);
                return false;
            }
        }
        return true;
    }
};

// 128 rows of a head from row `row` on, 64 columns a chunk.
template <int DHP>
__device__ __forceinline__ void load_rows(uint8_t* to, const CUtensorMap* map, uint64_t* bar, int head, int row) {
    ptx::mbar_arrive_expect_tx(bar, DHP / 64 * kChunk);
#pragma unroll
    for (int c = 0; c < DHP / 64; c++) ptx::tma_load_3d(to + c * kChunk, map, bar, c * 64, head, row);
}

// Zeros in the rows of a tile from `from` on, by one warp: what stands there
// belongs to another sequence or to none, and 0 times an infinity is no 0.
template <int DHP>
__device__ __forceinline__ void zero_rows(uint8_t* tile, int from) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int c = 0; c < DHP / 64; c++)
        for (int at = from * 128 + lane * 16; at < kChunk; at += 512)
            *reinterpret_cast<uint4*>(tile + c * kChunk + at) = make_uint4(0, 0, 0, 0);
    ptx::fence_proxy_async();
    __syncwarp();
}

// D (+)= A B^T over the heads' columns, both K-major tiles.
template <int DHP>
__device__ __forceinline__ void mma_dot(uint32_t d, uint32_t a, uint32_t b) {
    constexpr uint32_t idesc = ptx::instr_desc(1, 0, 0, kT, kT);
#pragma unroll
    for (int s = 0; s < DHP / 16; s++) {
        const uint32_t at = (s >> 2) * kChunk + (s & 3) * 32;
        ptx::mma_bf16(d, ptx::smem_desc(a + at, 16, 1024, 2), ptx::smem_desc(b + at, 16, 1024, 2), idesc, s > 0);
    }
}

// 32 columns of an output row.
__device__ __forceinline__ void store32(__nv_bfloat16* to, const uint32_t* v, float mul, int cols) {
#pragma unroll
    for (int g = 0; g < 4; g++) {
        if (8 * g >= cols) break;
        uint4 pk;
        __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&pk);
#pragma unroll
        for (int e = 0; e < 4; e++)
            h[e] = __floats2bfloat162_rn(__uint_as_float(v[8 * g + 2 * e]) * mul, __uint_as_float(v[8 * g + 2 * e + 1]) * mul);
        *reinterpret_cast<uint4*>(to + 8 * g) = pk;
    }
}

// Columns of a tile of 128 keys from k0 on that query i sees:
// c <= hi and (c > lo or c < front).
struct Cols {
    int hi, lo, front;
    __device__ __forceinline__ Cols(const WindowDesc& d, int i, int k0)
        : hi(i - k0), lo(d.window && i >= d.window ? i - d.window - k0 : -1), front(d.sinks - k0) {}
    __device__ __forceinline__ bool operator()(int c) const { return c <= hi && (c > lo || c < front); }
};
// Whether queries q0 .. q0 + 127 all see every key of the tile.
__device__ __forceinline__ bool all_seen(const WindowDesc& d, int q0, int k0) {
    return k0 + kT - 1 <= q0 && (d.window == 0 || q0 + kT - 1 - k0 < d.window || k0 + kT - 1 < d.sinks);
}

// ---------------------------------------------------------------------------
// Forward. A block has 256 neighbouring queries of one head, two tiles of 128:
//   warp 9     TMA: the queries, then keys and values tile by tile through a
//              ring of slots
//   warp 8     every MMA: S_g = Q_g K^T into TMEM columns [128 g, + 128),
//              O_g += P_g V into [256 + 128 g, ...), P_g (bf16) read from the
//              columns that held S_g. While one tile of queries is in its
//              softmax, the tensor cores run the other's products.
//   warps 4 g .. 4 g + 3   softmax of tile g, a query a thread: the scores come
//              from TMEM into registers once, weights go back as bf16 pairs
//              (half a step of 2^-9; their fp32 sum is taken before).
// O stays in TMEM. It is scaled only when a row's maximum rises by more than
// 2^8 above the one that its weights are taken against: smaller rises cost
// neither range (fp32) nor precision (the weights are floating point).
// ---------------------------------------------------------------------------
constexpr int kFwdThreads = 320;
constexpr float kRise = 8.f;

template <int DHP>
struct Fwd {
    static constexpr int TILE = DHP / 64 * kChunk;
    static constexpr int SLOTS = DHP == 128 ? 5 : 8;
    static constexpr int SMEM = (2 + SLOTS) * TILE + 512 + 1024;
};

}  // namespace

template <int DHP>
__global__ void __launch_bounds__(kFwdThreads, 1)
    window_tc_fwd_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                         const __grid_constant__ CUtensorMap tv, const __grid_constant__ WindowDesc d) {
    using F = Fwd<DHP>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* ring = smem + 2 * F::TILE;
    uint64_t* q_full = reinterpret_cast<uint64_t*>(ring + F::SLOTS * F::TILE);
    uint64_t* full = q_full + 1;
    uint64_t* empty = full + F::SLOTS;
    uint64_t* s_bar = empty + F::SLOTS;  // [2] scores of group g in TMEM
    uint64_t* p_bar = s_bar + 2;         // [2] weights of group g in TMEM (128 arrivals)
    uint64_t* o_bar = p_bar + 2;         // [2] product of group g added to O
    uint64_t* drain = o_bar + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    int* failed = reinterpret_cast<int*>(tmem_slot + 1);

    const int t = threadIdx.x, warp = t >> 5;
    const int h = blockIdx.x % d.Hq, hk = h / (d.Hq / d.Hkv);
    // last tiles first: without a window they are the longest
    const Rows w = find_rows(d, gridDim.x / d.Hq - 1 - blockIdx.x / d.Hq, 2 * kT);
    if (w.n <= 0) return;
    const int q0 = w.first, row0 = (int)w.row0;
    const bool two = q0 + kT < w.n;

    if (t == 0) {
        ptx::mbar_init(q_full, 1);
        for (int i = 0; i < F::SLOTS; i++) {
            ptx::mbar_init(&full[i], 1);
            ptx::mbar_init(&empty[i], 1);
        }
        for (int g = 0; g < 2; g++) {
            ptx::mbar_init(&s_bar[g], 1);
            ptx::mbar_init(&p_bar[g], 128);
            ptx::mbar_init(&o_bar[g], 1);
        }
        ptx::mbar_init(drain, 1);
        *failed = 0;
        ptx::fence_mbar_init();
    }
    if (warp == 8) {
        ptx::tmem_alloc(tmem_slot, 512);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const Waits wait{failed, d.err};
    bool ok = true;

    const KeyTiles tiles(d, q0, min(q0 + 2 * kT, w.n), kT);
    const int sink_tiles = d.sinks / kT + (d.sinks % kT != 0);
    auto uses = [&](int g, int kt) {
        const int first = q0 + g * kT;
        const int lo = d.window && first >= d.window ? (first - d.window + 1) / kT : 0;
        return (g == 0 || two) && kt * kT <= first && (kt >= lo || kt < sink_tiles);
    };

    if (warp == 9) {
        if ((t & 31) == 0) {
            ptx::mbar_arrive_expect_tx(q_full, (two ? 2 : 1) * F::TILE);
            for (int g = 0; g < (two ? 2 : 1); g++)
                for (int c = 0; c < DHP / 64; c++)
                    ptx::tma_load_3d(smem + g * F::TILE + c * kChunk, &tq, q_full, c * 64, h, row0 + q0 + g * kT);
            int it = 0;
            for (int x = 0; x < tiles.count && ok; x++) {
                const int row = row0 + tiles.at(x) * kT;
                for (int kv = 0; kv < 2; kv++, it++) {
                    const int slot = it % F::SLOTS, round = it / F::SLOTS;
                    if (round && !(ok = wait.lane(&empty[slot], round - 1))) break;
                    load_rows<DHP>(ring + slot * F::TILE, kv ? &tv : &tk, &full[slot], hk, row);
                }
            }
            // no copy may land after the block has left
            ptx::mbar_wait(q_full, 0, nullptr, 0);
            for (int i = max(0, it - F::SLOTS); i < it; i++)
                ptx::mbar_wait(&full[i % F::SLOTS], (i / F::SLOTS) & 1, nullptr, 0);
        }
    } else if (warp == 8) {
        const bool one = (t & 31) == 0;
        const uint32_t aQ = ptx::smem_u32(smem), aR = ptx::smem_u32(ring);
        constexpr uint32_t idesc = ptx::instr_desc(1, 0, 1, kT, DHP);
        uint32_t given[2] = {0, 0};  // weights taken, by group
        ok = wait(q_full, 0);
        for (int x = 0; x <= tiles.count && ok; x++) {
            const int ik = 2 * x, iv = 2 * x - 1;  // what the ring's slots hold: K0 V0 K1 V1 ...
            const int sk = ik % F::SLOTS, sv = iv > 0 ? iv % F::SLOTS : 0;
            const int kt = x < tiles.count ? tiles.at(x) : 0, before = x > 0 ? tiles.at(x - 1) : 0;
            if (x > 0) {
                if (!(ok = wait(&full[sv], iv / F::SLOTS))) break;
                if ((before + 1) * kT > w.n) zero_rows<DHP>(ring + sv * F::TILE, w.n - before * kT);
            }
            if (x < tiles.count && !(ok = wait(&full[sk], ik / F::SLOTS))) break;
#pragma unroll
            for (int g = 0; g < 2; g++) {
                if (x > 0 && uses(g, before)) {
                    if (!(ok = wait(&p_bar[g], given[g]))) break;
                    ptx::tc_fence_after();
                    if (one) {
#pragma unroll
                        for (int s = 0; s < kT / 16; s++)
                            ptx::mma_bf16_ts(tmem + 256 + 128 * g, tmem + 128 * g + 8 * s,
                                             ptx::smem_desc(aR + sv * F::TILE + s * 2048, kChunk, 1024, 2), idesc,
                                             given[g] > 0 || s > 0);
                        ptx::mma_commit(&o_bar[g]);
                    }
                    given[g]++;
                }
                if (x < tiles.count && uses(g, kt) && one) {
                    ptx::tc_fence_after();
                    mma_dot<DHP>(tmem + 128 * g, aQ + g * F::TILE, aR + sk * F::TILE);
                    ptx::mma_commit(&s_bar[g]);
                }
            }
            if (ok && one) {
                if (x > 0) ptx::mma_commit(&empty[sv]);
                if (x < tiles.count) ptx::mma_commit(&empty[sk]);
            }
            __syncwarp();
        }
        if (one) {
            ptx::mma_commit(drain);
            ptx::mbar_wait(drain, 0, nullptr, 0);
        }
    } else if (warp < 4 || two) {
        const int g = warp >> 2, lg = warp & 3;
        const int i = q0 + g * kT + lg * 32 + (t & 31);  // query of the sequence
        const uint32_t base = tmem + ((uint32_t)(lg * 32) << 16) + 128 * g;
        const uint32_t o_at = tmem + ((uint32_t)(lg * 32) << 16) + 256 + 128 * g;
        const float sl2 = d.scale * kLog2e;
        float ref = -INFINITY, sum = 0.f;  // what the weights are taken against (powers of two), their sum
        uint32_t done = 0;                 // tiles behind
        for (int x = 0; x < tiles.count; x++) {
            const int kt = tiles.at(x), k0 = kt * kT;
            if (!uses(g, kt)) continue;
            if (!(ok = wait(&s_bar[g], done))) break;
            ptx::tc_fence_after();
            uint32_t a[128];
#pragma unroll
            for (int c = 0; c < 4; c++) ptx::tmem_ld32(base + 32 * c, a + 32 * c);
#pragma unroll
            for (int c = 0; c < 4; c++) ptx::tmem_ld_wait_regs32(a + 32 * c);
            if (!all_seen(d, q0 + g * kT, k0)) {
                const Cols on(d, i, k0);
#pragma unroll
                for (int c = 0; c < 128; c++)
                    if (!on(c)) a[c] = 0xff800000u;
            }
            float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < 128; c += 2)
                m4[(c >> 1) & 3] = max3(m4[(c >> 1) & 3], __uint_as_float(a[c]), __uint_as_float(a[c + 1]));
            const float top = fmaxf(max3(m4[0], m4[1], m4[2]), m4[3]) * sl2;  // (the scale is positive)
            const bool rise = top > ref + kRise;  // ref -inf: the first finite score
            if (__any_sync(0xffffffffu, rise)) {
                const float turn = rise ? ex2(ref - top) : 1.f;
                if (rise) ref = top;
                sum *= turn;
                if (done) {
                    if (!(ok = wait(&o_bar[g], done - 1))) break;
                    ptx::tc_fence_after();
#pragma unroll 1
                    for (int c = 0; c < DHP; c += 16) {
                        uint32_t o[16];
                        ptx::tmem_ld16(o_at + c, o);
                        ptx::tmem_ld_wait_regs16(o);
#pragma unroll
                        for (int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * turn);
                        ptx::tmem_st16(o_at + c, o);
                    }
                }
            }
            const float safe = ref == -INFINITY ? 0.f : ref;
            const uint64_t SL2 = f2_pack(sl2, sl2), NEG = f2_pack(-safe, -safe);
            uint64_t s4[4] = {0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < 128; c += 32) {
                uint32_t pk[16];
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    float x0, x1;
                    f2_unpack(f2_fma(f2_pack(__uint_as_float(a[c + 2 * e]), __uint_as_float(a[c + 2 * e + 1])), SL2, NEG), x0, x1);
                    x0 = ex2(x0);
                    x1 = ex2(x1);
                    s4[e & 3] = f2_add(s4[e & 3], f2_pack(x0, x1));
                    const __nv_bfloat162 p = __floats2bfloat162_rn(x0, x1);
                    pk[e] = *reinterpret_cast<const uint32_t*>(&p);
                }
                ptx::tmem_st16(base + c / 2, pk);
            }
            float s0, s1;
            f2_unpack(f2_add(f2_add(s4[0], s4[1]), f2_add(s4[2], s4[3])), s0, s1);
            sum += s0 + s1;
            ptx::tmem_st_wait();
            ptx::tc_fence_before();
            ptx::mbar_arrive(&p_bar[g]);
            done++;
        }
        ok = ok && wait(&o_bar[g], done - 1);  // a query's own tile is always among its tiles
        ptx::tc_fence_after();
        if (ok) {
            const float mul = sum == 0.f ? 0.f : 1.f / sum;
            __nv_bfloat16* to = (__nv_bfloat16*)d.out.p + (w.row0 + i) * d.out.row + h * d.out.head;
#pragma unroll 1
            for (int c = 0; c < DHP; c += 32) {
                uint32_t v[32];
                ptx::tmem_ld32(o_at + c, v);
                ptx::tmem_ld_wait_regs32(v);
                if (i < w.n) store32(to + c, v, mul, d.dh - c);
            }
            if (i < w.n && d.lse) d.lse[h * d.ld_lse + w.row0 + i] = sum == 0.f ? -INFINITY : (ref + log2f(sum)) * kLn2;
        }
    }
    ptx::tc_fence_before();
    __syncthreads();
    if (warp == 8) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem, 512);
    }
}

// ---------------------------------------------------------------------------
// Gradient of the queries. A block has 128 queries of one head and walks the
// tiles of keys that they see:
//   warp 9     TMA: queries and dout, then keys and values through a ring
//   warp 8     every MMA: S = Q K^T into TMEM columns [0, 128),
//              dP = dout V^T into [128, 256), dQ += dS K into [256, ...), dS
//              (bf16) read from [384, 448). The next tile's S and dP run while
//              this one's dS is computed.
//   warps 0..7 dS = P (dP - D), two threads a query with 64 keys each. Before
//              the first tile they form D = rowdot(dout, out), which the second
//              kernel reads too.
// ---------------------------------------------------------------------------
constexpr int kBwdQThreads = 320;

template <int DHP>
struct BwdQ {
    static constexpr int TILE = DHP / 64 * kChunk;
    static constexpr int SLOTS = DHP == 128 ? 4 : 8;
    static constexpr int SMEM = (2 + SLOTS) * TILE + 256 * 4 + 512 + 1024;
};

template <int DHP>
__global__ void __launch_bounds__(kBwdQThreads, 1)
    window_tc_bwd_q_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                           const __grid_constant__ CUtensorMap tv, const __grid_constant__ CUtensorMap tg,
                           const __grid_constant__ WindowDesc d) {
    using F = BwdQ<DHP>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* ring = smem + 2 * F::TILE;
    float* sums = reinterpret_cast<float*>(ring + F::SLOTS * F::TILE);  // [2][128] halves of D
    uint64_t* q_full = reinterpret_cast<uint64_t*>(sums + 256);
    uint64_t* full = q_full + 1;
    uint64_t* empty = full + F::SLOTS;
    uint64_t* s_bar = empty + F::SLOTS;  // S and dP of a tile in TMEM
    uint64_t* r_bar = s_bar + 1;         // both read (256 arrivals)
    uint64_t* p_bar = r_bar + 1;         // dS in TMEM (256 arrivals)
    uint64_t* o_bar = p_bar + 1;         // product added to dQ
    uint64_t* drain = o_bar + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    int* failed = reinterpret_cast<int*>(tmem_slot + 1);

    const int t = threadIdx.x, warp = t >> 5;
    const int h = blockIdx.x % d.Hq, hk = h / (d.Hq / d.Hkv);
    const Rows w = find_rows(d, gridDim.x / d.Hq - 1 - blockIdx.x / d.Hq, kT);
    if (w.n <= 0) return;
    const int q0 = w.first, row0 = (int)w.row0;

    if (t == 0) {
        ptx::mbar_init(q_full, 1);
        for (int i = 0; i < F::SLOTS; i++) {
            ptx::mbar_init(&full[i], 1);
            ptx::mbar_init(&empty[i], 1);
        }
        ptx::mbar_init(s_bar, 1);
        ptx::mbar_init(r_bar, 256);
        ptx::mbar_init(p_bar, 256);
        ptx::mbar_init(o_bar, 1);
        ptx::mbar_init(drain, 1);
        *failed = 0;
        ptx::fence_mbar_init();
    }
    if (warp == 8) {
        ptx::tmem_alloc(tmem_slot, 512);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const Waits wait{failed, d.err};
    bool ok = true;
    const KeyTiles tiles(d, q0, min(q0 + kT, w.n), kT);

    if (warp == 9) {
        if ((t & 31) == 0) {
            ptx::mbar_arrive_expect_tx(q_full, 2 * F::TILE);
            for (int c = 0; c < DHP / 64; c++) {
                ptx::tma_load_3d(smem + c * kChunk, &tq, q_full, c * 64, h, row0 + q0);
                ptx::tma_load_3d(smem + F::TILE + c * kChunk, &tg, q_full, c * 64, h, row0 + q0);
            }
            int it = 0;
            for (int x = 0; x < tiles.count && ok; x++) {
                const int row = row0 + tiles.at(x) * kT;
                for (int kv = 0; kv < 2; kv++, it++) {
                    const int slot = it % F::SLOTS, round = it / F::SLOTS;
                    if (round && !(ok = wait.lane(&empty[slot], round - 1))) break;
                    load_rows<DHP>(ring + slot * F::TILE, kv ? &tv : &tk, &full[slot], hk, row);
                }
            }
            ptx::mbar_wait(q_full, 0, nullptr, 0);
            for (int i = max(0, it - F::SLOTS); i < it; i++)
                ptx::mbar_wait(&full[i % F::SLOTS], (i / F::SLOTS) & 1, nullptr, 0);
        }
    } else if (warp == 8) {
        const bool one = (t & 31) == 0;
        const uint32_t aQ = ptx::smem_u32(smem), aG = aQ + F::TILE, aR = ptx::smem_u32(ring);
        constexpr uint32_t idesc = ptx::instr_desc(1, 0, 1, kT, DHP);
        ok = wait(q_full, 0);
        for (int x = 0; x <= tiles.count && ok; x++) {
            if (x < tiles.count) {
                const int sk = 2 * x % F::SLOTS, sv = (2 * x + 1) % F::SLOTS, kt = tiles.at(x);
                if (!(ok = wait(&full[sk], 2 * x / F::SLOTS) && wait(&full[sv], (2 * x + 1) / F::SLOTS))) break;
                if ((kt + 1) * kT > w.n) zero_rows<DHP>(ring + sk * F::TILE, w.n - kt * kT);
                if (x > 0 && !(ok = wait(r_bar, x - 1))) break;
                ptx::tc_fence_after();
                if (one) {
                    mma_dot<DHP>(tmem, aQ, aR + sk * F::TILE);
                    mma_dot<DHP>(tmem + 128, aG, aR + sv * F::TILE);
                    ptx::mma_commit(s_bar);
                    ptx::mma_commit(&empty[sv]);
                }
            }
            if (x > 0) {
                const int sk = 2 * (x - 1) % F::SLOTS;
                if (!(ok = wait(p_bar, x - 1))) break;
                ptx::tc_fence_after();
                if (one) {
#pragma unroll
                    for (int s = 0; s < kT / 16; s++)
                        ptx::mma_bf16_ts(tmem + 256, tmem + 384 + 8 * s,
                                         ptx::smem_desc(aR + sk * F::TILE + s * 2048, kChunk, 1024, 2), idesc, x > 1 || s > 0);
                    ptx::mma_commit(o_bar);
                    ptx::mma_commit(&empty[sk]);
                }
            }
            __syncwarp();
        }
        if (one) {
            ptx::mma_commit(drain);
            ptx::mbar_wait(drain, 0, nullptr, 0);
        }
    } else {
        const int lg = warp & 3, half = warp >> 2, r = lg * 32 + (t & 31);
        const int i = q0 + r;
        const uint32_t base = tmem + ((uint32_t)(lg * 32) << 16);
        const float sl2 = d.scale * kLog2e;
        float lse2 = INFINITY, D = 0.f;  // a query that saw nothing has weights of 0
        if (i < w.n) {
            const float lse = d.lse[h * d.ld_lse + w.row0 + i];
            if (lse != -INFINITY) lse2 = lse * kLog2e;
            const __nv_bfloat16* g = (const __nv_bfloat16*)d.dout.p + (w.row0 + i) * d.dout.row + h * d.dout.head;
            const __nv_bfloat16* o = (const __nv_bfloat16*)d.out.p + (w.row0 + i) * d.out.row + h * d.out.head;
#pragma unroll
            for (int c = 0; c < DHP / 2; c += 8) {
                const int at = half * (DHP / 2) + c;
                if (at < d.dh) {
                    const uint4 x = *reinterpret_cast<const uint4*>(g + at), y = *reinterpret_cast<const uint4*>(o + at);
                    const __nv_bfloat162* x2 = reinterpret_cast<const __nv_bfloat162*>(&x);
                    const __nv_bfloat162* y2 = reinterpret_cast<const __nv_bfloat162*>(&y);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float2 a = __bfloat1622float2(x2[e]), b = __bfloat1622float2(y2[e]);
                        D = fmaf(a.x, b.x, D);
                        D = fmaf(a.y, b.y, D);
                    }
                }
            }
        }
        sums[half * 128 + r] = D;
        asm volatile("bar.sync 1, 256;" ::: "memory");
        D = sums[r] + sums[128 + r];
        if (half == 0 && i < w.n) d.dvec[(long long)h * d.T + w.row0 + i] = D;
        const uint64_t SL2 = f2_pack(sl2, sl2), NEG = f2_pack(-lse2, -lse2), ND = f2_pack(-D, -D);
        for (int x = 0; x < tiles.count; x++) {
            const int k0 = tiles.at(x) * kT;
            if (!(ok = wait(s_bar, x))) break;
            ptx::tc_fence_after();
            uint32_t a[64], g[64];
#pragma unroll
            for (int c = 0; c < 2; c++) {
                ptx::tmem_ld32(base + half * 64 + 32 * c, a + 32 * c);
                ptx::tmem_ld32(base + 128 + half * 64 + 32 * c, g + 32 * c);
            }
#pragma unroll
            for (int c = 0; c < 2; c++) {
                ptx::tmem_ld_wait_regs32(a + 32 * c);
                ptx::tmem_ld_wait_regs32(g + 32 * c);
            }
            ptx::tc_fence_before();
            ptx::mbar_arrive(r_bar);
            const bool whole = all_seen(d, q0, k0);
            const Cols on(d, i, k0);
            uint32_t pk[32];
#pragma unroll
            for (int e = 0; e < 32; e++) {
                float x0, x1, y0, y1;
                f2_unpack(f2_fma(f2_pack(__uint_as_float(a[2 * e]), __uint_as_float(a[2 * e + 1])), SL2, NEG), x0, x1);
                f2_unpack(f2_mul(f2_pack(ex2(x0), ex2(x1)),
                                 f2_add(f2_pack(__uint_as_float(g[2 * e]), __uint_as_float(g[2 * e + 1])), ND)),
                          y0, y1);
                if (!whole) {
                    y0 = on(half * 64 + 2 * e) ? y0 : 0.f;
                    y1 = on(half * 64 + 2 * e + 1) ? y1 : 0.f;
                }
                const __nv_bfloat162 p = __floats2bfloat162_rn(y0, y1);
                pk[e] = *reinterpret_cast<const uint32_t*>(&p);
            }
            if (x > 0) {
                if (!(ok = wait(o_bar, x - 1))) break;  // the product before has read its dS
                ptx::tc_fence_after();
            }
            ptx::tmem_st16(base + 384 + half * 32, pk);
            ptx::tmem_st16(base + 384 + half * 32 + 16, pk + 16);
            ptx::tmem_st_wait();
            ptx::tc_fence_before();
            ptx::mbar_arrive(p_bar);
        }
        ok = ok && wait(o_bar, tiles.count - 1);
        ptx::tc_fence_after();
        if (ok) {
            __nv_bfloat16* to = (__nv_bfloat16*)d.dq.p + (w.row0 + i) * d.dq.row + h * d.dq.head;
#pragma unroll 1
            for (int c = half * (DHP / 2); c < (half + 1) * (DHP / 2); c += 32) {
                uint32_t v[32];
                ptx::tmem_ld32(base + 256 + c, v);
                ptx::tmem_ld_wait_regs32(v);
                if (i < w.n) store32(to + c, v, d.scale, d.dh - c);
            }
        }
    }
    ptx::tc_fence_before();
    __syncthreads();
    if (warp == 8) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem, 512);
    }
}

// ---------------------------------------------------------------------------
// Gradients of keys and values. A block has 128 keys of one key head and walks
// the tiles of queries, of all heads that share it, that see any of them. The
// scores stand transposed, a key a row, so that both sums run over TMEM's
// columns:
//   warp 9     TMA: keys and values, then queries and dout through a ring
//   warp 10    lse and D of each tile of queries, into a ring of their own
//   warp 8     every MMA: S^T = K Q^T into TMEM columns [0, 128), dP^T = V dout^T
//              into [128, 256), dV += P^T dout into [256, ...), dK += dS^T Q into
//              [384, ...). P^T and dS^T (bf16) take the columns of the scores
//              that they come from.
//   warps 0..7 P and dS, two threads a key with 64 queries each: while P is
//              computed the tensor cores run dK and the next dP, while dS is,
//              dV and the next S.
// ---------------------------------------------------------------------------
constexpr int kBwdKvThreads = 352;
constexpr int kStats = 4;  // tiles of lse and D held

template <int DHP>
struct BwdKv {
    static constexpr int TILE = DHP / 64 * kChunk;
    static constexpr int SLOTS = DHP == 128 ? 4 : 8;
    static constexpr int SMEM = (2 + SLOTS) * TILE + kStats * 2 * kT * 4 + 512 + 1024;
};

template <int DHP>
__global__ void __launch_bounds__(kBwdKvThreads, 1)
    window_tc_bwd_kv_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                            const __grid_constant__ CUtensorMap tv, const __grid_constant__ CUtensorMap tg,
                            const __grid_constant__ WindowDesc d) {
    using F = BwdKv<DHP>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* ring = smem + 2 * F::TILE;
    float* stats = reinterpret_cast<float*>(ring + F::SLOTS * F::TILE);  // [kStats][lse | D][128]
    uint64_t* k_full = reinterpret_cast<uint64_t*>(stats + kStats * 2 * kT);
    uint64_t* full = k_full + 1;
    uint64_t* empty = full + F::SLOTS;
    uint64_t* st_full = empty + F::SLOTS;  // (32 arrivals)
    uint64_t* st_empty = st_full + kStats; // (256 arrivals)
    uint64_t* s_bar = st_empty + kStats;   // S^T in TMEM
    uint64_t* g_bar = s_bar + 1;           // dP^T in TMEM
    uint64_t* p_bar = g_bar + 1;           // P^T in TMEM (256 arrivals)
    uint64_t* ds_bar = p_bar + 1;          // dS^T in TMEM (256 arrivals)
    uint64_t* drain = ds_bar + 1;          // every product done
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    int* failed = reinterpret_cast<int*>(tmem_slot + 1);

    const int t = threadIdx.x, warp = t >> 5;
    const int hk = blockIdx.x % d.Hkv, group = d.Hq / d.Hkv;
    const Rows w = find_rows(d, blockIdx.x / d.Hkv, kT);
    if (w.n <= 0) return;
    const int k0 = w.first, row0 = (int)w.row0;
    const int first = k0 / kT, each = query_tiles_end(d, k0, w.n, kT) - first, count = each * group;

    if (t == 0) {
        ptx::mbar_init(k_full, 1);
        for (int i = 0; i < F::SLOTS; i++) {
            ptx::mbar_init(&full[i], 1);
            ptx::mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < kStats; i++) {
            ptx::mbar_init(&st_full[i], 32);
            ptx::mbar_init(&st_empty[i], 256);
        }
        ptx::mbar_init(s_bar, 1);
        ptx::mbar_init(g_bar, 1);
        ptx::mbar_init(p_bar, 256);
        ptx::mbar_init(ds_bar, 256);
        ptx::mbar_init(drain, 1);
        *failed = 0;
        ptx::fence_mbar_init();
    }
    if (warp == 8) {
        ptx::tmem_alloc(tmem_slot, 512);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const Waits wait{failed, d.err};
    bool ok = true;

    if (warp == 9) {
        if ((t & 31) == 0) {
            ptx::mbar_arrive_expect_tx(k_full, 2 * F::TILE);
            for (int c = 0; c < DHP / 64; c++) {
                ptx::tma_load_3d(smem + c * kChunk, &tk, k_full, c * 64, hk, row0 + k0);
                ptx::tma_load_3d(smem + F::TILE + c * kChunk, &tv, k_full, c * 64, hk, row0 + k0);
            }
            int it = 0;
            for (int x = 0; x < count && ok; x++) {
                const int h = hk * group + x / each, row = row0 + (first + x % each) * kT;
                for (int qg = 0; qg < 2; qg++, it++) {
                    const int slot = it % F::SLOTS, round = it / F::SLOTS;
                    if (round && !(ok = wait.lane(&empty[slot], round - 1))) break;
                    load_rows<DHP>(ring + slot * F::TILE, qg ? &tg : &tq, &full[slot], h, row);
                }
            }
            ptx::mbar_wait(k_full, 0, nullptr, 0);
            for (int i = max(0, it - F::SLOTS); i < it; i++)
                ptx::mbar_wait(&full[i % F::SLOTS], (i / F::SLOTS) & 1, nullptr, 0);
        }
    } else if (warp == 10) {
        for (int x = 0; x < count && ok; x++) {
            const int slot = x % kStats, h = hk * group + x / each, q0 = (first + x % each) * kT;
            float l[4], D[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int i = q0 + (t & 31) + 32 * e;
                // a query that saw nothing, or is none, has weights of 0
                l[e] = INFINITY;
                D[e] = 0.f;
                if (i < w.n) {
                    const float lse = d.lse[h * d.ld_lse + w.row0 + i];
                    if (lse != -INFINITY) l[e] = lse * kLog2e;
                    D[e] = d.dvec[(long long)h * d.T + w.row0 + i];
                }
            }
            if (x >= kStats && !(ok = wait(&st_empty[slot], x / kStats - 1))) break;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                stats[slot * 2 * kT + (t & 31) + 32 * e] = l[e];
                stats[slot * 2 * kT + kT + (t & 31) + 32 * e] = D[e];
            }
            ptx::mbar_arrive(&st_full[slot]);
        }
    } else if (warp == 8) {
        const bool one = (t & 31) == 0;
        const uint32_t aK = ptx::smem_u32(smem), aV = aK + F::TILE, aR = ptx::smem_u32(ring);
        constexpr uint32_t idesc = ptx::instr_desc(1, 0, 1, kT, DHP);
        // the slot that a tile's queries (0) or dout (1) are in, with zeros behind the sequence's end
        auto ready = [&](int x, int qg) {
            const int i = 2 * x + qg, slot = i % F::SLOTS, q0 = (first + x % each) * kT;
            ok = wait(&full[slot], i / F::SLOTS);
            if (ok && q0 + kT > w.n) zero_rows<DHP>(ring + slot * F::TILE, w.n - q0);
            return aR + slot * F::TILE;
        };
        // d += A (bf16 of 128 queries in 2 x 32 columns, 64 apart) times the rows at b
        auto add = [&](uint32_t d0, uint32_t a, uint32_t b, bool more) {
#pragma unroll
            for (int s = 0; s < kT / 16; s++)
                ptx::mma_bf16_ts(d0, a + 64 * (s >> 2) + 8 * (s & 3), ptx::smem_desc(b + s * 2048, kChunk, 1024, 2), idesc,
                                 more || s > 0);
        };
        ok = wait(k_full, 0);
        uint32_t aQ = 0, aG = 0;  // of the tile whose weights are awaited
        if (ok) aQ = ready(0, 0);
        if (ok) aG = ready(0, 1);
        if (ok && one) {
            ptx::tc_fence_after();
            mma_dot<DHP>(tmem, aK, aQ);
            ptx::mma_commit(s_bar);
            mma_dot<DHP>(tmem + 128, aV, aG);
            ptx::mma_commit(g_bar);
        }
        for (int x = 0; x < count && ok; x++) {
            const bool more = x + 1 < count;
            uint32_t nQ = 0, nG = 0;
            if (more) nQ = ready(x + 1, 0);
            if (!ok || !(ok = wait(p_bar, x))) break;
            if (one) {
                ptx::tc_fence_after();
                add(tmem + 256, tmem, aG, x > 0);
                ptx::mma_commit(&empty[(2 * x + 1) % F::SLOTS]);
                if (more) {
                    mma_dot<DHP>(tmem, aK, nQ);
                    ptx::mma_commit(s_bar);
                }
            }
            __syncwarp();
            if (more) nG = ready(x + 1, 1);
            if (!ok || !(ok = wait(ds_bar, x))) break;
            if (one) {
                ptx::tc_fence_after();
                add(tmem + 384, tmem + 128, aQ, x > 0);
                ptx::mma_commit(&empty[2 * x % F::SLOTS]);
                if (more) {
                    mma_dot<DHP>(tmem + 128, aV, nG);
                    ptx::mma_commit(g_bar);
                }
            }
            __syncwarp();
            aQ = nQ;
            aG = nG;
        }
        if (one) {
            ptx::mma_commit(drain);
            ptx::mbar_wait(drain, 0, nullptr, 0);
        }
    } else {
        const int lg = warp & 3, half = warp >> 2;
        const int j = k0 + lg * 32 + (t & 31);  // key of the sequence
        const uint32_t base = tmem + ((uint32_t)(lg * 32) << 16) + 64 * half;
        const float sl2 = d.scale * kLog2e;
        const uint64_t SL2 = f2_pack(sl2, sl2), MINUS = f2_pack(-1.f, -1.f);
        const bool no_end = d.window == 0 || d.window >= w.n || j < d.sinks;
        for (int x = 0; x < count; x++) {
            const int slot = x % kStats, q0 = (first + x % each) * kT;
            const float4* l4 = reinterpret_cast<const float4*>(stats + slot * 2 * kT + half * 64);
            const float4* d4 = l4 + kT / 4;
            const bool whole = all_seen(d, q0, k0);
            // queries q0 + c that see key j: lo <= c < hi
            const int lo = j - q0 - half * 64, hi = no_end ? kT : j + d.window - q0 - half * 64;
            if (!(ok = wait(&st_full[slot], x / kStats) && wait(s_bar, x))) break;
            ptx::tc_fence_after();
            uint32_t a[64], g[64];
#pragma unroll
            for (int c = 0; c < 2; c++) ptx::tmem_ld32(base + 32 * c, a + 32 * c);
#pragma unroll
            for (int c = 0; c < 2; c++) ptx::tmem_ld_wait_regs32(a + 32 * c);
            uint32_t pk[32];
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
                const float4 l = l4[e / 2];
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const int c = 2 * (e + u);
                    float x0, x1;
                    f2_unpack(f2_fma(f2_pack(__uint_as_float(a[c]), __uint_as_float(a[c + 1])), SL2,
                                     f2_mul(u ? f2_pack(l.z, l.w) : f2_pack(l.x, l.y), MINUS)),
                              x0, x1);
                    x0 = ex2(x0);
                    x1 = ex2(x1);
                    if (!whole) {
                        x0 = c >= lo && c < hi ? x0 : 0.f;
                        x1 = c + 1 >= lo && c + 1 < hi ? x1 : 0.f;
                    }
                    a[c] = __float_as_uint(x0);
                    a[c + 1] = __float_as_uint(x1);
                    const __nv_bfloat162 p = __floats2bfloat162_rn(x0, x1);
                    pk[e + u] = *reinterpret_cast<const uint32_t*>(&p);
                }
            }
            ptx::tmem_st16(base, pk);
            ptx::tmem_st16(base + 16, pk + 16);
            ptx::tmem_st_wait();
            ptx::tc_fence_before();
            ptx::mbar_arrive(p_bar);
            if (!(ok = wait(g_bar, x))) break;
            ptx::tc_fence_after();
#pragma unroll
            for (int c = 0; c < 2; c++) ptx::tmem_ld32(base + 128 + 32 * c, g + 32 * c);
#pragma unroll
            for (int c = 0; c < 2; c++) ptx::tmem_ld_wait_regs32(g + 32 * c);
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
                const float4 D = d4[e / 2];
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const int c = 2 * (e + u);
                    float y0, y1;
                    f2_unpack(f2_mul(f2_pack(__uint_as_float(a[c]), __uint_as_float(a[c + 1])),
                                     f2_fma(u ? f2_pack(D.z, D.w) : f2_pack(D.x, D.y), MINUS,
                                            f2_pack(__uint_as_float(g[c]), __uint_as_float(g[c + 1])))),
                              y0, y1);
                    if (!whole) {  // a hidden place stays 0 whatever dP is
                        y0 = c >= lo && c < hi ? y0 : 0.f;
                        y1 = c + 1 >= lo && c + 1 < hi ? y1 : 0.f;
                    }
                    const __nv_bfloat162 p = __floats2bfloat162_rn(y0, y1);
                    pk[e + u] = *reinterpret_cast<const uint32_t*>(&p);
                }
            }
            ptx::tmem_st16(base + 128, pk);
            ptx::tmem_st16(base + 144, pk + 16);
            ptx::tmem_st_wait();
            ptx::tc_fence_before();
            ptx::mbar_arrive(ds_bar);
            ptx::mbar_arrive(&st_empty[slot]);
        }
        ok = ok && wait(drain, 0);
        ptx::tc_fence_after();
        if (ok && !*(volatile int*)failed) {
            const uint32_t row = tmem + ((uint32_t)(lg * 32) << 16);
            __nv_bfloat16* dv = (__nv_bfloat16*)d.dv.p + (w.row0 + j) * d.dv.row + hk * d.dv.head;
            __nv_bfloat16* dk = (__nv_bfloat16*)d.dk.p + (w.row0 + j) * d.dk.row + hk * d.dk.head;
#pragma unroll 1
            for (int c = half * (DHP / 2); c < (half + 1) * (DHP / 2); c += 32) {
                uint32_t v[32], k[32];
                ptx::tmem_ld32(row + 256 + c, v);
                ptx::tmem_ld32(row + 384 + c, k);
                ptx::tmem_ld_wait_regs32(v);
                ptx::tmem_ld_wait_regs32(k);
                if (j < w.n) {
                    store32(dv + c, v, 1.f, d.dh - c);
                    store32(dk + c, k, d.scale, d.dh - c);
                }
            }
        }
    }
    ptx::tc_fence_before();
    __syncthreads();
    if (warp == 8) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem, 512);
    }
}

namespace {

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                             const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encoder() {
    static EncodeFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeFn>(f);
    });
    return fn;
}

// Columns, heads and rows of a tensor of heads; boxes of 64 columns of one
// head in 128 rows. What a box has past the columns or the rows reads as zeros.
bool make_map(CUtensorMap* m, const Heads& x, int T, int H, int dh) {
    EncodeFn enc = encoder();
    if (!enc) return false;
    cuuint64_t dims[3] = {(cuuint64_t)dh, (cuuint64_t)H, (cuuint64_t)T};
    cuuint64_t strides[2] = {(cuuint64_t)((H > 1 ? x.head : 8) * 2), (cuuint64_t)((T > 1 ? x.row : 8) * 2)};
    cuuint32_t box[3] = {64, 1, kT}, unit[3] = {1, 1, 1};
    return enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, x.p, dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Whether TMA, and 16-byte loads and stores, reach every row of x.
bool rows16(const Heads& x, int T, int H) {
    auto fits = [](long long s, int n) { return n <= 1 || (s % 8 == 0 && s > 0 && s < (1LL << 38)); };
    return reinterpret_cast<uintptr_t>(x.p) % 16 == 0 && fits(x.row, T) && fits(x.head, H);
}

template <typename K>
bool room(K kernel, int bytes) {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) == cudaSuccess;
}

long long tiles_of(const WindowDesc& d, int rows) { return ((long long)d.T + rows - 1) / rows + (d.offsets ? d.B : 0); }

template <int DHP>
int fwd(const WindowDesc& d, cudaStream_t s) {
    CUtensorMap q, k, v;
    if (!make_map(&q, d.q, d.T, d.Hq, d.dh) || !make_map(&k, d.k, d.T, d.Hkv, d.dh) || !make_map(&v, d.v, d.T, d.Hkv, d.dh))
        return -2;
    if (!room(window_tc_fwd_kernel<DHP>, Fwd<DHP>::SMEM)) return -5;
    const long long blocks = tiles_of(d, 2 * kT) * d.Hq;
    if (blocks > 0x7fffffff) return -2;
    window_tc_fwd_kernel<DHP><<<(unsigned)blocks, kFwdThreads, Fwd<DHP>::SMEM, s>>>(q, k, v, d);
    return cudaGetLastError() == cudaSuccess ? 0 : -5;
}

template <int DHP>
int bwd(const WindowDesc& d, cudaStream_t s) {
    CUtensorMap q, k, v, g;
    if (!make_map(&q, d.q, d.T, d.Hq, d.dh) || !make_map(&k, d.k, d.T, d.Hkv, d.dh) || !make_map(&v, d.v, d.T, d.Hkv, d.dh) ||
        !make_map(&g, d.dout, d.T, d.Hq, d.dh))
        return -2;
    if (!room(window_tc_bwd_q_kernel<DHP>, BwdQ<DHP>::SMEM) || !room(window_tc_bwd_kv_kernel<DHP>, BwdKv<DHP>::SMEM))
        return -5;
    const long long tiles = tiles_of(d, kT);
    if (tiles * d.Hq > 0x7fffffff) return -2;
    window_tc_bwd_q_kernel<DHP><<<(unsigned)(tiles * d.Hq), kBwdQThreads, BwdQ<DHP>::SMEM, s>>>(q, k, v, g, d);
    window_tc_bwd_kv_kernel<DHP><<<(unsigned)(tiles * d.Hkv), kBwdKvThreads, BwdKv<DHP>::SMEM, s>>>(q, k, v, g, d);
    return cudaGetLastError() == cudaSuccess ? 0 : -5;
}

}  // namespace

bool attention_window_tc_supported(const WindowDesc& d) {
    return d.dtype == kBF16 && d.dh % 8 == 0 && d.dh <= 128 && rows16(d.q, d.T, d.Hq) && rows16(d.k, d.T, d.Hkv) &&
           rows16(d.v, d.T, d.Hkv) && rows16(d.out, d.T, d.Hq);
}

int attention_window_tc(const WindowDesc& d, cudaStream_t s) { return d.dh <= 64 ? fwd<64>(d, s) : fwd<128>(d, s); }

bool attention_window_bwd_tc_supported(const WindowDesc& d) {
    return attention_window_tc_supported(d) && rows16(d.dout, d.T, d.Hq) && rows16(d.dq, d.T, d.Hq) &&
           rows16(d.dk, d.T, d.Hkv) && rows16(d.dv, d.T, d.Hkv);
}

int attention_window_bwd_tc(const WindowDesc& d, cudaStream_t s) { return d.dh <= 64 ? bwd<64>(d, s) : bwd<128>(d, s); }

}  // namespace nsb
