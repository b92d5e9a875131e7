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

// Waits of one block: what fails, and whether any role has.
struct Waits {
    volatile int* failed;  // shared memory
    int* err;
    __device__ __forceinline__ bool operator()(uint64_t* bar, uint32_t phase) const {
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
                    if (round && !(ok = wait(&empty[slot], round - 1))) break;
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

}  // namespace

bool attention_window_tc_supported(const WindowDesc& d) {
    return d.dtype == kBF16 && d.dh % 8 == 0 && d.dh <= 128 && rows16(d.q, d.T, d.Hq) && rows16(d.k, d.T, d.Hkv) &&
           rows16(d.v, d.T, d.Hkv) && rows16(d.out, d.T, d.Hq);
}

int attention_window_tc(const WindowDesc& d, cudaStream_t s) { return d.dh <= 64 ? fwd<64>(d, s) : fwd<128>(d, s); }

}  // namespace nsb
