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
#include "shared_memory.h"

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

// Waits of one block, a whole warp's: all of its lanes go on or none.
struct Waits {
    volatile int* failed;  // shared memory
    int* err;
    __device__ __forceinline__ bool operator()(uint64_t* bar, uint32_t phase) const {
        if (__all_sync(0xffffffffu, ptx::mbar_try_wait(bar, phase & 1))) return true;
        const long long t0 = clock64();
        while (!__all_sync(0xffffffffu, ptx::mbar_try_wait(bar, phase & 1))) {
            const bool late = clock64() - t0 > ptx::kWaitCycles;
            if (late) {
                *failed = 1;
                atomicCAS(err, 0, kErrTimeoutAttn);
            }
            if (__any_sync(0xffffffffu, late || *failed)) return false;
        }
        return true;
    }
};

// One lane of the warp (of all its lanes).
__device__ __forceinline__ bool elect() {
    uint32_t on;
    asm volatile(
        "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(on));
    return on;
}

// One arrival for a whole warp, behind what all of its lanes did.
__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) ptx::mbar_arrive(bar);
}

// A barrier of N threads, by whole warps: whether one of them gave up. Who leaves
// while the others will meet once more meets it with `gone`, and who gets true
// leaves without: so nobody stands at a barrier that another will not reach. Behind
// the last meeting of all a warp leaves by itself (and the flag ends the others'
// waits).
template <int N>
__device__ __forceinline__ bool meet(int id, bool gone) {
    int any;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.s32 p, %3, 0;\n\tbarrier.cta.red.or.pred q, %1, %2, p;\n\tselp.s32 %0, 1, 0, q;\n\t}"
        : "=r"(any)
        : "r"(id), "n"(N), "r"((int)gone)
        : "memory");
    return any;
}

// 128 rows of a head from row `row` on, 64 columns a chunk.
template <int DHP>
__device__ __forceinline__ void load_rows(uint8_t* to, const CUtensorMap* map, uint64_t* bar, int head, int row) {
    ptx::mbar_arrive_expect_tx(bar, DHP / 64 * kChunk);
#pragma unroll
    for (int c = 0; c < DHP / 64; c++) ptx::tma_load_3d(to + c * kChunk, map, bar, c * 64, head, row);
}

// Zeros in the rows of a tile from `from` on, by the warp that loads: what
// stands there belongs to another sequence or to none, and 0 times an infinity
// is no 0. Only a sequence's last tile has such rows.
template <int DHP>
__device__ __forceinline__ void zero_rows(uint8_t* tile, int from) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int c = 0; c < DHP / 64; c++)
        for (int at = from * 128 + lane * 16; at < kChunk; at += 512)
            *reinterpret_cast<uint4*>(tile + c * kChunk + at) = make_uint4(0, 0, 0, 0);
    ptx::fence_proxy_async();
}

// A tile into a slot of the ring, by the whole warp that loads; where rows from
// `end` on are to be zeros, the copy lands on a barrier of its own first.
template <int DHP>
__device__ __forceinline__ bool fill_slot(uint8_t* to, const CUtensorMap* map, uint64_t* full, uint64_t* landed, uint32_t& tails,
                                          const Waits& wait, int head, int row, int end) {
    const bool one = (threadIdx.x & 31) == 0;
    if (end >= kT) {
        if (one) load_rows<DHP>(to, map, full, head, row);
        return true;
    }
    if (one) load_rows<DHP>(to, map, landed, head, row);
    if (!wait(landed, tails)) {
        if (one) ptx::mbar_wait(landed, tails & 1, nullptr, 0);  // no copy may land after the block has left
        return false;
    }
    tails++;
    zero_rows<DHP>(to, end);
    warp_arrive(full);
    return true;
}

// A place in a ring of slots, and the phase of its barriers: it goes on by one
// or two without a division.
template <int SLOTS>
struct Turnstile {
    int slot = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ void skip(int n) {
        slot += n;
        if (slot >= SLOTS) {
            slot -= SLOTS;
            phase ^= 1;
        }
    }
};

// Descriptors of a tile at shared address `at`: K-major (its rows are the rows
// or columns of the product) and MN-major (its rows are summed over).
__device__ __forceinline__ uint64_t k_major(uint32_t at) { return ptx::smem_desc(at, 16, 1024, 2); }
__device__ __forceinline__ uint64_t mn_major(uint32_t at) { return ptx::smem_desc(at, kChunk, 1024, 2); }

// D = A B^T over the heads' columns, 16 a step, both K-major tiles.
template <int DHP>
__device__ __forceinline__ void mma_dot(uint32_t d, uint64_t a, uint64_t b) {
    constexpr uint32_t idesc = ptx::instr_desc(1, 0, 0, kT, kT);
#pragma unroll
    for (int s = 0; s < DHP / 16; s++) {
        const uint32_t at = ((s >> 2) * kChunk + (s & 3) * 32) >> 4;
        ptx::mma_bf16(d, a + at, b + at, idesc, s > 0);
    }
}
// D (+)= A B, A [128, 128] in TMEM, B an MN-major tile. A's columns, two bf16 in
// one of TMEM's, stand in runs of RUN columns that begin 2 RUN of TMEM's apart
// (RUN 128: side by side).
template <int DHP, int RUN>
__device__ __forceinline__ void mma_add(uint32_t d, uint32_t a, uint64_t b, bool more) {
    constexpr uint32_t idesc = ptx::instr_desc(1, 0, 1, kT, DHP);
#pragma unroll
    for (int s = 0; s < kT / 16; s++)
        ptx::mma_bf16_ts(d, a + 16 * s / RUN * RUN + 16 * s % RUN / 2, b + s * (2048 >> 4), idesc, more || s > 0);
}

// N columns of an output row, `cols` of which there are.
template <int N>
__device__ __forceinline__ void store_cols(__nv_bfloat16* to, const uint32_t* v, float mul, int cols) {
#pragma unroll
    for (int g = 0; g < N / 8; g++) {
        if (8 * g >= cols) break;
        uint4 pk;
        __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&pk);
#pragma unroll
        for (int e = 0; e < 4; e++)
            h[e] = __floats2bfloat162_rn(__uint_as_float(v[8 * g + 2 * e]) * mul, __uint_as_float(v[8 * g + 2 * e + 1]) * mul);
        *reinterpret_cast<uint4*>(to + 8 * g) = pk;
    }
}

// Bits 0 .. m - 1 of 32. Masks are words of bits: a test of a constant bit is
// one instruction a score, comparing columns took five (3200 cycles a tile of
// the queries' gradients in place of 1200 without a mask).
__device__ __forceinline__ uint32_t below(int m) { return m <= 0 ? 0u : m >= 32 ? ~0u : (1u << m) - 1; }
// Of 32 keys from j0 on those that query i sees.
__device__ __forceinline__ uint32_t keys_seen(const WindowDesc& d, int i, int j0) {
    const uint32_t hidden = d.window && i >= d.window ? below(i - d.window - j0 + 1) & ~below(d.sinks - j0) : 0u;
    return below(i - j0 + 1) & ~hidden;
}
// Of 32 queries from i0 on those that see key j (n: the sequence's rows).
__device__ __forceinline__ uint32_t queries_seeing(const WindowDesc& d, int j, int i0, int n) {
    const uint32_t past = d.window == 0 || d.window >= n || j < d.sinks ? 0u : ~below(j + d.window - i0);
    return ~below(j - i0) & ~past;
}
// Whether queries q0 .. q0 + 127 all see every key of the tile.
__device__ __forceinline__ bool all_seen(const WindowDesc& d, int q0, int k0) {
    return k0 + kT - 1 <= q0 && (d.window == 0 || q0 + kT - 1 - k0 < d.window || k0 + kT - 1 < d.sinks);
}

// ---------------------------------------------------------------------------
// Forward. A block has 256 neighbouring queries of one head, two tiles of 128:
//   warp 16    TMA: the queries, then keys and values tile by tile through a
//              ring of slots
//   warp 17    every MMA: S_g = Q_g K^T into TMEM columns [128 g, + 128),
//              O_g += P_g V into [256 + 128 g, ...), P_g (bf16) read from the
//              columns that held S_g. While one tile of queries is in its
//              softmax, the tensor cores run the other's products. (A warp for
//              each tile's products ran 8192 rows in 298 us in place of 240:
//              both then take turns on the tensor cores and end late.)
//   warps 8 g .. 8 g + 7   softmax of tile g, two threads a query with 64 keys
//              each, which exchange their maxima through shared memory (8192
//              rows: 242 us, a thread a query 243): the scores come from TMEM
//              into registers once, weights go back as bf16 pairs (off by 2^-9
//              of themselves at most; their fp32 sum is taken before). Weights in
//              two bf16, with a product of each, take 337 us in place of 244 and
//              leave outputs 1.6e-3 off in place of 2.1e-3, of which 1.6e-3 is
//              the rounding of outputs to bf16.
// O stays in TMEM. It is scaled only when a row's maximum rises by more than
// 2^8 above the one that its weights are taken against: smaller rises cost
// neither range (fp32) nor precision (the weights are floating point).
//
// Registers go from the warps that issue to those of the softmax, 64 and 104 a
// thread of 96 at launch (246 to 243 us).
//
// Bound by the turn from a product to its softmax and back: tensor cores and
// exponentials are each busy for 54 % of the time, and a tile's parts follow each
// other, overlapped by the other tile's alone. 8192 rows of 16 heads of 128
// columns, causal: 244 us, 1.13 PFLOP/s (0.68 of a measured library product);
// 20000 rows of 4 heads of 64, window 4000: 134 us.
// ---------------------------------------------------------------------------
constexpr int kFwdThreads = 640;  // (two of its warps idle: registers are split by groups of four)
constexpr float kRise = 8.f;

template <int DHP>
struct Fwd {
    static constexpr int TILE = DHP / 64 * kChunk;
    static constexpr int SLOTS = DHP == 128 ? 5 : 8;
    static constexpr int SMEM = (2 + SLOTS) * TILE + 4 * kT * 4 + 512;  // (no room to move its start)
    static_assert(SMEM <= 227 * 1024, "above what a block may have");
};

}  // namespace

template <int DHP>
__global__ void __launch_bounds__(kFwdThreads, 1)
    window_tc_fwd_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                         const __grid_constant__ CUtensorMap tv, const __grid_constant__ WindowDesc d) {
    using F = Fwd<DHP>;
    extern __shared__ __align__(1024) uint8_t smem[];
    if (ptx::smem_u32(smem) & 1023) {  // tiles begin on multiples of 1024
        if (threadIdx.x == 0) atomicCAS(d.err, 0, kErrBadShape);
        return;
    }
    uint8_t* ring = smem + 2 * F::TILE;
    float* tops = reinterpret_cast<float*>(ring + F::SLOTS * F::TILE);  // [2][2][128] of a group's halves
    uint64_t* q_full = reinterpret_cast<uint64_t*>(tops + 4 * kT);
    uint64_t* full = q_full + 1;
    uint64_t* empty = full + F::SLOTS;
    uint64_t* s_bar = empty + F::SLOTS;  // [2] scores of group g in TMEM
    uint64_t* p_bar = s_bar + 2;         // [2] weights of group g in TMEM (8 arrivals)
    uint64_t* o_bar = p_bar + 2;         // [2] product of group g added to O
    uint64_t* landed = o_bar + 2;        // a copy with rows to clear
    uint64_t* drain = landed + 1;
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
            ptx::mbar_init(&p_bar[g], 8);
            ptx::mbar_init(&o_bar[g], 1);
        }
        ptx::mbar_init(landed, 1);
        ptx::mbar_init(drain, 1);
        *failed = 0;
        ptx::fence_mbar_init();
    }
    if (warp == 17) {
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

    // (all four warps of a group at one instruction; together what the block was
    // launched with)
    if (warp >= 16) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        if (warp == 16) {
            const bool one = (t & 31) == 0;
            if (one) {
                ptx::mbar_arrive_expect_tx(q_full, (two ? 2 : 1) * F::TILE);
                for (int g = 0; g < (two ? 2 : 1); g++)
                    for (int c = 0; c < DHP / 64; c++)
                        ptx::tma_load_3d(smem + g * F::TILE + c * kChunk, &tq, q_full, c * 64, h, row0 + q0 + g * kT);
            }
            int it = 0;
            uint32_t tails = 0;
            for (int x = 0; x < tiles.count && ok; x++) {
                const int k0 = tiles.at(x) * kT;
                for (int kv = 0; kv < 2; kv++, it++) {
                    const int slot = it % F::SLOTS, round = it / F::SLOTS;
                    if (round && !(ok = wait(&empty[slot], round - 1))) break;
                    if (!(ok = fill_slot<DHP>(ring + slot * F::TILE, kv ? &tv : &tk, &full[slot], landed, tails, wait, hk,
                                              row0 + k0, kv ? w.n - k0 : kT)))
                        break;
                }
            }
            // no copy may land after the block has left
            if (one) {
                ptx::mbar_wait(q_full, 0, nullptr, 0);
                for (int i = max(0, it - F::SLOTS); i < it; i++)
                    ptx::mbar_wait(&full[i % F::SLOTS], (i / F::SLOTS) & 1, nullptr, 0);
            }
        } else if (warp == 17) {
            const uint32_t aQ = ptx::smem_u32(smem), aR = ptx::smem_u32(ring);
            uint32_t given[2] = {0, 0};  // weights taken, by group
            ok = wait(q_full, 0);
            for (int x = 0; x <= tiles.count && ok; x++) {
                const int ik = 2 * x, iv = 2 * x - 1;  // what the ring's slots hold: K0 V0 K1 V1 ...
                const int sk = ik % F::SLOTS, sv = iv > 0 ? iv % F::SLOTS : 0;
                const int kt = x < tiles.count ? tiles.at(x) : 0, before = x > 0 ? tiles.at(x - 1) : 0;
                if (x > 0 && !(ok = wait(&full[sv], iv / F::SLOTS))) break;
                if (x < tiles.count && !(ok = wait(&full[sk], ik / F::SLOTS))) break;
#pragma unroll
                for (int g = 0; g < 2; g++) {
                    if (x > 0 && uses(g, before)) {
                        if (!(ok = wait(&p_bar[g], given[g]))) break;
                        ptx::tc_fence_after();
                        if (elect()) {
                            mma_add<DHP, 64>(tmem + 256 + 128 * g, tmem + 128 * g, mn_major(aR + sv * F::TILE), given[g] > 0);
                            ptx::mma_commit(&o_bar[g]);
                        }
                        given[g]++;
                    }
                    if (x < tiles.count && uses(g, kt) && elect()) {
                        ptx::tc_fence_after();
                        mma_dot<DHP>(tmem + 128 * g, k_major(aQ + g * F::TILE), k_major(aR + sk * F::TILE));
                        ptx::mma_commit(&s_bar[g]);
                    }
                }
                if (ok && elect()) {
                    if (x > 0) ptx::mma_commit(&empty[sv]);
                    if (x < tiles.count) ptx::mma_commit(&empty[sk]);
                }
                __syncwarp();
            }
            if (elect()) {
                ptx::mma_commit(drain);
                ptx::mbar_wait(drain, 0, nullptr, 0);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
        if (warp < 8 || two) {
            const int g = warp >> 3, half = warp >> 2 & 1, lg = warp & 3, r = lg * 32 + (t & 31);
            const int i = q0 + g * kT + r;  // query of the sequence
            const uint32_t lanes = tmem + ((uint32_t)(lg * 32) << 16);
            const uint32_t base = lanes + 128 * g + 64 * half, o_at = lanes + 256 + 128 * g + half * (DHP / 2);
            const float sl2 = d.scale * kLog2e;
            float ref = -INFINITY, sum = 0.f;  // what the weights are taken against (powers of two), this half's sum
            uint32_t done = 0;                 // tiles behind
            // What the thread of this row's other half has. (It has read what was here
            // before: the scores that this thread waited for came after its weights.)
            auto swap = [&](float& v) {
                float* at = tops + g * 2 * kT;
                at[half * kT + r] = v;
                ok = !meet<64>(1 + g * 4 + lg, false);
                v = at[(half ^ 1) * kT + r];
                return ok;
            };
            auto await = [&](uint64_t* bar, uint32_t phase) {
                ok = wait(bar, phase);
                if (!ok) meet<64>(1 + g * 4 + lg, true);
                return ok;
            };
            for (int x = 0; x < tiles.count; x++) {
                const int kt = tiles.at(x), k0 = kt * kT;
                if (!uses(g, kt)) continue;
                if (!await(&s_bar[g], done)) break;
                ptx::tc_fence_after();
                uint32_t a[64];
                ptx::tmem_ld32(base, a);
                ptx::tmem_ld32(base + 32, a + 32);
                ptx::tmem_ld_wait_regs32(a);
                ptx::tmem_ld_wait_regs32(a + 32);
                if (!all_seen(d, q0 + g * kT, k0)) {
#pragma unroll
                    for (int c = 0; c < 64; c += 32) {
                        const uint32_t on = keys_seen(d, i, k0 + 64 * half + c);
#pragma unroll
                        for (int e = 0; e < 32; e++)
                            if (!(on >> e & 1)) a[c + e] = 0xff800000u;
                    }
                }
                float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < 64; c += 2)
                    m4[(c >> 1) & 3] = max3(m4[(c >> 1) & 3], __uint_as_float(a[c]), __uint_as_float(a[c + 1]));
                const float mine = fmaxf(max3(m4[0], m4[1], m4[2]), m4[3]);
                float top = mine;
                if (!swap(top)) break;
                top = fmaxf(top, mine) * sl2;  // (the scale is positive)
                const bool rise = top > ref + kRise;          // ref -inf: the first finite score
                if (__any_sync(0xffffffffu, rise)) {
                    const float turn = rise ? ex2(ref - top) : 1.f;
                    if (rise) ref = top;
                    sum *= turn;
                    if (done) {
                        if (!await(&o_bar[g], done - 1)) break;
                        ptx::tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < DHP / 2; c += 16) {
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
                uint64_t s4[2] = {0, 0};
#pragma unroll
                for (int c = 0; c < 64; c += 32) {
                    uint32_t pk[16];
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        float x0, x1;
                        f2_unpack(f2_fma(f2_pack(__uint_as_float(a[c + 2 * e]), __uint_as_float(a[c + 2 * e + 1])), SL2, NEG), x0, x1);
                        x0 = ex2(x0);
                        x1 = ex2(x1);
                        s4[e & 1] = f2_add(s4[e & 1], f2_pack(x0, x1));
                        const __nv_bfloat162 p = __floats2bfloat162_rn(x0, x1);
                        pk[e] = *reinterpret_cast<const uint32_t*>(&p);
                    }
                    ptx::tmem_st16(base + c / 2, pk);
                }
                float s0, s1;
                f2_unpack(f2_add(s4[0], s4[1]), s0, s1);
                sum += s0 + s1;
                ptx::tmem_st_wait();
                ptx::tc_fence_before();
                warp_arrive(&p_bar[g]);
                done++;
            }
            float rest = sum;
            if (ok && await(&o_bar[g], done - 1) && swap(rest)) {  // a query's own tile is always among its tiles
                ptx::tc_fence_after();
                sum += rest;
                const float mul = sum == 0.f ? 0.f : 1.f / sum;
                __nv_bfloat16* to = (__nv_bfloat16*)d.out.p + (w.row0 + i) * d.out.row + h * d.out.head;
#pragma unroll 1
                for (int c = 0; c < DHP / 2; c += 32) {
                    uint32_t v[32];
                    ptx::tmem_ld32(o_at + c, v);
                    ptx::tmem_ld_wait_regs32(v);
                    if (i < w.n) store_cols<32>(to + half * (DHP / 2) + c, v, mul, d.dh - half * (DHP / 2) - c);
                }
                if (half == 0 && i < w.n && d.lse)
                    d.lse[h * d.ld_lse + w.row0 + i] = sum == 0.f ? -INFINITY : (ref + log2f(sum)) * kLn2;
            }
        }
    }
    ptx::tc_fence_before();
    __syncthreads();
    if (warp == 17) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem, 512);
    }
}

// ---------------------------------------------------------------------------
// Gradient of the queries. A block has 128 queries of one head and walks the
// tiles of keys that they see:
//   warp 17    TMA: queries and dout, then keys and values through a ring
//   warp 16    the MMAs S = Q K^T into TMEM columns [0, 128) and
//              dP = dout V^T into [128, 256), a tile ahead of
//   warp 18    dQ += dS K into [256, ...), dS (bf16) read from [384, 448) and
//              [448, 512) in turn
//   warps 0..15   dS = P (dP - D), four threads a query with 32 keys each: their
//              registers hold both scores at once, and four warps a scheduler
//              hide each other's latencies. Before the first tile they form
//              D = rowdot(dout, out), which the second kernel reads too.
//
// Where few keys are seen (few_keys) a pass before sums dS, and D is corrected by
// that; it costs 2/3 of the block's time. Rounding dS to bf16 for the products
// remains (2^-9 of itself).
//
// Bound by the products' issue and turns: 8192 rows in 3 sequences, 16 heads of
// 128 columns, window 1024: 162 us, 0.52 PFLOP/s in S, dP and dQ.
// ---------------------------------------------------------------------------
constexpr int kBwdQThreads = 608;

template <int DHP>
struct BwdQ {
    static constexpr int TILE = DHP / 64 * kChunk;
    static constexpr int SLOTS = DHP == 128 ? 5 : 8;
    static constexpr int SMEM = (2 + SLOTS) * TILE + 4 * kT * 4 + 512;  // (no room to move its start)
    static_assert(SMEM <= 227 * 1024, "above what a block may have");
};

template <int DHP>
__global__ void __launch_bounds__(kBwdQThreads, 1)
    window_tc_bwd_q_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                           const __grid_constant__ CUtensorMap tv, const __grid_constant__ CUtensorMap tg,
                           const __grid_constant__ WindowDesc d) {
    using F = BwdQ<DHP>;
    extern __shared__ __align__(1024) uint8_t smem[];
    if (ptx::smem_u32(smem) & 1023) {  // tiles begin on multiples of 1024
        if (threadIdx.x == 0) atomicCAS(d.err, 0, kErrBadShape);
        return;
    }
    uint8_t* ring = smem + 2 * F::TILE;
    float* sums = reinterpret_cast<float*>(ring + F::SLOTS * F::TILE);  // [4][128] of a row's quarters
    uint64_t* q_full = reinterpret_cast<uint64_t*>(sums + 4 * kT);
    uint64_t* full = q_full + 1;
    uint64_t* empty = full + F::SLOTS;
    uint64_t* s_bar = empty + F::SLOTS;  // S and dP of a tile in TMEM
    uint64_t* r_bar = s_bar + 1;         // both read (16 arrivals)
    uint64_t* p_bar = r_bar + 1;         // dS in TMEM (16 arrivals)
    uint64_t* o_bar = p_bar + 1;         // [2] product added to dQ, of either dS
    uint64_t* landed = o_bar + 2;        // a copy with rows to clear
    uint64_t* drain = landed + 1;        // [2]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 2);
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
        ptx::mbar_init(r_bar, 16);
        ptx::mbar_init(p_bar, 16);
        ptx::mbar_init(&o_bar[0], 1);
        ptx::mbar_init(&o_bar[1], 1);
        ptx::mbar_init(landed, 1);
        ptx::mbar_init(&drain[0], 1);
        ptx::mbar_init(&drain[1], 1);
        *failed = 0;
        ptx::fence_mbar_init();
    }
    if (warp == 16) {
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
    const int first = few_keys(d, q0, min(q0 + kT, w.n)) ? tiles.count : 0;  // steps of the pass that only sums

    if (warp == 17) {
        const bool one = (t & 31) == 0;
        if (one) {
            ptx::mbar_arrive_expect_tx(q_full, 2 * F::TILE);
            for (int c = 0; c < DHP / 64; c++) {
                ptx::tma_load_3d(smem + c * kChunk, &tq, q_full, c * 64, h, row0 + q0);
                ptx::tma_load_3d(smem + F::TILE + c * kChunk, &tg, q_full, c * 64, h, row0 + q0);
            }
        }
        int it = 0;
        uint32_t tails = 0;
        for (int x = -first; x < tiles.count && ok; x++) {
            const int k0 = tiles.at(x < 0 ? x + first : x) * kT;
            for (int kv = 0; kv < 2; kv++, it++) {
                const int slot = it % F::SLOTS, round = it / F::SLOTS;
                if (round && !(ok = wait(&empty[slot], round - 1))) break;
                if (!(ok = fill_slot<DHP>(ring + slot * F::TILE, kv ? &tv : &tk, &full[slot], landed, tails, wait, hk,
                                          row0 + k0, kv ? kT : w.n - k0)))
                    break;
            }
        }
        if (one) {
            ptx::mbar_wait(q_full, 0, nullptr, 0);
            for (int i = max(0, it - F::SLOTS); i < it; i++)
                ptx::mbar_wait(&full[i % F::SLOTS], (i / F::SLOTS) & 1, nullptr, 0);
        }
    } else if (warp == 16) {
        const uint32_t aQ = ptx::smem_u32(smem), aG = aQ + F::TILE, aR = ptx::smem_u32(ring);
        Turnstile<F::SLOTS> ts;
        ok = wait(q_full, 0);
        auto both = [&](int step, bool keys) {  // keys: no other product reads them
            const int slot = ts.slot;
            const uint32_t k_at = aR + slot * F::TILE;
            if (!(ok = wait(&full[slot], ts.phase))) return;
            ts.skip(1);
            if (!(ok = wait(&full[ts.slot], ts.phase))) return;
            if (step > 0 && !(ok = wait(r_bar, step - 1))) return;
            ptx::tc_fence_after();
            if (elect()) {
                mma_dot<DHP>(tmem, k_major(aQ), k_major(k_at));
                mma_dot<DHP>(tmem + 128, k_major(aG), k_major(aR + ts.slot * F::TILE));
                ptx::mma_commit(s_bar);
                ptx::mma_commit(&empty[ts.slot]);
                if (keys) ptx::mma_commit(&empty[slot]);
            }
            __syncwarp();
            ts.skip(1);
        };
#pragma unroll 1
        for (int step = 0; step < first && ok; step++) both(step, true);
#pragma unroll 1
        for (int x = 0; x < tiles.count && ok; x++) both(first + x, false);
        if (elect()) {
            ptx::mma_commit(&drain[0]);
            ptx::mbar_wait(&drain[0], 0, nullptr, 0);
        }
    } else if (warp == 18) {
        const uint32_t aR = ptx::smem_u32(ring);
        Turnstile<F::SLOTS> ts;
        for (int x = 0; x < first; x++) ts.skip(2);
        for (int x = 0; x < tiles.count && ok; x++) {
            if (!(ok = wait(p_bar, x))) break;
            ptx::tc_fence_after();
            if (elect()) {
                mma_add<DHP, 128>(tmem + 256, tmem + 384 + 64 * (x & 1), mn_major(aR + ts.slot * F::TILE), x > 0);
                ptx::mma_commit(&o_bar[x & 1]);
                ptx::mma_commit(&empty[ts.slot]);
            }
            __syncwarp();
            ts.skip(2);
        }
        if (elect()) {
            ptx::mma_commit(&drain[1]);
            ptx::mbar_wait(&drain[1], 0, nullptr, 0);
        }
    } else {
        const int lg = warp & 3, part = warp >> 2, r = lg * 32 + (t & 31);
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
            for (int c = 0; c < DHP / 4; c += 8) {
                const int at = part * (DHP / 4) + c;
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
        // the sum of a row's four threads, in their order
        auto add_up = [&](float& v) {
            sums[part * kT + r] = v;
            ok = !meet<512>(1, false);
            v = ((sums[r] + sums[kT + r]) + sums[2 * kT + r]) + sums[3 * kT + r];
            return ok;
        };
        bool last = first == 0;  // whether all have met for the last time
        auto await = [&](uint64_t* bar, uint32_t phase) {
            ok = wait(bar, phase);
            if (!ok && !last) meet<512>(1, true);
            return ok;
        };
        add_up(D);
        const uint64_t SL2 = f2_pack(sl2, sl2), NEG = f2_pack(-lse2, -lse2);
        uint32_t a[32], g[32];
        auto gradients = [&](int step, int k0) {  // dS of the thread's 32 keys into g
            if (!await(s_bar, step)) return false;
            ptx::tc_fence_after();
            ptx::tmem_ld32(base + part * 32, a);
            ptx::tmem_ld32(base + 128 + part * 32, g);
            ptx::tmem_ld_wait_regs32(a);
            ptx::tmem_ld_wait_regs32(g);
            ptx::tc_fence_before();
            warp_arrive(r_bar);
            const uint64_t ND = f2_pack(-D, -D);
#pragma unroll
            for (int e = 0; e < 16; e++) {
                float x0, x1, y0, y1;
                f2_unpack(f2_fma(f2_pack(__uint_as_float(a[2 * e]), __uint_as_float(a[2 * e + 1])), SL2, NEG), x0, x1);
                f2_unpack(f2_mul(f2_pack(ex2(x0), ex2(x1)),
                                 f2_add(f2_pack(__uint_as_float(g[2 * e]), __uint_as_float(g[2 * e + 1])), ND)),
                          y0, y1);
                g[2 * e] = __float_as_uint(y0);
                g[2 * e + 1] = __float_as_uint(y1);
            }
            if (!all_seen(d, q0, k0)) {  // a hidden place is 0 whatever its dP is
                const uint32_t on = keys_seen(d, i, k0 + part * 32);
#pragma unroll
                for (int e = 0; e < 32; e++)
                    if (!(on >> e & 1)) g[e] = 0u;
            }
            return true;
        };
        if (first) {
            float rest = 0.f;  // sum of dS: what D is short of
#pragma unroll 1
            for (int x = 0; x < first && gradients(x, tiles.at(x) * kT); x++)
#pragma unroll
                for (int e = 0; e < 32; e++) rest += __uint_as_float(g[e]);
            ok = ok && !meet<512>(1, false);  // all have read the sums before
            if (ok && add_up(rest)) D += rest;
            last = true;
        }
        if (part == 0 && i < w.n) d.dvec[(long long)h * d.T + w.row0 + i] = D;
#pragma unroll 1
        for (int x = 0; x < tiles.count && ok && gradients(first + x, tiles.at(x) * kT); x++) {
            uint32_t pk[16];
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const __nv_bfloat162 p = __floats2bfloat162_rn(__uint_as_float(g[2 * e]), __uint_as_float(g[2 * e + 1]));
                pk[e] = *reinterpret_cast<const uint32_t*>(&p);
            }
            if (x > 1) {
                if (!await(&o_bar[x & 1], (x >> 1) - 1)) break;  // the product before the last has read its dS
                ptx::tc_fence_after();
            }
            ptx::tmem_st16(base + 384 + 64 * (x & 1) + part * 16, pk);
            ptx::tmem_st_wait();
            ptx::tc_fence_before();
            warp_arrive(p_bar);
        }
        const int end = tiles.count - 1;
        if (ok && await(&o_bar[end & 1], end >> 1)) {  // (the product before it was added before)
            ptx::tc_fence_after();
            __nv_bfloat16* to = (__nv_bfloat16*)d.dq.p + (w.row0 + i) * d.dq.row + h * d.dq.head;
            if constexpr (DHP == 128) {
                uint32_t v[32];
                ptx::tmem_ld32(base + 256 + part * 32, v);
                ptx::tmem_ld_wait_regs32(v);
                if (i < w.n) store_cols<32>(to + part * 32, v, d.scale, d.dh - part * 32);
            } else {
                uint32_t v[16];
                ptx::tmem_ld16(base + 256 + part * 16, v);
                ptx::tmem_ld_wait_regs16(v);
                if (i < w.n) store_cols<16>(to + part * 16, v, d.scale, d.dh - part * 16);
            }
        }
    }
    ptx::tc_fence_before();
    __syncthreads();
    if (warp == 16) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem, 512);
    }
}

// ---------------------------------------------------------------------------
// Gradients of keys and values. For 128 keys of one key head the tiles of
// queries, of all heads that share it, that see any of them are walked. How
// many these are differs by far (the first keys stay visible to all queries;
// without a window the last keys are seen by few), so all steps (a tile of
// keys with one of queries) of all tiles stand in one line that is cut into
// equal shares, one a block; a tile of keys that is cut leaves fp32 sums in
// the workspace, which a last kernel joins in the order of the blocks.
//
// The scores stand transposed, a key a row, so that both sums run over TMEM's
// columns:
//   warp 17    TMA: keys and values, then queries and dout through a ring
//   warp 18    lse and D of each tile of queries, into a ring of their own
//   warp 16    the MMAs S^T = K Q^T into TMEM columns [0, 128) and
//              dV += P^T dout into [256, ...),
//   warp 19    dP^T = V dout^T into [128, 256) and dK += dS^T Q into [384, ...).
//              P^T and dS^T (bf16) take the columns of the scores that they
//              come from.
//   warps 0..15   P and dS, four threads a key with 32 queries each: while P is
//              computed the tensor cores run dK and the next dP, while dS is,
//              dV and the next S. P and dS are off by 2^-9 of themselves at most.
//
// Bound as the queries' gradient is, with one product more: 8192 rows in 3
// sequences, 16 heads of 128 columns on 4 key heads, window 1024: 177 us,
// 0.63 PFLOP/s, and 18 us to join the cut tiles; 20000 rows of 4 heads of 64 on
// one, window 4000: 237 us and 9.
// ---------------------------------------------------------------------------
constexpr int kBwdKvThreads = 640;
constexpr int kStats = 4;      // tiles of lse and D held
constexpr int kMinSteps = 4;   // least steps a block: cutting a tile costs about two

template <int DHP>
struct BwdKv {
    static constexpr int TILE = DHP / 64 * kChunk;
    static constexpr int SLOTS = DHP == 128 ? 4 : 8;
    static constexpr int SMEM = (2 + SLOTS) * TILE + kStats * 2 * kT * 4 + 512 + 1024;
};

// Steps of a sequence, of one query head: tile t of nt has
// min(nt - t, reach), the `front` first nt - t.
struct Steps {
    long long nt, front, reach;
    __device__ __forceinline__ Steps(const WindowDesc& d, int n) {
        nt = (n + kT - 1) / kT;
        front = d.window ? min(nt, (long long)d.sinks / kT + (d.sinks % kT != 0)) : nt;
        reach = ((long long)d.window + 2 * kT - 2) / kT;
    }
    __device__ __forceinline__ long long of(int t) const { return t < front ? nt - t : min(nt - t, reach); }
    // those of the tiles before t
    __device__ __forceinline__ long long before(long long t) const {
        const long long f = min(t, front), s = f * nt - f * (f - 1) / 2;
        if (t <= front) return s;
        const long long u = nt - front, v = nt - t;  // tiles behind the front, and from t on: their steps v, v - 1 .. 1, or reach
        auto tail = [&](long long k) { return k <= reach ? k * (k + 1) / 2 : reach * (reach + 1) / 2 + (k - reach) * reach; };
        return s + tail(u) - tail(v);
    }
    __device__ __forceinline__ long long all() const { return before(nt); }
};

// The sequence b with its rows and the steps of one query head before it.
struct Seq {
    int row0, n;
    long long before;
};
// The first sequence for which less(steps up to its end, tiles up to its end)
// no longer holds; `all` receives the steps of every sequence where none is
// found. By whole warps.
template <typename F>
__device__ __forceinline__ bool find_seq(const WindowDesc& d, Seq* out, long long* tiles, long long* all, F past) {
    const int lane = threadIdx.x & 31;
    long long steps = 0, rows = 0;
    for (int b0 = 0; b0 < d.B; b0 += 32) {
        int lo = 0, n = 0;
        if (b0 + lane < d.B) {
            lo = d.offsets ? min(max(d.offsets[b0 + lane], 0), d.T) : 0;
            n = d.offsets ? min(max(d.offsets[b0 + lane + 1], lo), d.T) - lo : d.T;
        }
        const long long own = Steps(d, n).all(), nt = (n + kT - 1) / kT;
        long long s = own, r = nt;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long u = __shfl_up_sync(0xffffffffu, s, o), v = __shfl_up_sync(0xffffffffu, r, o);
            if (lane >= o) s += u, r += v;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, past(steps + s, rows + r));
        if (hit) {
            const int src = __ffs(hit) - 1;
            *out = Seq{__shfl_sync(0xffffffffu, lo, src), __shfl_sync(0xffffffffu, n, src),
                       steps + __shfl_sync(0xffffffffu, s - own, src)};
            *tiles = rows + __shfl_sync(0xffffffffu, r - nt, src);
            return true;
        }
        steps += __shfl_sync(0xffffffffu, s, 31);
        rows += __shfl_sync(0xffffffffu, r, 31);
    }
    *all = steps;
    return false;
}
// Steps of all heads, and a block's share of them.
__device__ __forceinline__ long long all_steps(const WindowDesc& d) {
    Seq q;
    long long tiles, all = 0;
    find_seq(d, &q, &tiles, &all, [](long long, long long) { return false; });
    return all * d.Hq;
}
__device__ __forceinline__ long long quotient(long long a, long long b) {  // (64 bits take a hundred instructions)
    return a < 0x7fffffff && b < 0x7fffffff ? (int)a / (int)b : a / b;
}
__device__ __forceinline__ long long share(long long all, int blocks) {
    return max((long long)kMinSteps, quotient(all + blocks - 1, blocks));
}

// A piece of a block's share: steps [x0, x1) of `count` of one tile of keys.
struct Piece {
    int row0, n, k0, hk;
    int first, each;  // first tile of queries, and how many a head
    int x0, x1, count;
};
__device__ __forceinline__ Piece piece_at(const WindowDesc& d, long long at, long long end) {
    Seq q{0, 0, 0};
    long long tiles, all;
    const int group = d.Hq / d.Hkv;
    find_seq(d, &q, &tiles, &all, [&](long long steps, long long) { return steps * d.Hq > at; });
    const Steps s(d, q.n);
    long long rest = at - q.before * d.Hq;
    const long long head = s.all() * group;
    Piece p;
    p.row0 = q.row0;
    p.n = q.n;
    p.hk = (int)quotient(rest, head);
    rest -= p.hk * head;
    int t = 0;  // the last tile whose steps begin at or before `rest`
    for (int step = 1 << 24; step; step >>= 1)
        if (t + step < s.nt && s.before(t + step) * group <= rest) t += step;
    p.k0 = t * kT;
    p.first = t;
    p.each = (int)s.of(t);
    p.count = p.each * group;
    p.x0 = (int)(rest - s.before(t) * group);
    p.x1 = (int)min((long long)p.count, p.x0 + (end - at));
    return p;
}

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
    uint64_t* k_empty = k_full + 1;        // read by the last scores of a piece, which all other warps have begun
    uint64_t* full = k_empty + 1;
    uint64_t* empty = full + F::SLOTS;
    uint64_t* st_full = empty + F::SLOTS;
    uint64_t* st_empty = st_full + kStats; // (16 arrivals)
    uint64_t* s_bar = st_empty + kStats;   // S^T in TMEM
    uint64_t* g_bar = s_bar + 1;           // dP^T in TMEM
    uint64_t* p_bar = g_bar + 1;           // P^T in TMEM (16 arrivals)
    uint64_t* ds_bar = p_bar + 1;          // dS^T in TMEM (16 arrivals)
    uint64_t* sum_bar = ds_bar + 1;        // a piece's sums in TMEM
    uint64_t* out_bar = sum_bar + 1;       // and read (16 arrivals)
    uint64_t* landed = out_bar + 1;        // a copy with rows to clear
    uint64_t* drain = landed + 1;          // [2]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 2);
    int* failed = reinterpret_cast<int*>(tmem_slot + 1);
    Piece* pieces = reinterpret_cast<Piece*>(failed + 1);  // [2], written with a piece's keys

    const int t = threadIdx.x, warp = t >> 5;
    const int group = d.Hq / d.Hkv;
    const long long all = all_steps(d), per = share(all, gridDim.x);
    const long long begin = blockIdx.x * per, end = min(all, begin + per);
    if (begin >= end) return;

    if (t == 0) {
        ptx::mbar_init(k_full, 1);
        ptx::mbar_init(k_empty, 2 + 17);
        for (int i = 0; i < F::SLOTS; i++) {
            ptx::mbar_init(&full[i], 1);
            ptx::mbar_init(&empty[i], 1 + (i & 1));  // dout, in the odd slots, has two readers
        }
        for (int i = 0; i < kStats; i++) {
            ptx::mbar_init(&st_full[i], 1);
            ptx::mbar_init(&st_empty[i], 16);
        }
        ptx::mbar_init(s_bar, 1);
        ptx::mbar_init(g_bar, 1);
        ptx::mbar_init(p_bar, 16);
        ptx::mbar_init(ds_bar, 16);
        ptx::mbar_init(sum_bar, 2);
        ptx::mbar_init(out_bar, 16);
        ptx::mbar_init(landed, 1);
        ptx::mbar_init(&drain[0], 1);
        ptx::mbar_init(&drain[1], 1);
        *failed = 0;
        ptx::fence_mbar_init();
    }
    if (warp == 16) {
        ptx::tmem_alloc(tmem_slot, 512);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const Waits wait{failed, d.err};
    bool ok = true;
    // step: counted over all pieces; piece: likewise
    int step = 0, piece = 0;

    // the next piece, once its keys are there; its steps go through the heads, and
    // the tiles of queries of each
    auto next_piece = [&](Piece& p) {
        ok = wait(k_full, piece);
        if (ok) p = pieces[piece & 1];
        return ok;
    };
    if (warp == 17) {
        const bool one = (t & 31) == 0;
        int keys = 0, copies = 0;  // loads started
        uint32_t tails = 0;
        for (long long at = begin; at < end && ok; piece++) {
            const Piece p = piece_at(d, at, end);
            at += p.x1 - p.x0;
            if (piece && !(ok = wait(k_empty, piece - 1))) break;
            keys = piece + 1;
            if (one) {
                pieces[piece & 1] = p;
                ptx::mbar_arrive_expect_tx(k_full, 2 * F::TILE);
                for (int c = 0; c < DHP / 64; c++) {
                    ptx::tma_load_3d(smem + c * kChunk, &tk, k_full, c * 64, p.hk, p.row0 + p.k0);
                    ptx::tma_load_3d(smem + F::TILE + c * kChunk, &tv, k_full, c * 64, p.hk, p.row0 + p.k0);
                }
            }
            int h = p.hk * group + p.x0 / p.each, q = p.x0 % p.each;
            for (int x = p.x0; x < p.x1 && ok; x++, step++) {
                const int q0 = (p.first + q) * kT;
                for (int qg = 0; qg < 2; qg++) {
                    const int i = 2 * step + qg, slot = i % F::SLOTS, round = i / F::SLOTS;
                    if (round && !(ok = wait(&empty[slot], round - 1))) break;
                    if (!(ok = fill_slot<DHP>(ring + slot * F::TILE, qg ? &tg : &tq, &full[slot], landed, tails, wait, h,
                                              p.row0 + q0, p.n - q0)))
                        break;
                    copies = i + 1;
                }
                if (++q == p.each) q = 0, h++;
            }
        }
        // no copy may land after the block has left
        if (one) {
            if (keys) ptx::mbar_wait(k_full, (keys - 1) & 1, nullptr, 0);
            for (int i = max(0, copies - F::SLOTS); i < copies; i++)
                ptx::mbar_wait(&full[i % F::SLOTS], (i / F::SLOTS) & 1, nullptr, 0);
        }
    } else if (warp == 18) {
        Piece p;
        for (long long at = begin; at < end && next_piece(p); piece++) {
            warp_arrive(k_empty);
            at += p.x1 - p.x0;
            int h = p.hk * group + p.x0 / p.each, q = p.x0 % p.each;
            for (int x = p.x0; x < p.x1; x++, step++) {
                const int slot = step % kStats, q0 = (p.first + q) * kT;
                float l[4], D[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int i = q0 + (t & 31) + 32 * e;
                    // (both negated.) A query that saw nothing, or is none, has weights of 0
                    l[e] = -INFINITY;
                    D[e] = 0.f;
                    if (i < p.n) {
                        const float lse = d.lse[h * d.ld_lse + p.row0 + i];
                        if (lse != -INFINITY) l[e] = -lse * kLog2e;
                        D[e] = -d.dvec[(long long)h * d.T + p.row0 + i];
                    }
                }
                if (step >= kStats && !(ok = wait(&st_empty[slot], step / kStats - 1))) break;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    stats[slot * 2 * kT + (t & 31) + 32 * e] = l[e];
                    stats[slot * 2 * kT + kT + (t & 31) + 32 * e] = D[e];
                }
                warp_arrive(&st_full[slot]);
                if (++q == p.each) q = 0, h++;
            }
            if (!ok) break;
        }
    } else if (warp == 16) {
        const uint32_t aK = ptx::smem_u32(smem), aR = ptx::smem_u32(ring);
        Turnstile<F::SLOTS> ts;  // queries of the next scores; their dout is one further
        Piece p;
        for (long long at = begin; at < end && next_piece(p); piece++) {
            at += p.x1 - p.x0;
            if (!(ok = wait(&full[ts.slot], ts.phase))) break;
            ptx::tc_fence_after();
            if (elect()) {
                mma_dot<DHP>(tmem, k_major(aK), k_major(aR + ts.slot * F::TILE));
                ptx::mma_commit(s_bar);
                if (p.x1 - p.x0 == 1) ptx::mma_commit(k_empty);
            }
            __syncwarp();
            for (int x = p.x0; x < p.x1; x++, step++) {
                const int more = p.x1 - 1 - x;
                ts.skip(1);
                const int g_slot = ts.slot;
                if (!(ok = wait(&full[g_slot], ts.phase))) break;
                ts.skip(1);
                if (more && !(ok = wait(&full[ts.slot], ts.phase))) break;
                // the piece before has been read out of the sums
                if (x == p.x0 && piece && !(ok = wait(out_bar, piece - 1))) break;
                if (!(ok = wait(p_bar, step))) break;
                ptx::tc_fence_after();
                if (elect()) {
                    mma_add<DHP, 32>(tmem + 256, tmem, mn_major(aR + g_slot * F::TILE), x > p.x0);
                    if (more) {
                        mma_dot<DHP>(tmem, k_major(aK), k_major(aR + ts.slot * F::TILE));
                        ptx::mma_commit(s_bar);
                        if (more == 1) ptx::mma_commit(k_empty);
                    } else {
                        ptx::mma_commit(sum_bar);
                    }
                    ptx::mma_commit(&empty[g_slot]);
                }
                __syncwarp();
            }
            if (!ok) break;
        }
        if (elect()) {
            ptx::mma_commit(&drain[0]);
            ptx::mbar_wait(&drain[0], 0, nullptr, 0);
        }
    } else if (warp == 19) {
        const uint32_t aV = ptx::smem_u32(smem) + F::TILE, aR = ptx::smem_u32(ring);
        Turnstile<F::SLOTS> ts;  // queries of the step whose dS is awaited
        Piece p;
        for (long long at = begin; at < end && next_piece(p); piece++) {
            at += p.x1 - p.x0;
            Turnstile<F::SLOTS> next = ts;  // dout of the next scores
            next.skip(1);
            if (!(ok = wait(&full[next.slot], next.phase))) break;
            ptx::tc_fence_after();
            if (elect()) {
                mma_dot<DHP>(tmem + 128, k_major(aV), k_major(aR + next.slot * F::TILE));
                ptx::mma_commit(g_bar);
                ptx::mma_commit(&empty[next.slot]);
                if (p.x1 - p.x0 == 1) ptx::mma_commit(k_empty);
            }
            __syncwarp();
            for (int x = p.x0; x < p.x1; x++, step++) {
                const int more = p.x1 - 1 - x;
                next.skip(2);
                if (more && !(ok = wait(&full[next.slot], next.phase))) break;
                if (x == p.x0 && piece && !(ok = wait(out_bar, piece - 1))) break;
                if (!(ok = wait(ds_bar, step))) break;
                ptx::tc_fence_after();
                if (elect()) {
                    mma_add<DHP, 32>(tmem + 384, tmem + 128, mn_major(aR + ts.slot * F::TILE), x > p.x0);
                    if (more) {
                        mma_dot<DHP>(tmem + 128, k_major(aV), k_major(aR + next.slot * F::TILE));
                        ptx::mma_commit(g_bar);
                        ptx::mma_commit(&empty[next.slot]);
                        if (more == 1) ptx::mma_commit(k_empty);
                    } else {
                        ptx::mma_commit(sum_bar);
                    }
                    ptx::mma_commit(&empty[ts.slot]);
                }
                __syncwarp();
                ts.skip(2);
            }
            if (!ok) break;
        }
        if (elect()) {
            ptx::mma_commit(&drain[1]);
            ptx::mbar_wait(&drain[1], 0, nullptr, 0);
        }
    } else {
        const int lg = warp & 3, part = warp >> 2;
        const uint32_t row = tmem + ((uint32_t)(lg * 32) << 16), base = row + 32 * part;
        const float sl2 = d.scale * kLog2e;
        const uint64_t SL2 = f2_pack(sl2, sl2);
        Piece p;
        for (long long at = begin; at < end && next_piece(p); piece++) {
            warp_arrive(k_empty);
            const int slot_of_part = at == begin ? 0 : 1;
            at += p.x1 - p.x0;
            int q = p.x0 % p.each;
            const int j = p.k0 + lg * 32 + (t & 31);  // key of the sequence
            for (int x = p.x0; x < p.x1; x++, step++) {
                const int slot = step % kStats, q0 = (p.first + q) * kT;
                if (++q == p.each) q = 0;
                const float4* l4 = reinterpret_cast<const float4*>(stats + slot * 2 * kT + part * 32);
                const float4* d4 = l4 + kT / 4;
                if (!(ok = wait(&st_full[slot], step / kStats) && wait(s_bar, step))) break;
                ptx::tc_fence_after();
                uint32_t a[32], g[32], pk[16];
                ptx::tmem_ld32(base, a);
                ptx::tmem_ld_wait_regs32(a);
#pragma unroll
                for (int e = 0; e < 16; e += 2) {
                    const float4 l = l4[e / 2];
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        const int c = 2 * (e + u);
                        float x0, x1;
                        f2_unpack(f2_fma(f2_pack(__uint_as_float(a[c]), __uint_as_float(a[c + 1])), SL2,
                                         u ? f2_pack(l.z, l.w) : f2_pack(l.x, l.y)),
                                  x0, x1);
                        a[c] = __float_as_uint(ex2(x0));
                        a[c + 1] = __float_as_uint(ex2(x1));
                    }
                }
                if (!all_seen(d, q0, p.k0)) {
                    const uint32_t on = queries_seeing(d, j, q0 + part * 32, p.n);
#pragma unroll
                    for (int e = 0; e < 32; e++)
                        if (!(on >> e & 1)) a[e] = 0u;
                }
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const __nv_bfloat162 h2 = __floats2bfloat162_rn(__uint_as_float(a[2 * e]), __uint_as_float(a[2 * e + 1]));
                    pk[e] = *reinterpret_cast<const uint32_t*>(&h2);
                }
                ptx::tmem_st16(base, pk);
                ptx::tmem_st_wait();
                ptx::tc_fence_before();
                warp_arrive(p_bar);
                if (!(ok = wait(g_bar, step))) break;
                ptx::tc_fence_after();
                ptx::tmem_ld32(base + 128, g);
                ptx::tmem_ld_wait_regs32(g);
#pragma unroll
                for (int e = 0; e < 16; e += 2) {
                    const float4 D = d4[e / 2];
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        const int c = 2 * (e + u);
                        float y0, y1;
                        f2_unpack(f2_mul(f2_pack(__uint_as_float(a[c]), __uint_as_float(a[c + 1])),
                                         f2_add(u ? f2_pack(D.z, D.w) : f2_pack(D.x, D.y),
                                                f2_pack(__uint_as_float(g[c]), __uint_as_float(g[c + 1])))),
                                  y0, y1);
                        const __nv_bfloat162 h2 = __floats2bfloat162_rn(y0, y1);
                        pk[e + u] = *reinterpret_cast<const uint32_t*>(&h2);
                    }
                }
                ptx::tmem_st16(base + 128, pk);
                ptx::tmem_st_wait();
                ptx::tc_fence_before();
                warp_arrive(ds_bar);
                warp_arrive(&st_empty[slot]);
            }
            if (!ok || !(ok = wait(sum_bar, piece))) break;
            ptx::tc_fence_after();
            const bool alone = p.x1 - p.x0 == p.count;
            __nv_bfloat16* dv = (__nv_bfloat16*)d.dv.p + (p.row0 + j) * d.dv.row + p.hk * d.dv.head;
            __nv_bfloat16* dk = (__nv_bfloat16*)d.dk.p + (p.row0 + j) * d.dk.row + p.hk * d.dk.head;
            // [dv | dk][column][key]
            float* rest = d.parts + ((long long)blockIdx.x * 2 + slot_of_part) * (2 * DHP * kT) + lg * 32 + (t & 31);
#pragma unroll 1
            for (int c = part * (DHP / 4); c < (part + 1) * (DHP / 4); c += 16) {
                uint32_t v[16], k[16];
                ptx::tmem_ld16(row + 256 + c, v);
                ptx::tmem_ld16(row + 384 + c, k);
                ptx::tmem_ld_wait_regs16(v);
                ptx::tmem_ld_wait_regs16(k);
                if (!alone) {
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        rest[(c + e) * kT] = __uint_as_float(v[e]);
                        rest[(DHP + c + e) * kT] = __uint_as_float(k[e]);
                    }
                } else if (j < p.n) {
                    store_cols<16>(dv + c, v, 1.f, d.dh - c);
                    store_cols<16>(dk + c, k, d.scale, d.dh - c);
                }
            }
            ptx::tc_fence_before();
            warp_arrive(out_bar);
        }
    }
    ptx::tc_fence_before();
    __syncthreads();
    if (warp == 16) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem, 512);
    }
}

// Joins the sums of a tile of keys that several blocks share, block after
// block: eight columns of a key's dv or dk a thread. grid (tiles of keys, Hkv,
// shares of the columns).
template <int DHP>
__global__ void __launch_bounds__(256) window_tc_join_kernel(const __grid_constant__ WindowDesc d, int blocks) {
    const int group = d.Hq / d.Hkv, hk = blockIdx.y;
    const long long per = share(all_steps(d), blocks);
    Seq q;
    long long tiles, all;
    if (!find_seq(d, &q, &tiles, &all, [&](long long, long long r) { return r > (long long)blockIdx.x; })) return;
    const Steps s(d, q.n);
    const int t = (int)(blockIdx.x - tiles);
    const long long from = q.before * d.Hq + hk * s.all() * group + s.before(t) * group, to = from + s.of(t) * group;
    const int c0 = (int)quotient(from, per), c1 = (int)quotient(to - 1, per);
    if (c0 == c1) return;
    const int r = threadIdx.x & (kT - 1), which = threadIdx.x / kT, j = t * kT + r;
    if (j >= q.n) return;
    constexpr long long kPart = 2 * DHP * kT;
    const Heads& x = which ? d.dk : d.dv;
    const float mul = which ? d.scale : 1.f;
    for (int c = blockIdx.z * 8; c < d.dh; c += gridDim.z * 8) {
        const float* parts = d.parts + (which * DHP + c) * kT + r;
        const float* first = parts + ((long long)c0 * 2 + (from != c0 * per ? 1 : 0)) * kPart;
        float sum[8];
#pragma unroll
        for (int e = 0; e < 8; e++) sum[e] = first[e * kT];
#pragma unroll 4
        for (int b = c0 + 1; b <= c1; b++)
#pragma unroll
            for (int e = 0; e < 8; e++) sum[e] += parts[b * 2 * kPart + e * kT];
        uint4 pk;
        __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&pk);
#pragma unroll
        for (int e = 0; e < 4; e++) h[e] = __floats2bfloat162_rn(sum[2 * e] * mul, sum[2 * e + 1] * mul);
        *reinterpret_cast<uint4*>((__nv_bfloat16*)x.p + (q.row0 + j) * x.row + hk * x.head + c) = pk;
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

long long tiles_of(const WindowDesc& d, int rows) { return ((long long)d.T + rows - 1) / rows + (d.offsets ? d.B : 0); }

template <int DHP>
int fwd(const WindowDesc& d, cudaStream_t s) {
    CUtensorMap q, k, v;
    if (!make_map(&q, d.q, d.T, d.Hq, d.dh) || !make_map(&k, d.k, d.T, d.Hkv, d.dh) || !make_map(&v, d.v, d.T, d.Hkv, d.dh))
        return -2;
    static size_t most[kMaxDevices];
    if (!allow_shared(window_tc_fwd_kernel<DHP>, Fwd<DHP>::SMEM, most)) return -5;
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
    static size_t most_q[kMaxDevices], most_kv[kMaxDevices];
    if (!allow_shared(window_tc_bwd_q_kernel<DHP>, BwdQ<DHP>::SMEM, most_q) ||
        !allow_shared(window_tc_bwd_kv_kernel<DHP>, BwdKv<DHP>::SMEM, most_kv))
        return -5;
    const long long tiles = tiles_of(d, kT);
    if (tiles * d.Hq > 0x7fffffff) return -2;
    const int blocks = num_sms();
    window_tc_bwd_q_kernel<DHP><<<(unsigned)(tiles * d.Hq), kBwdQThreads, BwdQ<DHP>::SMEM, s>>>(q, k, v, g, d);
    window_tc_bwd_kv_kernel<DHP><<<blocks, kBwdKvThreads, BwdKv<DHP>::SMEM, s>>>(q, k, v, g, d);
    window_tc_join_kernel<DHP><<<dim3((unsigned)tiles, d.Hkv, 4), 256, 0, s>>>(d, blocks);
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

// Two pieces of each block may be cut: [dv | dk][columns][128 keys] of each.
size_t attention_window_bwd_tc_parts(int dh) {
    return (size_t)num_sms() * 2 * 2 * (dh <= 64 ? 64 : 128) * kT * sizeof(float);
}

int attention_window_bwd_tc(const WindowDesc& d, cudaStream_t s) { return d.dh <= 64 ? bwd<64>(d, s) : bwd<128>(d, s); }

}  // namespace nsb
