// Products of 8-bit floating point codes with a scale for each block of 128
// (no counterpart in the reference):
//
//   C[m,n] = sum over blocks b of 128 k of  sa(m,b) sb(n,b) sum_k A[m,k] B[n,k]
//
// The tensor cores sum a block's 128 exact products in fp32 (tcgen05
// kind::f8f6f4, accumulators in TMEM); the scales vary from block to block, so
// every block's sum is read back from TMEM, scaled and added to an fp32
// accumulator in registers, while the tensor cores work on the next block in
// another part of TMEM.
#include <cuda.h>
#include <cuda_fp8.h>
#include <string.h>

#include <mutex>

#include "fp8.h"
#include "gemm.h"
#include "ptx.cuh"

namespace nsb {

namespace {

// ---------------------------------------------------------------------------
// 128 x BN tiles, one persistent CTA an SM
//   warps 0, 3   copy: A and B by TMA into a ring of stages (128 x 128 codes
//                of A, BN x 128 of B, 128-byte swizzle), the k-blocks' scales
//                into a ring of their own, deep enough to cover a read from
//                DRAM; with a row list the rows of A by 16-byte cp.async in
//                the swizzled order (TMA's four-row gather took 2700 cycles
//                for 128 rows)
//   warps 1, 2   MMA issuers, each one's k-blocks' products into parts of TMEM
//                of its own: while one is held up by the tensor cores' queue
//                or waits for a part, the other's products run
//   warps 4..11  a warp owns 32 rows and half the columns: scales and adds
//                every k-block's part, stores the tile
// The scaling bounds it: a k-block of 128 x 256 takes the tensor cores 512
// cycles and the eight warps about 1080, in which each issues some 220
// instructions, 64 of them packed FMAs. 8192 x 4096 x 4096 into bf16: 133 us,
// 2.07 PFLOP/s; under the power cap 155 to 160. In copies of the kernel: 131 us
// with the FMAs but no reads of TMEM, 116 with the reads alone, 108 with
// neither, where 84 would be the tensor cores' (at twice the bf16 rate); what
// holds the 108 is not known.
// The accumulators of a 128 x 256 tile are 128 registers a thread, so the
// first four warps give theirs up: 72 + 2 * 216 of the 3 * 168 registers that
// the three warpgroups are launched with.
// ---------------------------------------------------------------------------
struct TileParams {
    int M, N, K;
    const uint8_t* a;
    long long lda;
    int a_rows;
    const float* sa;
    long long ld_sa;
    const float* sb;
    long long ld_sb, sb_stride;
    void* c;
    int c_dtype;
    long long ldc, c_stride;
    int groups;  // row groups (ROWS) or k groups; 0: one product
    const int* offsets;
    const int* counts;
    const int* rows;
    int row_div;
    int m_tiles, n_tiles, nb;  // nb: 128-wide scale blocks along N
    int split;                 // CTAs of a cluster that share a tile's k-blocks
    int tma_out, vec_out;
    int* err;
};

constexpr int kBand = 16;  // n tiles whose m tiles run together
constexpr int kEpi = 8;
constexpr int kThreads = 128 + 32 * kEpi;
constexpr int kMaxGroups = 1024;
constexpr int kSlots = 4;  // groups of k-blocks whose scales are in flight

template <int BN, bool VEC, bool ROWS, bool PAIR>
struct TileCfg {
    static constexpr int BM = PAIR ? 256 : 128;       // rows of a tile
    static constexpr int BROWS = PAIR ? BN / 2 : BN;  // rows of B that this CTA loads
    static_assert(!PAIR || (!VEC && !ROWS), "pairs take one product with block scales");
    static_assert(BN == 128 || BN == 256 || (BN == 192 && VEC), "a warp's columns lie in one scale block");
    static constexpr int A_BYTES = 128 * 128;
    static constexpr int STAGE = A_BYTES + BROWS * 128;
    static constexpr int STAGES = BROWS == 128 ? 6 : 4;
    static constexpr int PCOLS = BN == 128 ? 128 : 256;  // columns of a part of TMEM
    static constexpr int PARTS = 512 / PCOLS;
    static constexpr int COLS = BN / 2;      // columns of a warp
    static constexpr int STAGING = kEpi * 2048;  // 32 rows x 64 bytes a warp
    static constexpr int SLOT = 128 + (VEC ? BN : 4);  // a k-block's row scales, then column or block scales
    static constexpr int SLOTK = VEC ? 2 : 4;  // k-blocks of a group: one wait for all their scales
    static constexpr int SCALES = kSlots * SLOTK * SLOT * 4;
    // tiles that are few share their k-blocks over a cluster; the sums meet in
    // the ring's place, rows 4 floats apart in banks
    static constexpr bool SPLITS = BN == 128 && !ROWS;
    static constexpr int SUM_LD = BN + 4;
    static_assert(!SPLITS || 128 * SUM_LD * 4 <= STAGES * STAGE, "a tile's sums fit the ring");
    static constexpr int TABLE = ROWS ? (2 * kMaxGroups + 1) * 4 : 0;
    static constexpr int SMEM = 1024 + STAGES * STAGE + STAGING + SCALES + 512 + TABLE;
    static_assert(SMEM <= 227 * 1024, "above the shared memory of a block");
    // (a wait on parity is only good for a phase whose predecessor the waiter
    // has seen complete, so an issuer must come by at every phase of a barrier)
    static_assert(STAGES % 2 == 0 && PARTS % 2 == 0, "a stage and a part always meet the same one of two issuers");
};

// Waits of the pipeline. A wait that runs out of time records the error,
// raises the CTA's flag and returns false; from then on no wait of the CTA
// lasts. Copying warps and MMA issuers then stop issuing and drain what they
// have in flight, so that nothing lands in shared memory or TMEM that is no
// longer theirs; the scaling warps run to their end on stale data.
struct Pipe {
    volatile int* dead;
    int* err;
    int code;
    __device__ __forceinline__ bool slow(uint64_t* bar, uint32_t parity) const {
        const long long t0 = clock64();
        while (!ptx::mbar_try_wait(bar, parity)) {
            if (*dead) return false;
            if (clock64() - t0 > ptx::kWaitCycles) {
                *dead = 1;
                if (err) atomicCAS(err, 0, code);
                return false;
            }
        }
        return true;
    }
    __device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity) const {
        return ptx::mbar_try_wait(bar, parity) || slow(bar, parity);
    }
    // Where the CTA gave up: waits, with a limit of its own, for the phases of
    // `bars` that the last `most` of `uses` uses of a ring complete.
    __device__ __forceinline__ void drain(uint64_t* bars, int ring, int uses, int most) const {
        if (!*dead) return;
        const long long t0 = clock64();
        for (int i = max(0, uses - most); i < uses; i++)
            while (!ptx::mbar_try_wait(&bars[i % ring], i / ring & 1))
                if (clock64() - t0 > ptx::kWaitCycles) return;
    }
};

struct Unit {
    int g, m0, row_end, n0, kb0, kb1;
};

// Tile u of the work: tiles of a group run along n first, those of a single
// product in bands of kBand n tiles, so that tiles in flight share operands.
template <int BM, int BN, bool ROWS>
__device__ __forceinline__ Unit unit_at(const TileParams& p, const int* start, int u) {
    Unit w;
    if (ROWS) {
        int t = u / p.n_tiles;
        int lo = 0, hi = p.groups;  // start[lo] <= t < start[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (start[mid] <= t) lo = mid;
            else hi = mid;
        }
        w.g = lo;
        w.m0 = start[kMaxGroups + 1 + lo] + (t - start[lo]) * BM;
        w.row_end = min(p.M, start[kMaxGroups + 1 + lo] + p.counts[lo]);
        w.n0 = u % p.n_tiles * BN;
        w.kb0 = 0;
        w.kb1 = (p.K + 127) / 128;
        return w;
    }
    const int tiles = p.m_tiles * p.n_tiles;
    w.g = u / tiles;
    u -= w.g * tiles;
    const int band = u / (kBand * p.m_tiles);
    u -= band * kBand * p.m_tiles;
    const int width = min(kBand, p.n_tiles - band * kBand);
    w.m0 = u / width * BM;
    w.n0 = (band * kBand + u % width) * BN;
    w.row_end = p.M;
    w.kb0 = 0;
    w.kb1 = (p.K + 127) / 128;
    if (p.groups) {
        const int off = max(0, p.offsets[w.g]);
        w.kb0 = off / 128;
        w.kb1 = min(w.kb1, (off + p.counts[w.g] + 127) / 128);
    }
    return w;
}

// First tile (of `rows` rows) of every group into start[0..groups], its first
// row behind them. By one warp.
__device__ __forceinline__ void group_starts(const TileParams& p, int rows, int* start, int lane) {
    int run = 0;
    for (int g0 = 0; g0 < p.groups; g0 += 32) {
        const int g = g0 + lane;
        int n = 0;
        if (g < p.groups) {
            const int off = max(0, p.offsets[g]), end = max(off, min(p.M, off + p.counts[g]));
            start[kMaxGroups + 1 + g] = off;
            n = (end - off + rows - 1) / rows;
        }
        int inc = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += t;
        }
        if (g < p.groups) start[g] = run + inc - n;
        run += __shfl_sync(0xffffffffu, inc, 31);
    }
    if (lane == 0) start[p.groups] = run;
}

__device__ __forceinline__ float4 cluster_load4(const float* p, unsigned rank) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(ptx::cluster_addr(p, rank))
                 : "memory");
    return v;
}

template <int BN, bool VEC, bool ROWS, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1)
    fp8_tile_kernel(const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap tb,
                    const __grid_constant__ CUtensorMap tc, const TileParams p) {
    using C = TileCfg<BN, VEC, ROWS, PAIR>;
    constexpr uint32_t IDESC = ptx::instr_desc(0, 0, 0, C::BM, BN);
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* staging = smem + C::STAGES * C::STAGE;
    float* slots = reinterpret_cast<float*>(staging + C::STAGING);
    uint64_t* full = reinterpret_cast<uint64_t*>(staging + C::STAGING + C::SCALES);
    uint64_t* empty = full + C::STAGES;
    uint64_t* part_full = empty + C::STAGES;
    uint64_t* part_empty = part_full + C::PARTS;
    uint64_t* slot_full = part_empty + C::PARTS;
    uint64_t* slot_empty = slot_full + kSlots;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(slot_empty + kSlots);
    int* dead = reinterpret_cast<int*>(tmem_slot + 1);
    int* start = reinterpret_cast<int*>(staging + C::STAGING + C::SCALES + 512);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // a pair's first CTA issues its MMAs; CTA r of a splitting cluster takes the
    // r-th share of the k-blocks
    const uint32_t rank = PAIR ? ptx::cluster_ctarank() : 0;
    const int split = C::SPLITS ? p.split : 1, share_of = split > 1 ? (int)ptx::cluster_ctarank() : 0;
    const bool gather = ROWS && p.rows;
    if (threadIdx.x == 0) {
        *dead = 0;
        for (int s = 0; s < C::STAGES; s++) {
            // TMA's arrival and, with gathered rows, every copying thread's
            ptx::mbar_init(&full[s], gather ? 65 : 1);
            ptx::mbar_init(&empty[s], 1);
        }
        for (int s = 0; s < kSlots; s++) {
            ptx::mbar_init(&slot_full[s], 64);
            ptx::mbar_init(&slot_empty[s], kEpi);
        }
        for (int s = 0; s < C::PARTS; s++) {
            ptx::mbar_init(&part_full[s], 1);
            ptx::mbar_init(&part_empty[s], PAIR ? 2 * kEpi : kEpi);
        }
        ptx::fence_mbar_init();
        ptx::prefetch_tmap(&ta);
        ptx::prefetch_tmap(&tb);
        if (p.tma_out) ptx::prefetch_tmap(&tc);
    }
    if (warp == 1) {
        if (PAIR) {
            ptx::tmem_alloc_pair(tmem_slot, 512);
            ptx::tmem_relinquish_pair();
        } else {
            ptx::tmem_alloc(tmem_slot, 512);
            ptx::tmem_relinquish();
        }
    }
    if (ROWS && warp == 4) group_starts(p, C::BM, start, lane);
    ptx::tc_fence_before();
    __syncwarp();
    if (PAIR) ptx::cluster_sync();
    else __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const int total = ROWS ? start[p.groups] * p.n_tiles : p.m_tiles * p.n_tiles * (p.groups ? p.groups : 1);
    const int first = PAIR ? blockIdx.x / 2 : blockIdx.x / split;
    const int stride = PAIR ? gridDim.x / 2 : gridDim.x / split;
    auto unit = [&](int u) {
        Unit w = unit_at<C::BM, BN, ROWS>(p, start, u);
        if (C::SPLITS && split > 1) {
            const int share = (w.kb1 - w.kb0 + split - 1) / split;
            w.kb0 = min(w.kb1, w.kb0 + share_of * share);
            w.kb1 = min(w.kb1, w.kb0 + share);
        }
        return w;
    };

    if (warp < 4) {
        // (all four warps of the group at one instruction, and the registers
        // that the compiler counts on in the branch itself)
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (warp == 1 || warp == 2) {
            if (lane == 0 && rank == 0) {
                const int mine = warp - 1;
                const Pipe pipe{dead, p.err, kErrTimeoutMma};
                int it = 0;  // k-blocks so far: number `it` uses stage it % STAGES and part it % PARTS
                int last = -1;
                for (int u = first; u < total; u += stride) {
                    const Unit w = unit(u);
                    for (int kb = w.kb0; kb < w.kb1; kb++, it++) {
                        if ((it & 1) != mine) continue;
                        const int stage = it % C::STAGES, part = it % C::PARTS;
                        if (!pipe.wait(&full[stage], it / C::STAGES & 1)) goto issued;
                        if (!pipe.wait(&part_empty[part], (it / C::PARTS & 1) ^ 1)) goto issued;
                        last = it;
                        // gathered rows came through the generic proxy; the fence is
                        // here, where no copies are in flight that it would wait for
                        if (gather) ptx::fence_proxy_async();
                        ptx::tc_fence_after();
                        const uint32_t sa = ptx::smem_u32(smem + stage * C::STAGE), sb = sa + C::A_BYTES;
    #pragma unroll
                        for (int k = 0; k < 4; k++) {
                            const uint64_t da = ptx::smem_desc(sa + k * 32, 16, 1024, 2);
                            const uint64_t db = ptx::smem_desc(sb + k * 32, 16, 1024, 2);
                            if (PAIR) ptx::mma_f8_pair(tmem + part * C::PCOLS, da, db, IDESC, k > 0);
                            else ptx::mma_f8(tmem + part * C::PCOLS, da, db, IDESC, k > 0);
                        }
                        if (PAIR) {
                            ptx::mma_commit_pair(&empty[stage]);
                            ptx::mma_commit_pair(&part_full[part]);
                        } else {
                            ptx::mma_commit(&empty[stage]);
                            ptx::mma_commit(&part_full[part]);
                        }
                    }
                }
            issued:
                // the MMAs are done before TMEM is freed (else the scaling warps
                // have waited for them)
                pipe.drain(empty, C::STAGES, last + 1, 1);
                pipe.drain(part_full, C::PARTS, last + 1, 1);
            }
        } else {
            const int t = (warp == 0 ? 0 : 32) + lane;  // 0..63
            int slot = 0, stage = 0, loads = 0;
            uint32_t slot_phase = 0, phase = 0;
            const Pipe pipe{dead, p.err, kErrTimeoutProducer};
            for (int u = first; u < total; u += stride) {
                Unit w = unit(u);
                if (PAIR) w.m0 += rank * 128;
                // the rows whose scales this thread copies; rows past the end
                // take the first one's, and are not stored
                const float* srow[2];
    #pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int m = w.m0 + t + 64 * i;
                    const int r = m >= w.row_end ? 0 : gather ? min(max(0, p.rows[m]) / p.row_div, p.a_rows - 1) : m;
                    srow[i] = p.sa + r;
                }
                const float* sb = p.sb;
                if (!VEC)
                    sb += (ROWS ? w.g * p.sb_stride : 0) +
                          (long long)min(w.n0 / 128 + (t & 1) * (BN / 256), p.nb - 1) * p.ld_sb;
                // gathered: pieces t % 4 and t % 4 + 4 (of 16 bytes) of rows t / 4,
                // t / 4 + 16, ...; rows past the end read the first one's
                const uint8_t* from[8];
                if (gather) {
    #pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const int m = w.m0 + t / 4 + 16 * i;
                        const int r = m < w.row_end ? min(max(0, p.rows[m]) / p.row_div, p.a_rows - 1) : 0;
                        from[i] = p.a + (size_t)r * p.lda + (t & 3) * 16;
                    }
                }
                for (int kb = w.kb0; kb < w.kb1; kb++) {
                    const int in = (kb - w.kb0) % C::SLOTK;
                    if (in == 0 && !pipe.wait(&slot_empty[slot], slot_phase ^ 1)) goto copied;
                    float* to = slots + (slot * C::SLOTK + in) * C::SLOT;
    #pragma unroll
                    for (int i = 0; i < 2; i++) ptx::cp_async4(to + t + 64 * i, srow[i] + kb * p.ld_sa);
                    if (VEC) {
    #pragma unroll
                        for (int i = 0; i < BN / 64; i++) {
                            const int n = w.n0 + t + 64 * i;
                            if (n < p.N) ptx::cp_async4(to + 128 + t + 64 * i, sb + kb * p.ld_sb + n);
                        }
                    } else if (t < 2) {
                        ptx::cp_async4(to + 128 + t, sb + kb);
                    }
                    if (in == C::SLOTK - 1 || kb + 1 == w.kb1) {
                        ptx::cp_async_arrive(&slot_full[slot]);
                        if (++slot == kSlots) {
                            slot = 0;
                            slot_phase ^= 1;
                        }
                    }
                    if (!gather && warp != 0) continue;
                    if (!pipe.wait(&empty[stage], phase ^ 1)) goto copied;
                    uint8_t* sa = smem + stage * C::STAGE;
                    if (t == 0) {
                        loads++;
                        if (PAIR) {
                            // both CTAs' loads complete on the first one's barrier
                            const uint32_t bar = ptx::cluster_addr(&full[stage], 0);
                            if (rank == 0) ptx::mbar_arrive_expect_tx(&full[stage], 2 * C::STAGE);
                            ptx::tma_load_2d_pair(sa, &ta, bar, kb * 128, w.m0);
                            ptx::tma_load_3d_pair(sa + C::A_BYTES, &tb, bar, kb * 128, w.n0 + rank * C::BROWS, 0);
                        } else {
                            ptx::mbar_arrive_expect_tx(&full[stage], gather ? C::STAGE - C::A_BYTES : C::STAGE);
                            if (!gather) ptx::tma_load_2d(sa, &ta, &full[stage], kb * 128, w.m0);
                            ptx::tma_load_3d(sa + C::A_BYTES, &tb, &full[stage], kb * 128, w.n0, ROWS ? w.g : 0);
                        }
                    }
                    uint64_t* landed = &full[stage];
                    if (++stage == C::STAGES) {
                        stage = 0;
                        phase ^= 1;
                    }
                    if (!gather) continue;
                    // row r's piece q lies at piece q ^ (r % 8)
                    uint8_t* lo = sa + (t >> 2) * 128 + (((t & 3) ^ (t >> 2 & 7)) << 4);
                    uint8_t* hi = sa + (t >> 2) * 128 + (((t & 3) ^ (t >> 2 & 7) ^ 4) << 4);
                    if (kb * 128 + 128 <= p.K) {
    #pragma unroll
                        for (int i = 0; i < 8; i++) {
                            ptx::cp_async16(lo + i * 2048, from[i]);
                            ptx::cp_async16(hi + i * 2048, from[i] + 64);
                            from[i] += 128;
                        }
                    } else {
                        const int k = kb * 128 + (t & 3) * 16;
                        const int b0 = max(0, min(16, p.K - k)), b1 = max(0, min(16, p.K - k - 64));
    #pragma unroll
                        for (int i = 0; i < 8; i++) {
                            ptx::cp_async16(lo + i * 2048, b0 ? from[i] : p.a, b0);
                            ptx::cp_async16(hi + i * 2048, b1 ? from[i] + 64 : p.a, b1);
                        }
                    }
                    ptx::cp_async_arrive(landed);
                }
            }
            // every load has landed and been used before the CTA exits (bounded)
            if (t == 0)
                for (int s = 0; s < C::STAGES; s++) {
                    if (!pipe.wait(&empty[stage], phase ^ 1)) break;
                    if (++stage == C::STAGES) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
        copied:
            ptx::cp_async_wait_all();
            // or at least landed, where the CTA gave up (those of a pair's second
            // CTA complete on the first one's barriers, and the two leave together)
            if (t == 0 && rank == 0) pipe.drain(full, C::STAGES, loads, C::STAGES);
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        const int quarter = warp & 3, half = (warp - 4) >> 2;
        uint8_t* stg = staging + (warp - 4) * 2048;
        int part = 0, slot = 0;
        uint32_t part_phase = 0, slot_phase = 0;
        const Pipe pipe{dead, p.err, kErrTimeoutEpilogue};
        const uint32_t lane_base = tmem + ((uint32_t)(quarter * 32) << 16) + half * C::COLS;
        for (int u = first; u < total; u += stride) {
            Unit w = unit(u);
            if (PAIR) w.m0 += rank * 128;
            const int row = w.m0 + quarter * 32 + lane;
            const bool valid = row < w.row_end;
            const int col0 = w.n0 + half * C::COLS;
            float acc[C::COLS];
#pragma unroll
            for (int j = 0; j < C::COLS; j++) acc[j] = 0.f;
            int in = 0;
            // block scales: this row's, times the block's, of the group's k-blocks;
            // column scales: four rows' of one k-block (the fragment's)
            constexpr int NS = VEC ? 4 : C::SLOTK;
            float sr[NS];
            for (int kb = w.kb0; kb < w.kb1; kb++) {
                const float* sc = slots + (slot * C::SLOTK + in) * C::SLOT;
                if (in == 0) pipe.wait(&slot_full[slot], slot_phase);
                if (VEC) {
#pragma unroll
                    for (int i = 0; i < 4; i++) sr[i] = sc[quarter * 32 + i * 8 + (lane >> 2)];
                } else if (in == 0) {
#pragma unroll
                    for (int i = 0; i < NS; i++)
                        sr[i] = sc[i * C::SLOT + quarter * 32 + lane] * sc[i * C::SLOT + 128 + half];
                }
                const float s = sr[0];
                if (!VEC) {
#pragma unroll
                    for (int i = 0; i + 1 < NS; i++) sr[i] = sr[i + 1];
                }
                pipe.wait(&part_full[part], part_phase);
                __syncwarp();
                ptx::tc_fence_after();
                const uint32_t t = lane_base + part * C::PCOLS;
                if constexpr (VEC) {
                    // fragments of 16 rows x 32 columns: of each a thread has two
                    // rows (lane / 4, + 8) and the columns 2 (lane % 4) of every 8,
                    // so it needs 4 row and 32 column scales, not 1 and 128
                    const uint64_t* v = reinterpret_cast<const uint64_t*>(sc + 128 + half * C::COLS) + (lane & 3);
                    uint32_t r[2][16];
                    ptx::tmem_ld_frag32(t, r[0]);
#pragma unroll
                    for (int c = 0; c < C::COLS / 32; c++) {
                        uint64_t q[4];
#pragma unroll
                        for (int j = 0; j < 4; j++) q[j] = v[c * 16 + j * 4];
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            ptx::tmem_ld_wait_regs16(r[h]);
                            if (h == 0) ptx::tmem_ld_frag32(t + (16u << 16) + c * 32, r[1]);
                            else if (c + 1 < C::COLS / 32) ptx::tmem_ld_frag32(t + (c + 1) * 32, r[0]);
#pragma unroll
                            for (int j = 0; j < 8; j++) {
                                float* o = acc + ((c * 2 + h) * 8 + j) * 2;
                                const float sj = sr[h * 2 + (j & 1)];
                                const uint64_t x =
                                    f2_pack(__uint_as_float(r[h][2 * j]), __uint_as_float(r[h][2 * j + 1]));
                                f2_unpack(f2_fma(f2_mul(x, q[j >> 1]), f2_pack(sj, sj), f2_pack(o[0], o[1])), o[0], o[1]);
                            }
                        }
                    }
                } else {
                    // 16 columns at a time, the next 16 on their way; packed pairs
                    // halve the FMA instructions
                    uint32_t r[2][16];
                    ptx::tmem_ld16(t, r[0]);
                    const uint64_t s2 = f2_pack(s, s);
#pragma unroll
                    for (int c = 0; c < C::COLS / 16; c++) {
                        ptx::tmem_ld_wait_regs16(r[c & 1]);
                        if (c + 1 < C::COLS / 16) ptx::tmem_ld16(t + (c + 1) * 16, r[(c + 1) & 1]);
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            float* o = acc + c * 16 + 2 * j;
                            const uint64_t x =
                                f2_pack(__uint_as_float(r[c & 1][2 * j]), __uint_as_float(r[c & 1][2 * j + 1]));
                            f2_unpack(f2_fma(x, s2, f2_pack(o[0], o[1])), o[0], o[1]);
                        }
                    }
                }
                ptx::tc_fence_before();
                __syncwarp();
                if (PAIR) ptx::mbar_arrive_cluster_if(ptx::cluster_addr(&part_empty[part], 0), lane == 0);
                else ptx::mbar_arrive_if(&part_empty[part], lane == 0);
                if (++in == C::SLOTK || kb + 1 == w.kb1) {
                    ptx::mbar_arrive_if(&slot_empty[slot], lane == 0);
                    in = 0;
                    if (++slot == kSlots) {
                        slot = 0;
                        slot_phase ^= 1;
                    }
                }
                if (++part == C::PARTS) {
                    part = 0;
                    part_phase ^= 1;
                }
            }
            if constexpr (C::SPLITS) {
                if (split > 1) {
                    // (this CTA's loads have all been used: its last part was read)
                    float* sum = reinterpret_cast<float*>(smem) + half * C::COLS;
                    if constexpr (VEC) {
#pragma unroll
                        for (int j = 0; j < C::COLS / 2; j++)
                            *reinterpret_cast<float2*>(
                                sum + (quarter * 32 + (j >> 3 & 1) * 16 + (j & 1) * 8 + (lane >> 2)) * C::SUM_LD +
                                (j >> 4) * 32 + (j >> 1 & 3) * 8 + (lane & 3) * 2) = make_float2(acc[2 * j], acc[2 * j + 1]);
                    } else {
#pragma unroll
                        for (int j = 0; j < C::COLS / 4; j++)
                            *reinterpret_cast<float4*>(sum + (quarter * 32 + lane) * C::SUM_LD + 4 * j) =
                                make_float4(acc[4 * j], acc[4 * j + 1], acc[4 * j + 2], acc[4 * j + 3]);
                    }
                    continue;
                }
            }
            if constexpr (VEC) {
                if (p.tma_out) {
                    const int y = w.m0 + quarter * 32;
                    // 64 bytes of this warp's 32 rows, written into its staging buffer by
                    // `fill`, leave by TMA (which clips at the tensor's end)
                    auto leave = [&](int x, int z, auto fill) {
                        if (lane == 0) ptx::bulk_wait_read0();
                        __syncwarp();
                        fill();
                        ptx::fence_proxy_async();
                        __syncwarp();
                        if (lane == 0) {
                            ptx::tma_store_3d(&tc, stg, x, y, z);
                            ptx::bulk_commit();
                        }
                    };
                    // (staging's 16-byte piece q of row r lies at q ^ (r / 2 % 4))
                    const int es = p.c_dtype == kBF16 ? 2 : 4;
#pragma unroll
                    for (int c = 0; c < C::COLS / 32; c++)
#pragma unroll
                        for (int b = 0; b < 2; b++) {
                            const int x = col0 + c * 32 + b * 16;
                            if ((es == 2 && b) || x >= p.N || y >= p.M) continue;
                            leave(x, w.g, [&] {
#pragma unroll
                                for (int h = 0; h < 2; h++)
#pragma unroll
                                    for (int j = 0; j < 8; j++) {
                                        const int r = h * 16 + (j & 1) * 8 + (lane >> 2);
                                        const float* o = acc + ((c * 2 + h) * 8 + j) * 2;
                                        if (es == 2) {  // columns 8 (j / 2) + 2 (lane % 4)
                                            *reinterpret_cast<__nv_bfloat162*>(
                                                stg + r * 64 + (((j >> 1) ^ (r >> 1 & 3)) << 4) + (lane & 3) * 4) =
                                                __floats2bfloat162_rn(o[0], o[1]);
                                        } else if (j >> 2 == b) {  // 8 (j / 2 % 2) + 2 (lane % 4)
                                            const int q = (j >> 1 & 1) * 2 + ((lane & 3) >> 1);
                                            *reinterpret_cast<float2*>(stg + r * 64 + ((q ^ (r >> 1 & 3)) << 4) +
                                                                       (lane & 1) * 8) = make_float2(o[0], o[1]);
                                        }
                                    }
                            });
                        }
                    continue;
                }
                // row by row, two columns a thread
                const size_t base = (size_t)w.g * p.c_stride;
#pragma unroll
                for (int c = 0; c < C::COLS / 32; c++)
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            const int m = w.m0 + quarter * 32 + h * 16 + (j & 1) * 8 + (lane >> 2);
                            const int n = col0 + c * 32 + (j >> 1) * 8 + (lane & 3) * 2;
                            const float* o = acc + ((c * 2 + h) * 8 + j) * 2;
                            if (m >= w.row_end) continue;
#pragma unroll
                            for (int i = 0; i < 2; i++) {
                                if (n + i >= p.N) continue;
                                const size_t at = base + (size_t)m * p.ldc + n + i;
                                if (p.c_dtype == kBF16) reinterpret_cast<__nv_bfloat16*>(p.c)[at] = f2bf(o[i]);
                                else reinterpret_cast<float*>(p.c)[at] = o[i];
                            }
                        }
                continue;
            }
            // a slab of 32 rows leaves by TMA where all of them are the tile's
            // (the store clips at the tensor's end), else row by row
            const int y = w.m0 + quarter * 32;
            const int gz = ROWS ? 0 : w.g;
            const bool tma = p.tma_out && (!ROWS || y + 32 <= w.row_end);
#pragma unroll
            for (int c = 0; c < C::COLS / 32; c++) {
                const int col = col0 + c * 32;
                if (col >= p.N) continue;
                const float* f = acc + c * 32;
                if (tma) {
                    if (y >= p.M) continue;
                    const int boxes = p.c_dtype == kBF16 ? 1 : 2;
#pragma unroll
                    for (int b = 0; b < 2; b++) {
                        const int x = col + b * 16;
                        if (b >= boxes || (b && x >= p.N)) continue;
                        uint8_t* dst = stg;
                        if (lane == 0) ptx::bulk_wait_read0();
                        __syncwarp();
#pragma unroll
                        for (int q = 0; q < 4; q++) {
                            uint4 o;
                            if (p.c_dtype == kBF16) {
                                __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&o);
#pragma unroll
                                for (int i = 0; i < 4; i++) h[i] = __floats2bfloat162_rn(f[8 * q + 2 * i], f[8 * q + 2 * i + 1]);
                            } else {
                                o = make_uint4(__float_as_uint(f[16 * b + 4 * q]), __float_as_uint(f[16 * b + 4 * q + 1]),
                                               __float_as_uint(f[16 * b + 4 * q + 2]),
                                               __float_as_uint(f[16 * b + 4 * q + 3]));
                            }
                            *reinterpret_cast<uint4*>(dst + lane * 64 + ((q ^ ((lane >> 1) & 3)) << 4)) = o;
                        }
                        ptx::fence_proxy_async();
                        __syncwarp();
                        if (lane == 0) {
                            ptx::tma_store_3d(&tc, dst, x, y, gz);
                            ptx::bulk_commit();
                        }
                    }
                } else if (valid) {
                    const size_t at = (size_t)gz * p.c_stride + (size_t)row * p.ldc + col;
                    const bool vec16 = p.vec_out && col + 32 <= p.N;
                    if (p.c_dtype == kBF16) {
                        __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(p.c) + at;
#pragma unroll
                        for (int q = 0; q < 4; q++) {
                            uint4 t;
                            __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&t);
#pragma unroll
                            for (int i = 0; i < 4; i++) h[i] = __floats2bfloat162_rn(f[8 * q + 2 * i], f[8 * q + 2 * i + 1]);
                            if (vec16) {
                                reinterpret_cast<uint4*>(o)[q] = t;
                            } else {
                                const __nv_bfloat16* e = reinterpret_cast<const __nv_bfloat16*>(&t);
#pragma unroll
                                for (int i = 0; i < 8; i++)
                                    if (col + 8 * q + i < p.N) o[8 * q + i] = e[i];
                            }
                        }
                    } else {
                        float* o = reinterpret_cast<float*>(p.c) + at;
#pragma unroll
                        for (int q = 0; q < 8; q++) {
                            if (vec16) {
                                reinterpret_cast<float4*>(o)[q] = make_float4(f[4 * q], f[4 * q + 1], f[4 * q + 2], f[4 * q + 3]);
                            } else {
#pragma unroll
                                for (int i = 0; i < 4; i++)
                                    if (col + 4 * q + i < p.N) o[4 * q + i] = f[4 * q + i];
                            }
                        }
                    }
                }
            }
        }
        if (lane == 0) ptx::bulk_wait_all();
        __syncwarp();
    }

    ptx::tc_fence_before();
    // (a pair leaves together: each other's shared memory is read and arrived at)
    __syncwarp();
    if (PAIR) ptx::cluster_sync();
    else __syncthreads();
    if (warp == 1) {
        ptx::tc_fence_after();
        if (PAIR) ptx::tmem_dealloc_pair(tmem, 512);
        else ptx::tmem_dealloc(tmem, 512);
    }
    if constexpr (C::SPLITS) {
        if (split > 1) {
            // the shares are added in rank order; rank r stores every split-th row
            ptx::cluster_sync();
            const Unit w = unit_at<C::BM, BN, ROWS>(p, start, first);
            const float* sum = reinterpret_cast<const float*>(smem);
            constexpr int QUADS = BN / 4;
            for (int i = threadIdx.x; i < 128 / split * QUADS; i += kThreads) {
                const int r = i / QUADS * split + share_of, n = w.n0 + i % QUADS * 4, m = w.m0 + r;
                if (m >= w.row_end || n >= p.N) continue;
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                for (int q = 0; q < split; q++) {
                    const float4 t = cluster_load4(sum + r * C::SUM_LD + i % QUADS * 4, q);
                    v.x += t.x, v.y += t.y, v.z += t.z, v.w += t.w;
                }
                const size_t at = (size_t)m * p.ldc + n;
                const float f[4] = {v.x, v.y, v.z, v.w};
                if (p.c_dtype == kBF16) {
                    __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(p.c) + at;
                    if (p.vec_out && n + 4 <= p.N) {
                        reinterpret_cast<__nv_bfloat162*>(o)[0] = __floats2bfloat162_rn(v.x, v.y);
                        reinterpret_cast<__nv_bfloat162*>(o)[1] = __floats2bfloat162_rn(v.z, v.w);
                    } else {
                        for (int j = 0; j < 4; j++)
                            if (n + j < p.N) o[j] = f2bf(f[j]);
                    }
                } else {
                    float* o = reinterpret_cast<float*>(p.c) + at;
                    if (p.vec_out && n + 4 <= p.N) {
                        *reinterpret_cast<float4*>(o) = v;
                    } else {
                        for (int j = 0; j < 4; j++)
                            if (n + j < p.N) o[j] = f[j];
                    }
                }
            }
            ptx::cluster_sync();  // no CTA leaves while others read its sums
        }
    }
}

// ---------------------------------------------------------------------------
// Few rows of A (or few for each expert): the sides change places. 128 rows of
// B, the weights, are the MMA's rows and BN rows of A its columns, so a tile
// reads no more than the weights and what there is of A. What bounds it is
// the stream of the weights, so everything serves loads in flight: a deep
// ring, eight parts of TMEM, and for one product the k-blocks of a tile split
// over a cluster of CTAs, whose sums meet in shared memory in rank order.
// 1 x 4096 x 4096: 7.5 us (2.6 us of HBM time, the rest latency); 24 tokens x 4
// of 64 experts, 2048 x 1024: 22.3 us (4.8 TB/s, 5 to 7 tiles an SM; 28 us with
// one CTA an SM).
//   warp 0       weights by TMA
//   warps 1, 8   MMA issuers, every other k-block each
//   warps 2..3   rows of A by cp.async (listed, or in order) and the scales
//   warps 4..7   a warp owns 32 weight rows: scales and adds, stores
// ---------------------------------------------------------------------------
constexpr int kSmallThreads = 288;

template <int BN, bool VEC>
struct SmallCfg {
    static constexpr int W_BYTES = 128 * 128;
    static constexpr int STAGE = W_BYTES + BN * 128;
    static constexpr int CTAS = 2;  // an SM: the copies and sums of one hide the other's
    static constexpr int STAGES = 4;
    static constexpr int PARTS = 8;
    static constexpr int SLOTK = 4;
    static constexpr int SLOT = BN + (VEC ? 128 : 4);  // scales of A's rows, then of B's rows or block
    static constexpr int SCALES = kSlots * SLOTK * SLOT * 4;
    static constexpr int SMEM = 1024 + STAGES * STAGE + SCALES + 512 + (2 * kMaxGroups + 1) * 4;
    static_assert(CTAS * (SMEM + 1024) <= 228 * 1024, "above the shared memory of an SM");
    static_assert(CTAS * PARTS * BN <= 512, "above the columns of TMEM");
    static_assert(STAGES % 2 == 0 && PARTS % 2 == 0, "a stage and a part always meet the same one of two issuers");
    static_assert(BN * 128 * 4 <= STAGES * STAGE, "the cluster's sums take the ring's place");
};

struct SmallParams {
    TileParams t;  // M: rows of A in order; N: weight rows
    int split;     // CTAs of a cluster that share a tile's k-blocks
};

__device__ __forceinline__ float cluster_loadf(const float* p, unsigned rank) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(ptx::cluster_addr(p, rank)) : "memory");
    return v;
}

template <int BN>
__device__ __forceinline__ Unit small_unit(const TileParams& p, const int* start, int u) {
    Unit w;
    int t = u / p.n_tiles;
    w.n0 = u % p.n_tiles * 128;
    w.kb0 = 0;
    w.kb1 = (p.K + 127) / 128;
    w.g = 0;
    w.m0 = t * BN;
    w.row_end = p.M;
    if (p.groups) {
        int lo = 0, hi = p.groups;  // start[lo] <= t < start[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (start[mid] <= t) lo = mid;
            else hi = mid;
        }
        w.g = lo;
        w.m0 = start[kMaxGroups + 1 + lo] + (t - start[lo]) * BN;
        w.row_end = min(p.M, start[kMaxGroups + 1 + lo] + p.counts[lo]);
    }
    return w;
}

template <int BN, bool VEC>
__global__ void __launch_bounds__(kSmallThreads, SmallCfg<BN, VEC>::CTAS)
    fp8_small_kernel(const __grid_constant__ CUtensorMap tw, const __grid_constant__ SmallParams sp) {
    using C = SmallCfg<BN, VEC>;
    const TileParams& p = sp.t;
    constexpr uint32_t IDESC = ptx::instr_desc(0, 0, 0, 128, BN);
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float* slots = reinterpret_cast<float*>(smem + C::STAGES * C::STAGE);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::STAGES * C::STAGE + C::SCALES);
    uint64_t* empty = full + C::STAGES;
    uint64_t* part_full = empty + C::STAGES;
    uint64_t* part_empty = part_full + C::PARTS;
    uint64_t* slot_full = part_empty + C::PARTS;
    uint64_t* slot_empty = slot_full + kSlots;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(slot_empty + kSlots);
    int* dead = reinterpret_cast<int*>(tmem_slot + 1);
    int* start = reinterpret_cast<int*>(smem + C::STAGES * C::STAGE + C::SCALES + 512);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        *dead = 0;
        for (int s = 0; s < C::STAGES; s++) {
            ptx::mbar_init(&full[s], 65);
            ptx::mbar_init(&empty[s], 1);
        }
        for (int s = 0; s < C::PARTS; s++) {
            ptx::mbar_init(&part_full[s], 1);
            ptx::mbar_init(&part_empty[s], 4);
        }
        for (int s = 0; s < kSlots; s++) {
            ptx::mbar_init(&slot_full[s], 64);
            ptx::mbar_init(&slot_empty[s], 4);
        }
        ptx::fence_mbar_init();
        ptx::prefetch_tmap(&tw);
    }
    if (warp == 1) {
        ptx::tmem_alloc(tmem_slot, C::PARTS * BN);
        ptx::tmem_relinquish();
    }
    if (p.groups && warp == 4) group_starts(p, BN, start, lane);
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const int total = (p.groups ? start[p.groups] : p.m_tiles) * p.n_tiles;
    // a cluster takes one tile, rank r the r-th share of its k-blocks; without
    // clusters the CTAs take tiles in turn
    const int rank = sp.split > 1 ? blockIdx.x % sp.split : 0;
    const int first = sp.split > 1 ? blockIdx.x / sp.split : blockIdx.x;
    const int stride = sp.split > 1 ? total : gridDim.x;
    const int kblocks = (p.K + 127) / 128, share = (kblocks + sp.split - 1) / sp.split;
    const int kb0 = min(kblocks, rank * share), kb1 = min(kblocks, kb0 + share);

    if (warp == 0) {
        if (lane == 0) {
            const Pipe pipe{dead, p.err, kErrTimeoutProducer};
            int stage = 0, loads = 0;
            uint32_t phase = 0;
            for (int u = first; u < total; u += stride) {
                const Unit w = small_unit<BN>(p, start, u);
                for (int kb = kb0; kb < kb1; kb++, loads++) {
                    if (!pipe.wait(&empty[stage], phase ^ 1)) goto loaded;
                    ptx::mbar_arrive_expect_tx(&full[stage], C::W_BYTES);
                    ptx::tma_load_3d(smem + stage * C::STAGE, &tw, &full[stage], kb * 128, w.n0, w.g);
                    if (++stage == C::STAGES) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
            // every load has landed and been used before the CTA exits (bounded)
            for (int s = 0; s < C::STAGES; s++) {
                if (!pipe.wait(&empty[stage], phase ^ 1)) break;
                if (++stage == C::STAGES) {
                    stage = 0;
                    phase ^= 1;
                }
            }
        loaded:
            pipe.drain(full, C::STAGES, loads, C::STAGES);  // or at least landed, where the CTA gave up
        }
        __syncwarp();
    } else if (warp == 1 || warp == 8) {
        if (lane == 0) {
            const Pipe pipe{dead, p.err, kErrTimeoutMma};
            const int mine = warp == 1 ? 0 : 1;
            int it = 0;  // k-blocks so far: number `it` uses stage it % STAGES and part it % PARTS
            int last = -1;
            for (int u = first; u < total; u += stride)
                for (int kb = kb0; kb < kb1; kb++, it++) {
                    if ((it & 1) != mine) continue;
                    const int stage = it % C::STAGES, part = it % C::PARTS;
                    if (!pipe.wait(&full[stage], it / C::STAGES & 1)) goto issued;
                    if (!pipe.wait(&part_empty[part], (it / C::PARTS & 1) ^ 1)) goto issued;
                    last = it;
                    ptx::fence_proxy_async();  // A's rows came through the generic proxy
                    ptx::tc_fence_after();
                    const uint32_t sw = ptx::smem_u32(smem + stage * C::STAGE), sa = sw + C::W_BYTES;
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        ptx::mma_f8(tmem + part * BN, ptx::smem_desc(sw + k * 32, 16, 1024, 2),
                                    ptx::smem_desc(sa + k * 32, 16, 1024, 2), IDESC, k > 0);
                    ptx::mma_commit(&empty[stage]);
                    ptx::mma_commit(&part_full[part]);
                }
        issued:
            // the MMAs are done before TMEM is freed (else the scaling warps have
            // waited for them)
            pipe.drain(empty, C::STAGES, last + 1, 1);
            pipe.drain(part_full, C::PARTS, last + 1, 1);
        }
        __syncwarp();
    } else if (warp < 4) {
        const Pipe pipe{dead, p.err, kErrTimeoutProducer};
        const int t = threadIdx.x - 64;  // 0..63
        int slot = 0, stage = 0;
        uint32_t slot_phase = 0, phase = 0;
        auto source = [&](const Unit& w, int i) {  // row of A behind row i of the tile, -1 past the end
            const int m = w.m0 + i;
            if (m >= w.row_end) return -1;
            return p.rows ? min(max(0, p.rows[m]) / p.row_div, p.a_rows - 1) : m;
        };
        constexpr int PIECES = BN / 8;  // 16-byte pieces of a k-block that this thread copies
        Unit next;
        int ahead[PIECES + 1];  // the next tile's rows, looked up while this one's are copied
        auto look = [&](int u) {
            if (u >= total) return;
            next = small_unit<BN>(p, start, u);
#pragma unroll
            for (int i = 0; i < PIECES; i++) ahead[i] = source(next, t / 8 + 8 * i);
            ahead[PIECES] = source(next, min(t, BN - 1));
        };
        look(first);
        for (int u = first; u < total; u += stride) {
            const Unit w = next;
            int arow[PIECES];
#pragma unroll
            for (int i = 0; i < PIECES; i++) arow[i] = ahead[i];
            const float* srow = p.sa + max(0, ahead[PIECES]);
            look(u + stride);
            const float* sb = p.sb + w.g * p.sb_stride;
            if (!VEC) sb += (long long)(w.n0 / 128) * p.ld_sb;
            for (int kb = kb0; kb < kb1; kb++) {
                const int in = (kb - kb0) % C::SLOTK;
                if (in == 0 && !pipe.wait(&slot_empty[slot], slot_phase ^ 1)) goto copied;
                float* to = slots + (slot * C::SLOTK + in) * C::SLOT;
                if (t < BN) ptx::cp_async4(to + t, srow + kb * p.ld_sa);
                if (VEC) {
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const int n = w.n0 + t + 64 * i;
                        if (n < p.N) ptx::cp_async4(to + BN + t + 64 * i, sb + kb * p.ld_sb + n);
                    }
                } else if (t == 0) {
                    ptx::cp_async4(to + BN, sb + kb);
                }
                if (in == C::SLOTK - 1 || kb + 1 == kb1) {
                    ptx::cp_async_arrive(&slot_full[slot]);
                    if (++slot == kSlots) {
                        slot = 0;
                        slot_phase ^= 1;
                    }
                }
                if (!pipe.wait(&empty[stage], phase ^ 1)) goto copied;
                uint8_t* sa = smem + stage * C::STAGE + C::W_BYTES;
                const int k = kb * 128 + (t & 7) * 16;
                const int bytes = max(0, min(16, p.K - k));
#pragma unroll
                for (int i = 0; i < PIECES; i++) {
                    const int r = t / 8 + 8 * i;  // r % 8 = t / 8: the swizzle's row
                    const bool on = arow[i] >= 0 && bytes > 0;
                    ptx::cp_async16(sa + r * 128 + (((t & 7) ^ (t >> 3)) << 4),
                                    on ? p.a + (size_t)arow[i] * p.lda + k : p.a, on ? bytes : 0);
                }
                ptx::cp_async_arrive(&full[stage]);
                if (++stage == C::STAGES) {
                    stage = 0;
                    phase ^= 1;
                }
            }
        }
    copied:
        ptx::cp_async_wait_all();
        __syncwarp();
    } else {
        const Pipe pipe{dead, p.err, kErrTimeoutEpilogue};
        const int quarter = warp & 3;
        int part = 0, slot = 0;
        uint32_t part_phase = 0, slot_phase = 0;
        for (int u = first; u < total; u += stride) {
            const Unit w = small_unit<BN>(p, start, u);
            const int n_in = quarter * 32 + lane, n = w.n0 + n_in;
            float acc[BN];
#pragma unroll
            for (int j = 0; j < BN; j++) acc[j] = 0.f;
            int in = 0;
            for (int kb = kb0; kb < kb1; kb++) {
                if (in == 0) pipe.wait(&slot_full[slot], slot_phase);
                const float* sc = slots + (slot * C::SLOTK + in) * C::SLOT;
                const float s = VEC ? sc[BN + n_in] : sc[BN];
                pipe.wait(&part_full[part], part_phase);
                __syncwarp();
                ptx::tc_fence_after();
                const uint32_t t = tmem + ((uint32_t)(quarter * 32) << 16) + part * BN;
                uint32_t r[2][16];
                ptx::tmem_ld16(t, r[0]);
#pragma unroll
                for (int c = 0; c < BN / 16; c++) {
                    float m[16];
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const float4 q = reinterpret_cast<const float4*>(sc)[c * 4 + j];
                        m[4 * j] = q.x * s;
                        m[4 * j + 1] = q.y * s;
                        m[4 * j + 2] = q.z * s;
                        m[4 * j + 3] = q.w * s;
                    }
                    ptx::tmem_ld_wait_regs16(r[c & 1]);
                    if (c + 1 < BN / 16) ptx::tmem_ld16(t + (c + 1) * 16, r[(c + 1) & 1]);
#pragma unroll
                    for (int j = 0; j < 16; j++) acc[c * 16 + j] = fmaf(__uint_as_float(r[c & 1][j]), m[j], acc[c * 16 + j]);
                }
                ptx::tc_fence_before();
                __syncwarp();
                ptx::mbar_arrive_if(&part_empty[part], lane == 0);
                if (++in == C::SLOTK || kb + 1 == kb1) {
                    ptx::mbar_arrive_if(&slot_empty[slot], lane == 0);
                    in = 0;
                    if (++slot == kSlots) {
                        slot = 0;
                        slot_phase ^= 1;
                    }
                }
                if (++part == C::PARTS) {
                    part = 0;
                    part_phase ^= 1;
                }
            }
            if (sp.split > 1) {
                // (this CTA's loads have all been used: its last part was read)
                float* sum = reinterpret_cast<float*>(smem);
#pragma unroll
                for (int j = 0; j < BN; j++) sum[j * 128 + n_in] = acc[j];
                continue;
            }
#pragma unroll
            for (int j = 0; j < BN; j++) {
                const int m = w.m0 + j;
                if (m < w.row_end && n < p.N) {
                    if (p.c_dtype == kBF16) reinterpret_cast<__nv_bfloat16*>(p.c)[(size_t)m * p.ldc + n] = f2bf(acc[j]);
                    else reinterpret_cast<float*>(p.c)[(size_t)m * p.ldc + n] = acc[j];
                }
            }
        }
    }

    ptx::tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem, C::PARTS * BN);
    }
    if (sp.split > 1) {
        // the k-blocks' shares are added in rank order; rank r stores every
        // split-th row of the tile
        ptx::cluster_sync();
        if (first < total) {
            const Unit w = small_unit<BN>(p, start, first);
            const float* sum = reinterpret_cast<const float*>(smem);
            const int n_in = threadIdx.x & 127, n = w.n0 + n_in;
            for (int j = rank * 2 + (threadIdx.x >> 7); threadIdx.x < 256 && j < BN; j += sp.split * 2) {
                const int m = w.m0 + j;
                if (m >= w.row_end) break;
                float v = 0.f;
                for (int r = 0; r < sp.split; r++) v += cluster_loadf(sum + j * 128 + n_in, r);
                if (n < p.N) {
                    if (p.c_dtype == kBF16) reinterpret_cast<__nv_bfloat16*>(p.c)[(size_t)m * p.ldc + n] = f2bf(v);
                    else reinterpret_cast<float*>(p.c)[(size_t)m * p.ldc + n] = v;
                }
            }
        }
        ptx::cluster_sync();  // no CTA leaves while others read its sums
    }
}

// An empty sum (K = 0): zeros into C, of row groups into their own rows alone.
__global__ void fp8_zero_kernel(const Fp8Gemm d) {
    const int g = blockIdx.y;
    long long r0 = 0, r1 = d.M;
    if (d.groups && !d.group_k) {
        r0 = max(0, d.offsets[g]);
        r1 = min((long long)d.M, r0 + d.counts[g]);
    }
    const long long n = (r1 - r0) * d.N, at0 = g * (d.group_k ? d.c_stride : 0) + r0 * d.ldc;
    for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x) {
        const long long at = at0 + i / d.N * d.ldc + i % d.N;
        if (d.c_dtype == kBF16) reinterpret_cast<__nv_bfloat16*>(d.c)[at] = f2bf(0.f);
        else reinterpret_cast<float*>(d.c)[at] = 0.f;
    }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encoder() {
    static EncodeTiledFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(f);
    });
    return fn;
}

// Codes [rows, cols] with ld bytes a row: boxes of 128 columns and box rows.
bool map_codes2(CUtensorMap* m, const void* p, long long cols, long long rows, long long ld, int box) {
    EncodeTiledFn enc = encoder();
    if (!enc) return false;
    cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)ld};
    cuuint32_t boxes[2] = {128, (cuuint32_t)box}, one[2] = {1, 1};
    return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(p), dims, strides, boxes, one,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The same, one such array for each of z groups, stride bytes apart.
bool map_codes3(CUtensorMap* m, const void* p, long long cols, long long rows, long long ld, long long z,
                long long stride, int box) {
    EncodeTiledFn enc = encoder();
    if (!enc) return false;
    cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)z};
    cuuint64_t strides[2] = {(cuuint64_t)ld, (cuuint64_t)(z > 1 ? stride : ld * rows)};
    cuuint32_t boxes[3] = {128, (cuuint32_t)box, 1}, one[3] = {1, 1, 1};
    return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(p), dims, strides, boxes, one,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Output boxes of 32 rows x 64 bytes, 64-byte swizzle.
bool map_out(CUtensorMap* m, void* p, int dtype, long long cols, long long rows, long long ld, long long z,
             long long stride) {
    EncodeTiledFn enc = encoder();
    if (!enc) return false;
    const int es = dtype == kBF16 ? 2 : 4;
    cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)z};
    cuuint64_t strides[2] = {(cuuint64_t)(ld * es), (cuuint64_t)((z > 1 ? stride : ld * rows) * es)};
    cuuint32_t boxes[3] = {(cuuint32_t)(64 / es), 32, 1}, one[3] = {1, 1, 1};
    return enc(m, dtype == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, p, dims,
               strides, boxes, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The attribute belongs to the current device: set once for each.
template <typename Kernel>
bool allow_smem(Kernel k, int bytes, bool* done) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return false;
    if (!done[dev]) {
        if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
        done[dev] = true;
    }
    return true;
}

TileParams params(const Fp8Gemm& d, int bm, int bn) {
    TileParams p;
    p.M = d.M;
    p.N = d.N;
    p.K = d.K;
    p.a = d.a;
    p.lda = d.lda;
    p.a_rows = (int)d.a_rows;
    p.sa = d.sa;
    p.ld_sa = d.ld_sa;
    p.sb = d.sb;
    p.ld_sb = d.ld_sb;
    p.sb_stride = d.sb_stride;
    p.c = d.c;
    p.c_dtype = d.c_dtype;
    p.ldc = d.ldc;
    p.c_stride = d.c_stride;
    p.groups = d.groups;
    p.offsets = d.offsets;
    p.counts = d.counts;
    p.rows = d.rows;
    p.row_div = d.row_div;
    p.m_tiles = (d.M + bm - 1) / bm;
    p.n_tiles = (d.N + bn - 1) / bn;
    p.nb = (d.N + 127) / 128;
    p.tma_out = p.vec_out = 0;
    p.split = 1;
    p.err = d.err;
    return p;
}

template <int BN, bool VEC>
int launch_small(const Fp8Gemm& d, cudaStream_t st) {
    using C = SmallCfg<BN, VEC>;
    static bool done[kMaxDevices] = {};
    auto k = fp8_small_kernel<BN, VEC>;
    if (!allow_smem(k, C::SMEM, done)) return -5;
    SmallParams sp;
    sp.t = params(d, BN, 128);
    CUtensorMap tw;
    if (!map_codes3(&tw, d.b, d.K, d.N, d.ldb, d.groups ? d.groups : 1, d.b_stride, 128)) return -2;
    // tiles: of A's rows for each group at most one that is not full
    const long long rows = d.groups ? (long long)d.M / BN + (d.M < d.groups ? d.M : d.groups) : sp.t.m_tiles;
    const long long units = rows * sp.t.n_tiles;
    if (units > 0x7fffffff) return -2;
    const int sms = num_sms() * C::CTAS, kblocks = (d.K + 127) / 128;
    sp.split = 1;
    if (!d.groups)
        while (sp.split < 8 && units * sp.split * 2 <= sms && kblocks >= sp.split * 4) sp.split *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(sp.split > 1 ? units * sp.split : units < sms ? units : sms));
    cfg.blockDim = dim3(kSmallThreads);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = sp.split;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k, tw, sp) == cudaSuccess ? 0 : -5;
}

template <int BN, bool VEC, bool ROWS, bool PAIR>
int launch_tiles(const Fp8Gemm& d, cudaStream_t st) {
    using C = TileCfg<BN, VEC, ROWS, PAIR>;
    static bool done[kMaxDevices] = {};
    auto k = fp8_tile_kernel<BN, VEC, ROWS, PAIR>;
    if (!allow_smem(k, C::SMEM, done)) return -5;
    const int es = d.c_dtype == kBF16 ? 2 : 4;
    const bool aligned = !(reinterpret_cast<uintptr_t>(d.c) & 15) && d.ldc * es % 16 == 0 && d.c_stride * es % 16 == 0;
    TileParams p = params(d, C::BM, BN);
    p.vec_out = aligned;
    CUtensorMap ta, tb, tc;
    memset(&tc, 0, sizeof(tc));
    if (!map_codes2(&ta, d.a, d.K, d.a_rows, d.lda, 128)) return -2;
    if (!map_codes3(&tb, d.b, d.K, d.N, d.ldb, ROWS ? d.groups : 1, d.b_stride, C::BROWS)) return -2;
    // a TMA store clips rows to whole 16-byte pieces, so ragged ones go another way
    p.tma_out = aligned && (long long)d.N * es % 16 == 0 &&
                map_out(&tc, d.c, d.c_dtype, d.N, d.M, d.ldc, d.group_k ? d.groups : 1, d.c_stride);
    long long units = (long long)p.m_tiles * p.n_tiles;
    if (ROWS) units = ((long long)p.m_tiles + d.groups) * p.n_tiles;  // at most
    else if (d.groups) units *= d.groups;
    if (units > 0x7fffffff) return -2;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    // (a tile's group of rows or of k-blocks is not split)
    if (C::SPLITS && !d.groups)
        while (p.split < 8 && units * p.split * 2 <= num_sms() && (d.K + 127) / 128 >= p.split * 4) p.split *= 2;
    at.val.clusterDim.x = PAIR ? 2 : p.split;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    // one CTA an SM; of pairs as many as find two SMs of one cluster
    long long slots = num_sms();
    if (PAIR) {
        static int pairs[kMaxDevices] = {};
        int dev = 0;
        cudaGetDevice(&dev);
        if (pairs[dev] == 0) {
            cfg.gridDim = dim3(2);
            if (cudaOccupancyMaxActiveClusters(&pairs[dev], k, &cfg) != cudaSuccess || pairs[dev] < 1) return -5;
        }
        slots = pairs[dev];
    }
    if (p.split > 1) cfg.gridDim = dim3((unsigned)(units * p.split));  // one tile a cluster
    else cfg.gridDim = dim3((unsigned)((units < slots ? units : slots) * (PAIR ? 2 : 1)));
    return cudaLaunchKernelEx(&cfg, k, ta, tb, tc, p) == cudaSuccess ? 0 : -5;
}

}  // namespace

int fp8_gemm(const Fp8Gemm& d, cudaStream_t st) {
    if (d.M < 0 || d.N < 0 || d.K < 0 || d.groups < 0 || (d.c_dtype != kF32 && d.c_dtype != kBF16)) return -1;
    if (d.groups > 1024) return -2;
    if (d.M == 0 || d.N == 0) return 0;
    if (!d.c || d.ldc < d.N) return -1;
    if (d.groups && (!d.offsets || !d.counts)) return -1;
    if (d.K == 0) {  // an empty sum (a weight gradient of no tokens)
        fp8_zero_kernel<<<dim3(64, d.groups ? d.groups : 1), 256, 0, st>>>(d);
        return cudaGetLastError() == cudaSuccess ? 0 : -5;
    }
    if (!d.a || !d.sa || !d.b || !d.sb) return -1;
    auto codes = [](const void* p, long long ld, int cols) {
        return !(reinterpret_cast<uintptr_t>(p) & 15) && ld % 16 == 0 && ld >= cols;
    };
    if (!codes(d.a, d.lda, d.K) || !codes(d.b, d.ldb, d.K) || d.b_stride % 16) return -1;
    const int kb = (d.K + 127) / 128;
    if (d.ld_sa < d.a_rows || d.ld_sb < (d.b_rows ? d.N : kb)) return -1;
    if (d.rows && d.row_div <= 0) return -1;
    if (d.a_rows <= 0) return -1;
    const int sms = num_sms();
    const int rows = d.groups && !d.group_k ? (d.M + d.groups - 1) / d.groups : d.M;
    // Few rows: the weights' stream bounds the product. Of groups the host knows
    // the rows of C, padding included, not their numbers, so segments that start
    // on multiples of 128 count as full ones and take the tiles (608 x 4 of 64
    // experts, 1024 x 2048, 38 rows each: 94 us there, 40 without padding).
    // (One product of 4096 x
    // 4096: 16 rows 8.3 us here and 9.7 on tiles, 24 rows 9.4 and 10.5, 48 rows
    // 11.1 and 10.1; groups of 1024 x 2048 with 38 rows on average 40 us and 92,
    // with 100 rows 75 and 110, of 1024 x 1024 with 112 rows 19.8 and 22.3.)
    if (!d.group_k && rows <= (d.groups ? 128 : 32)) {
        if (rows <= 16) return d.b_rows ? launch_small<16, true>(d, st) : launch_small<16, false>(d, st);
        return d.b_rows ? launch_small<32, true>(d, st) : launch_small<32, false>(d, st);
    }
    // The tile's width with the least rounds x time of a k-block, which goes
    // about as width + 64.
    const long long m_tiles = (d.M + 127) / 128 * (long long)(d.group_k ? d.groups : 1);
    auto cost = [&](int bn) { return (m_tiles * ((d.N + bn - 1) / bn) + sms - 1) / sms * (bn + 64); };
    if (d.groups && !d.group_k)
        return cost(128) < cost(256) ? launch_tiles<128, false, true, false>(d, st)
                                     : launch_tiles<256, false, true, false>(d, st);
    if (d.b_rows) {
        if (cost(192) < cost(256) && cost(192) <= cost(128)) return launch_tiles<192, true, false, false>(d, st);
        return cost(128) < cost(256) ? launch_tiles<128, true, false, false>(d, st)
                                     : launch_tiles<256, true, false, false>(d, st);
    }
    // Pairs of CTAs read a third less from L2, but wait for one another: from
    // two rounds of tiles on (8192 x 4096 x 4096: 133 us against 139; 2048 x
    // 2048 x 2048, under one round: 15.1 against 14.2).
    const long long pairs = (long long)((d.M + 255) / 256) * ((d.N + 255) / 256);
    if (pairs >= sms) return launch_tiles<256, false, false, true>(d, st);
    return cost(128) < cost(256) ? launch_tiles<128, false, false, false>(d, st)
                                 : launch_tiles<256, false, false, false>(d, st);
}

}  // namespace nsb
