// Quantisation to 8-bit floating point (e4m3) with a scale for each block of
// 128 (no counterpart in the reference).
//
//   scale = max(max |x| * (1 / 448), 2^-100),  code = e4m3(x * (1 / scale))
//
// 448 is the largest finite e4m3 value; its reciprocal is rounded to fp32, a
// multiplication in place of a division, for the quotient's last bit does not
// matter: code and scale are read back together. The floor keeps 1 / scale finite for
// blocks of zeros and of numbers so small that their quotient underflows. A
// NaN becomes a NaN code and leaves its block's scale alone; an infinity
// makes the scale infinite and the whole block NaN when it is read back.
//
// One block of threads takes 128 x 128 values, so that one read of x serves
// both orientations and all three forms of scales. A half-warp owns 4 rows, a
// lane 8 columns of them (one 16-byte load of bf16 a row), so row maxima are 4
// shuffles and the 4 codes of a column are one word of the transpose, which
// goes through 16 KB of shared memory, the words of a column exchanged
// (word ^ 2 (column / 8)) so that neither side has bank conflicts.
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include <type_traits>

#include "fp8.h"
#include "gemm.h"

namespace nsb {

namespace {

constexpr unsigned kAll = 0xffffffffu;
constexpr float kTopInv = 1.f / 448.f;
constexpr float kFloor = 7.888609052210118e-31f;  // 2^-100

__device__ __forceinline__ float scale_of(float amax) { return fmaxf(amax * kTopInv, kFloor); }

__device__ __forceinline__ uint32_t code4(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
}

// the same of four values times k, two at a time
__device__ __forceinline__ uint32_t code4(float a, float b, float c, float d, float k) {
    const uint64_t kk = f2_pack(k, k);
    f2_unpack(f2_mul(f2_pack(a, b), kk), a, b);
    f2_unpack(f2_mul(f2_pack(c, d), kk), c, d);
    return code4(a, b, c, d);
}

__device__ __forceinline__ void store8(uint8_t* dst, uint2 v, int n) {
    if (n >= 8) {
        *reinterpret_cast<uint2*>(dst) = v;
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; i++)
        if (i < n) dst[i] = (uint8_t)((i < 4 ? v.x >> 8 * i : v.y >> 8 * (i - 4)) & 0xff);
}

__device__ __forceinline__ float ex2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// the smaller one, NaN where either is
__device__ __forceinline__ float min_nan(float a, float b) {
    float d;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// x Phi(x) without erff's branches: Phi(-a) = erfc(z) / 2 for z = a / sqrt(2),
// erfc(z) = exp(-z^2) erfcx(z), and erfcx(z) = t P(t) with t = 1 / (1 + 0.38 z)
// and a polynomial of degree 6 fitted for this code (Lawson-weighted least
// squares over z in [0, 10]), so that nothing cancels on the negative side.
// Largest relative error, measured against 64 bits: 1.5e-6 for |x| up to 1,
// 2.1e-6 down to -4, 6.5e-6 to -8, 1.9e-5 to -13: the polynomial's 1.4e-6, and
// z^2 log2(e), whose roundings the exponential multiplies by z^2. Below about
// -13.2 the result is 0, as its code is: 2^-100 is a block's smallest scale.
// Two values at a time on packed fp32 pairs, which halves the FMA
// instructions that bound this pass.
// a stops at 20, where Phi(-a) is long 0 in fp32, so that +inf meets no
// inf * 0 and stays +inf; -inf gives NaN as it does in x Phi(x), and NaN NaN.
__device__ __forceinline__ void gelu_tail2(float& x0, float& x1) {
    const uint64_t a = f2_pack(fabsf(min_nan(x0, 20.f)), fabsf(min_nan(x1, 20.f)));
    const uint64_t z = f2_mul(a, f2_pack(0.70710678f, 0.70710678f));
    float d0, d1, e0, e1;
    f2_unpack(f2_fma(z, f2_pack(0.38f, 0.38f), f2_pack(1.f, 1.f)), d0, d1);
    f2_unpack(f2_mul(f2_mul(z, z), f2_pack(-1.44269504f, -1.44269504f)), e0, e1);
    const uint64_t t = f2_pack(rcp_approx(d0), rcp_approx(d1));
    const uint64_t e = f2_pack(ex2_approx(e0), ex2_approx(e1));
    auto c = [](float v) { return f2_pack(v, v); };
    uint64_t q = c(-0.125199478f);
    q = f2_fma(q, t, c(0.335197723f));
    q = f2_fma(q, t, c(-0.068613310f));
    q = f2_fma(q, t, c(0.246798871f));
    q = f2_fma(q, t, c(0.181039411f));
    q = f2_fma(q, t, c(0.216480016f));
    q = f2_fma(q, t, c(0.214295747f));
    q = f2_mul(q, f2_mul(t, e));
    f2_unpack(f2_fma(f2_mul(a, c(-0.5f)), q, f2_pack(fmaxf(x0, 0.f), fmaxf(x1, 0.f))), x0, x1);
}

template <int ACT>
__device__ __forceinline__ float activate(float x) {
    if constexpr (ACT == kSilu) return x * rcp_approx(1.f + ex2_approx(x * -1.44269504f));
    else return act_fwd(x, ACT);
}

constexpr int kThreads = 512;

// Blocks stay and take tiles in turn; of bf16 the next tile's values are on
// their way into shared memory (every thread fetches the pieces that it will
// read itself) while this one's are worked on (16384 x 2048 behind a GELU, both
// orientations: 52 -> 47 us, of which GELU's two special-function operations a
// value take 15).
template <typename T, bool BLOCK, bool VEC, int ACT>
__global__ void __launch_bounds__(kThreads, 2) quantize_kernel(const QuantDesc d, int cb, int tiles) {
    constexpr bool AHEAD = VEC && sizeof(T) == 2;
    __shared__ __align__(8) uint32_t tile[128 * 32];  // [column][word of 4 rows]
    __shared__ float part[16][128];      // column maxima of the 16 warps
    __shared__ float inv[128];
    extern __shared__ uint4 ahead[];     // [2][4][kThreads]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int half = warp * 2 + (lane >> 4);  // 0..31: rows 4 half ..
    const int cl = lane & 15;
    auto source = [&](int r) -> long long {  // row of x behind row r, -1 for none
        if (r >= d.M) return -1;
        if (!d.rows) return r;
        const int at = d.rows[r];
        if (at < 0) return -1;
        const int src = d.row_div ? at / d.row_div : r;
        if (src < d.x_rows) return src;
        if (d.err) atomicCAS(d.err, 0, kErrBadIndex);
        return -1;
    };
    auto fetch = [&](int t, int b) {
        const int r0 = t / cb * 128 + half * 4, c0 = t % cb * 128 + cl * 8;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const long long src = source(r0 + i);
            if (src >= 0 && c0 + 8 <= d.K)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                                 (uint32_t)__cvta_generic_to_shared(ahead + (b * 4 + i) * kThreads + threadIdx.x)),
                             "l"(reinterpret_cast<const T*>(d.x) + src * d.ld + c0)
                             : "memory");
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    if (AHEAD && blockIdx.x < tiles) fetch(blockIdx.x, 0);
    int buf = 0;
    for (int t = blockIdx.x; t < tiles; t += gridDim.x, buf ^= 1) {
        const int bx = t % cb, by = t / cb;
        const int r0 = by * 128 + half * 4, c0 = bx * 128 + cl * 8;
        if (AHEAD) {
            if (t + (int)gridDim.x < tiles) {
                fetch(t + gridDim.x, buf ^ 1);
                asm volatile("cp.async.wait_group 1;" ::: "memory");
            } else {
                asm volatile("cp.async.wait_group 0;" ::: "memory");
            }
        }
        float v[4][8];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const long long src = source(r0 + i);
            const bool in = src >= 0;
            const T* p = reinterpret_cast<const T*>(d.x) + src * d.ld + c0;
            if (VEC && in && c0 + 8 <= d.K) {
                if constexpr (sizeof(T) == 2) {
                    const uint4 t = ahead[(buf * 4 + i) * kThreads + threadIdx.x];
                    const __nv_bfloat16* h = reinterpret_cast<const __nv_bfloat16*>(&t);
#pragma unroll
                    for (int j = 0; j < 8; j++) v[i][j] = bf2f(h[j]);
                } else {
                    const float4 t0 = reinterpret_cast<const float4*>(p)[0], t1 = reinterpret_cast<const float4*>(p)[1];
                    v[i][0] = t0.x, v[i][1] = t0.y, v[i][2] = t0.z, v[i][3] = t0.w;
                    v[i][4] = t1.x, v[i][5] = t1.y, v[i][6] = t1.z, v[i][7] = t1.w;
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++) v[i][j] = in && c0 + j < d.K ? (float)p[j] : 0.f;
            }
        }
        if (ACT) {
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    if constexpr (ACT == kGelu) {
                        gelu_tail2(v[i][j], v[i][j + 1]);
                    } else {
                        v[i][j] = activate<ACT>(v[i][j]);
                        v[i][j + 1] = activate<ACT>(v[i][j + 1]);
                    }
                }
        }
        if constexpr (BLOCK) {
            float m = 0.f;
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 8; j++) m = fmaxf(m, fabsf(v[i][j]));
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kAll, m, o));
            if (lane == 0) part[0][warp] = m;
            __syncthreads();
#pragma unroll
            for (int q = 0; q < kThreads / 32; q++) m = fmaxf(m, part[0][q]);
            const float s = scale_of(m), k = 1.f / s;
            if (threadIdx.x == 0) {
                if (d.s) d.s[by * d.ld_s + bx] = s;
                if (d.st) d.st[bx * d.ld_st + by] = s;
            }
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 8; j++) v[i][j] *= k;
            if (d.q) {
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (r0 + i < d.M)
                        store8(d.q + (size_t)(r0 + i) * d.ld_q + c0,
                               make_uint2(code4(v[i][0], v[i][1], v[i][2], v[i][3]),
                                          code4(v[i][4], v[i][5], v[i][6], v[i][7])),
                               d.K - c0);
            }
            if (!d.qt) {
                __syncthreads();  // (part is written again)
                continue;
            }
#pragma unroll
            for (int j = 0; j < 8; j++)
                tile[(cl * 8 + j) * 32 + (half ^ (cl * 2))] = code4(v[0][j], v[1][j], v[2][j], v[3][j]);
        } else {
            if (d.q) {
                // lane i of the half-warp turns the maximum of row i into its scale
                float mine = 0.f;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    float m = 0.f;
#pragma unroll
                    for (int j = 0; j < 8; j += 2) m = max3(m, fabsf(v[i][j]), fabsf(v[i][j + 1]));
#pragma unroll
                    for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kAll, m, o));
                    if (cl == i) mine = m;
                }
                const float s = scale_of(mine), inverse = 1.f / s;
                if (cl < 4 && r0 + cl < d.M) d.s[bx * d.ld_s + r0 + cl] = s;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float k = __shfl_sync(kAll, inverse, (lane & 16) + i);
                    if (r0 + i < d.M)
                        store8(d.q + (size_t)(r0 + i) * d.ld_q + c0,
                               make_uint2(code4(v[i][0], v[i][1], v[i][2], v[i][3], k),
                                          code4(v[i][4], v[i][5], v[i][6], v[i][7], k)),
                               d.K - c0);
                }
            }
            if (!d.qt) continue;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                float m = max3(0.f, fabsf(v[0][j]), fabsf(v[1][j]));
                m = max3(m, fabsf(v[2][j]), fabsf(v[3][j]));
                m = fmaxf(m, __shfl_xor_sync(kAll, m, 16));
                if (lane < 16) part[warp][j * 16 + cl] = m;  // column cl * 8 + j
            }
            __syncthreads();
            if (threadIdx.x < 128) {
                float m = 0.f;
#pragma unroll
                for (int q = 0; q < kThreads / 32; q++) m = fmaxf(m, part[q][threadIdx.x]);
                const float s = scale_of(m);
                inv[threadIdx.x] = 1.f / s;
                const int c = bx * 128 + (threadIdx.x & 15) * 8 + (threadIdx.x >> 4);
                if (c < d.K) d.st[by * d.ld_st + c] = s;
            }
            __syncthreads();
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float k = inv[j * 16 + cl];
                tile[(cl * 8 + j) * 32 + (half ^ (cl * 2))] =
                    code4(v[0][j], v[1][j], v[2][j], v[3][j], k);
            }
        }
        __syncthreads();
        const int r = by * 128 + cl * 8;
#pragma unroll
        for (int c = half; c < 128; c += kThreads / 16) {
            const int col = bx * 128 + c;
            if (col < d.K && r < d.M)
                store8(d.qt + (size_t)col * d.ld_qt + r,
                       *reinterpret_cast<const uint2*>(tile + c * 32 + ((cl * 2) ^ ((c >> 3) * 2))), d.M - r);
        }
        __syncthreads();  // the next tile's words take their place
    }
}

template <bool BLOCK>
int quantize(const QuantDesc& d, cudaStream_t st) {
    const bool f = d.dtype == kF32;
    if (d.M < 0 || d.K <= 0 || (!f && d.dtype != kBF16) || d.ld < d.K || d.act < 0 || d.act > kGeluMoe) return -1;
    if (d.rows && d.row_div < 0) return -1;
    if (d.x_rows < (d.rows && d.row_div ? 0 : d.M)) return -1;
    if (d.M == 0) return 0;  // (what has no elements has no address)
    if (!d.x || (!d.q && !d.qt)) return -1;
    auto codes = [](const void* p, long long ld, int cols) {
        return !(reinterpret_cast<uintptr_t>(p) & 15) && ld % 16 == 0 && ld >= cols;
    };
    const int rb = (d.M + 127) / 128, cb = (d.K + 127) / 128;
    if (d.q && (!codes(d.q, d.ld_q, d.K) || !d.s || d.ld_s < (BLOCK ? cb : d.M))) return -1;
    if (d.qt && (!codes(d.qt, d.ld_qt, d.M) || !d.st || d.ld_st < (BLOCK ? rb : d.K))) return -1;
    if ((long long)rb * cb > 0x7fffffff) return -2;
    const int tiles = rb * cb, most = 2 * num_sms(), grid = tiles < most ? tiles : most;
    const bool vec = !(reinterpret_cast<uintptr_t>(d.x) & 15) && d.ld * (f ? 4 : 2) % 16 == 0;
    bool ok = true;
    auto go = [&](auto act) {
        constexpr int ACT = decltype(act)::value;
        if (f && vec) {
            quantize_kernel<float, BLOCK, true, ACT><<<grid, kThreads, 0, st>>>(d, cb, tiles);
        } else if (f) {
            quantize_kernel<float, BLOCK, false, ACT><<<grid, kThreads, 0, st>>>(d, cb, tiles);
        } else if (!vec) {
            quantize_kernel<__nv_bfloat16, BLOCK, false, ACT><<<grid, kThreads, 0, st>>>(d, cb, tiles);
        } else {
            auto k = quantize_kernel<__nv_bfloat16, BLOCK, true, ACT>;
            constexpr int smem = 8 * kThreads * (int)sizeof(uint4);
            static bool done[kMaxDevices] = {};  // the attribute belongs to the current device
            int dev = 0;
            if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) {
                ok = false;
                return;
            }
            if (!done[dev])
                done[dev] = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) == cudaSuccess;
            k<<<grid, kThreads, smem, st>>>(d, cb, tiles);
        }
    };
    if constexpr (BLOCK) {
        go(std::integral_constant<int, kIdentity>());
    } else {
        switch (d.act) {
            case kRelu: go(std::integral_constant<int, kRelu>()); break;
            case kLeaky: go(std::integral_constant<int, kLeaky>()); break;
            case kSigmoid: go(std::integral_constant<int, kSigmoid>()); break;
            case kTanh: go(std::integral_constant<int, kTanh>()); break;
            case kSilu: go(std::integral_constant<int, kSilu>()); break;
            case kGelu:
            case kGeluMoe: go(std::integral_constant<int, kGelu>()); break;
            default: go(std::integral_constant<int, kIdentity>());
        }
    }
    return cudaGetLastError() == cudaSuccess && ok ? 0 : -5;
}

}  // namespace

int fp8_quantize(const QuantDesc& d, cudaStream_t s) { return quantize<false>(d, s); }
int fp8_quantize_block(const QuantDesc& d, cudaStream_t s) { return quantize<true>(d, s); }

}  // namespace nsb
