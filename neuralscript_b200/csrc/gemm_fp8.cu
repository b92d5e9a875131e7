// Products of 8-bit floating point codes with a scale for each block of 128
// (no counterpart in the reference):
//
//   C[m,n] = sum over blocks b of 128 k of  sa(m,b) sb(n,b) sum_k A[m,k] B[n,k]
#include <cuda_fp8.h>

#include "fp8.h"
#include "gemm.h"

namespace nsb {

namespace {

__device__ __forceinline__ float value(uint8_t c) {
    __nv_fp8_e4m3 t;
    t.__x = c;
    return (float)t;
}

// 64 x 64 outputs a block of 256 threads, blocks of 128 k summed apart.
__global__ void __launch_bounds__(256) fp8_simple_kernel(const Fp8Gemm d) {
    __shared__ float As[16][65], Bs[16][65];
    const int g = blockIdx.z;
    int m0 = blockIdx.y * 64, m_end = d.M;
    long long k0 = 0, k1 = d.K;
    const uint8_t* b = d.b;
    const float* sb = d.sb;
    char* c = reinterpret_cast<char*>(d.c);
    if (d.groups && d.group_k) {
        k0 = d.offsets[g];
        k1 = min((long long)d.K, k0 + d.counts[g]);
        c += g * d.c_stride * (d.c_dtype == kBF16 ? 2 : 4);
    } else if (d.groups) {
        m0 += d.offsets[g];
        m_end = min(d.M, d.offsets[g] + d.counts[g]);
        b += g * d.b_stride;
        sb += g * d.sb_stride;
    }
    if (m0 >= m_end) return;
    const int n0 = blockIdx.x * 64, tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    float acc[4][4] = {};
    for (long long kb = k0 / 128; kb * 128 < k1; kb++) {
        float part[4][4] = {};
        for (int ks = 0; ks < 128; ks += 16) {
            for (int e = threadIdx.x; e < 1024; e += 256) {
                const int kk = e % 16, i = e / 16;
                const long long k = kb * 128 + ks + kk;
                const int m = m0 + i, n = n0 + i;
                long long am = m;
                if (d.rows && m < m_end) am = d.rows[m] < 0 ? -1 : d.rows[m] / d.row_div;
                As[kk][i] = m < m_end && k < k1 && am >= 0 ? value(d.a[am * d.lda + k]) : 0.f;
                Bs[kk][i] = n < d.N && k < k1 ? value(b[(long long)n * d.ldb + k]) : 0.f;
            }
            __syncthreads();
            for (int kk = 0; kk < 16; kk++)
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int j = 0; j < 4; j++) part[i][j] = fmaf(As[kk][ty + 16 * i], Bs[kk][tx + 16 * j], part[i][j]);
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
                if (m >= m_end || n >= d.N) continue;
                long long am = m;
                if (d.rows) am = d.rows[m] < 0 ? -1 : d.rows[m] / d.row_div;
                if (am < 0) continue;
                const float s = d.sa[kb * d.ld_sa + am] *
                                (d.b_rows ? sb[kb * d.ld_sb + n] : sb[(long long)(n / 128) * d.ld_sb + kb]);
                acc[i][j] = fmaf(part[i][j], s, acc[i][j]);
            }
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
            if (m >= m_end || n >= d.N) continue;
            const size_t at = (size_t)m * d.ldc + n;
            if (d.c_dtype == kBF16) reinterpret_cast<__nv_bfloat16*>(c)[at] = f2bf(acc[i][j]);
            else reinterpret_cast<float*>(c)[at] = acc[i][j];
        }
}

__global__ void fp8_zero_kernel(const Fp8Gemm d) {
    const size_t n = (size_t)d.M * d.N;
    for (size_t i = blockIdx.x * (size_t)blockDim.x + threadIdx.x; i < n; i += (size_t)gridDim.x * blockDim.x) {
        const size_t at = blockIdx.y * (size_t)d.c_stride + i / d.N * d.ldc + i % d.N;
        if (d.c_dtype == kBF16) reinterpret_cast<__nv_bfloat16*>(d.c)[at] = f2bf(0.f);
        else reinterpret_cast<float*>(d.c)[at] = 0.f;
    }
}

}  // namespace

int fp8_gemm(const Fp8Gemm& d, cudaStream_t st) {
    if (d.M < 0 || d.N < 0 || d.K < 0 || d.groups < 0 || (d.c_dtype != kF32 && d.c_dtype != kBF16)) return -1;
    if (d.groups > 1024) return -2;
    if (d.M == 0 || d.N == 0) return 0;
    if (!d.c || d.ldc < d.N) return -1;
    if (d.K == 0) {  // an empty sum (a weight gradient of no tokens)
        fp8_zero_kernel<<<dim3(64, d.group_k ? d.groups : 1), 256, 0, st>>>(d);
        return cudaGetLastError() == cudaSuccess ? 0 : -5;
    }
    if (!d.a || !d.sa || !d.b || !d.sb) return -1;
    auto codes = [](const void* p, long long ld, int cols) {
        return !(reinterpret_cast<uintptr_t>(p) & 15) && ld % 16 == 0 && ld >= cols;
    };
    if (!codes(d.a, d.lda, d.K) || !codes(d.b, d.ldb, d.K) || d.b_stride % 16) return -1;
    const int kb = (d.K + 127) / 128;
    if (d.ld_sa < d.a_rows || d.ld_sb < (d.b_rows ? d.N : kb)) return -1;
    if (d.groups && (!d.offsets || !d.counts)) return -1;
    if (d.rows && d.row_div <= 0) return -1;
    const dim3 grid((d.N + 63) / 64, (d.M + 63) / 64, d.groups ? d.groups : 1);
    fp8_simple_kernel<<<grid, 256, 0, st>>>(d);
    return cudaGetLastError() == cudaSuccess ? 0 : -5;
}

}  // namespace nsb
