// 8-bit floating point (e4m3) with a scale for each block of 128: the
// quantisation and the products. Device pointers.
//
// Codes lie row by row, every row on a 16-byte boundary. Scales of single
// rows are block-major: that of row r and columns [128 b, 128 b + 128) at
// scale[b * ld_scale + r]. Scales of 128 x 128 blocks lie row by row:
// scale[(r / 128) * ld_scale + c / 128].
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "common.cuh"

namespace nsb {

struct QuantDesc {
    const void* x = nullptr;
    int dtype = kF32;
    long long ld = 0;
    int M = 0, K = 0;  // rows of the result (gathered ones with `rows`) and columns
    int act = 0;       // activation applied first
    // Row r of the result is row rows[r] / row_div of x, row r itself where
    // row_div is 0, and zeros for a negative entry, or one past the x_rows rows
    // of x, which goes into err
    const int* rows = nullptr;
    int row_div = 1;
    int x_rows = 0x7fffffff;
    int* err = nullptr;
    uint8_t* q = nullptr;  // [M, ld_q]
    long long ld_q = 0;
    float* s = nullptr;
    long long ld_s = 0;
    uint8_t* qt = nullptr;  // [K, ld_qt]: the transpose, a scale for each 128 along M
    long long ld_qt = 0;
    float* st = nullptr;
    long long ld_st = 0;
};
// A scale for each 1 x 128 of x (q, s) and / or for each 128 x 1 (qt, st).
int fp8_quantize(const QuantDesc& d, cudaStream_t s);
// A scale for each 128 x 128; q and qt hold the same codes.
int fp8_quantize_block(const QuantDesc& d, cudaStream_t s);

struct Fp8Gemm {
    int M = 0, N = 0, K = 0;
    const uint8_t* a = nullptr;  // [a_rows, lda] codes
    long long lda = 0;
    long long a_rows = 0;
    const float* sa = nullptr;  // row scales, block-major
    long long ld_sa = 0;
    const uint8_t* b = nullptr;  // [N, ldb] codes, for each group b_stride further
    long long ldb = 0, b_stride = 0;
    const float* sb = nullptr;  // 128 x 128 scales (b_rows 0) or row scales (1)
    long long ld_sb = 0, sb_stride = 0;
    int b_rows = 0;
    void* c = nullptr;
    int c_dtype = kF32;
    long long ldc = 0, c_stride = 0;
    // groups > 0: group g owns rows [offsets[g], offsets[g] + counts[g]) of C
    // (group_k 0), or sums over those columns of A and B into C + g * c_stride
    // (group_k 1; the offsets are multiples of 128)
    int groups = 0;
    int group_k = 0;
    const int* offsets = nullptr;
    const int* counts = nullptr;
    const int* rows = nullptr;  // row r of the product is row rows[r] / row_div of A
    int row_div = 1;
    int* err = nullptr;
};
int fp8_gemm(const Fp8Gemm& d, cudaStream_t s);

}  // namespace nsb
