// Mixture of experts with k experts a token: routing, the order of the
// (token, choice) pairs by expert, and the weighted sum of the experts'
// outputs, each with its gradient. Device pointers; deterministic.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "common.cuh"

namespace nsb {

constexpr int kTopkMaxE = 1024;  // experts
constexpr int kTopkMaxK = 32;    // experts a token (one lane of a warp each)

struct RouteDesc {
    const void* logits = nullptr;
    int dtype = kF32;
    long long ld = 0;
    int M = 0, E = 0, k = 0;
    int sigmoid = 0;               // else softmax
    const float* bias = nullptr;   // [E], selection only
    const uint8_t* active = nullptr;  // [E], 0 = dead
    int groups = 1, topk_groups = 1;
    int renorm = 1;
    float scale = 1.f;
    // set by the launch: 16-byte rows of logits; bias and active on 16-byte
    // boundaries; lanes that hold a group (0: groups do not fall on whole lanes)
    int vec = 0, vec_e = 0, lanes = 0;
};

int moe_topk_route(const RouteDesc& d, int* idx, float* w, cudaStream_t s);
int moe_topk_route_bwd(const RouteDesc& d, const float* dw, const int* idx, void* dlogits, long long ld_d,
                       cudaStream_t s);

// Rows that the ordered pairs take at most.
size_t moe_dispatch_rows(long long M, int k, int E, int align);
int moe_dispatch(const int* idx, int M, int k, int E, int align, int* offsets, int* counts, int* rows, int* pos,
                 cudaStream_t s);

// o has R rows; a place past them, and in the gradient a pair past the last,
// is left out and goes into err.
int moe_combine(const void* o, int dtype, long long ld_o, int R, const int* pos, const float* w, int M, int k, int D,
                void* y, long long ld_y, int* err, cudaStream_t s);
int moe_combine_bwd(const void* dy, const void* o, int dtype, long long ld_dy, long long ld_o, const int* rows,
                    const int* pos, const float* w, int M, int k, int R, int D, void* d_o, long long ld_do, float* dw,
                    int* err, cudaStream_t s);

}  // namespace nsb
