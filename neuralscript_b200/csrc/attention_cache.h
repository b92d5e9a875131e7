// Attention that answers token by token: rotary positions, a paged cache of
// keys and values, attention of one new token over it, and attention with a
// sliding window and a few first tokens that stay visible, for prompts and
// training. Device pointers; deterministic, without atomics on results.
//
// Heads: a tensor [rows, heads, dh] has its own strides from row to row and
// from head to head, the dh columns of a head lie side by side. Hq query
// heads share Hkv key heads, Hq / Hkv neighbours one.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "common.cuh"

namespace nsb {

constexpr int kMaxAxes = 4;         // axes of a position
constexpr int kTurnMaxHead = 1024;  // columns of a head that is rotated
constexpr int kAttnMaxHead = 128;   // columns of a head in attention
constexpr int kPagedMaxBatch = 8192;
constexpr int kWindowMaxRows = 1 << 30;

// A tensor of heads: row t, head h at p + t * row + h * head.
struct Heads {
    void* p = nullptr;
    long long row = 0, head = 0;
};

// A cache: key (or value) `place` of page n, head h at
// p + n * page + place * slot + h * head.
struct Pages {
    void* p = nullptr;
    long long page = 0, slot = 0, head = 0;
};

// Rotation of the first 2 * n columns of a head by the angles pos * freq:
// pair i is (i, i + n), or (2 i, 2 i + 1) where interleaved, and belongs to
// the first axis whose `end` is above it.
struct Turn {
    const int* pos = nullptr;  // [axes, ld_pos]
    long long ld_pos = 0;
    int axes = 1;
    int end[kMaxAxes] = {};
    const float* freq = nullptr;  // [n] radians a position
    int n = 0;
    int interleaved = 0;
    float scale = 1.f;
    float sign = 1.f;  // -1: the gradient
};

int rope(const Turn& t, int dtype, const Heads& x, const Heads& y, int T, int H, int dh, cudaStream_t s);

struct AppendDesc {
    int dtype = kF32;
    int T = 0, dh = 0, Hkv = 0, Hq = 0;
    Heads k, v, q, q_out;          // q, q_out: none, or rotated beside the keys
    const int *seq = nullptr, *at = nullptr;  // [T] sequence (negative: none) and place of every token
    const int* table = nullptr;    // [B, ld_table] pages of every sequence
    long long ld_table = 0;
    int B = 0, width = 0;          // sequences, and pages that the table has for each
    int pages = 0, page = 0;       // pages of the cache, places in one
    Pages kc, vc;
    Turn turn;                     // n = 0: keys and queries as they are
    int* err = nullptr;
};
int kv_append(const AppendDesc& d, cudaStream_t s);

struct PagedDesc {
    int dtype = kF32;
    int B = 0, Hq = 0, Hkv = 0, dh = 0;
    Heads q, out;
    Pages kc, vc;
    int pages = 0, page = 0;
    const int* table = nullptr;
    long long ld_table = 0;
    int width = 0;
    const int* lens = nullptr;  // [B] keys of every sequence, the new token's among them
    int window = 0, sinks = 0;  // window 0: all
    float scale = 1.f;
    float* lse = nullptr;  // [B, Hq]
    void* workspace = nullptr;
    size_t workspace_bytes = 0;
    int* err = nullptr;
};
size_t attention_paged_workspace(int B, int Hq, int Hkv, int dh);
int attention_paged(const PagedDesc& d, cudaStream_t s);
int attention_paged_launches();

struct WindowDesc {
    int dtype = kF32;
    int T = 0, Hq = 0, Hkv = 0, dh = 0;
    const int* offsets = nullptr;  // [B + 1]: sequence b has rows [offsets[b], offsets[b + 1]); none: one of T rows
    int B = 1;
    int window = 0, sinks = 0;
    float scale = 1.f;
    Heads q, k, v, out;
    float* lse = nullptr;  // [Hq, ld_lse]
    long long ld_lse = 0;
    Heads dout, dq, dk, dv;   // backward
    void* workspace = nullptr;
    size_t workspace_bytes = 0;
    float* dvec = nullptr;    // in the workspace: [Hq, T] rowdot(dout, out)
    float* parts = nullptr;   // on the tensor cores also sums of tiles that several blocks share
    int* err = nullptr;
};
int attention_window(const WindowDesc& d, cudaStream_t s);
// on the tensor cores (attention_window_tc.cu): bf16, 16-byte rows
bool attention_window_tc_supported(const WindowDesc& d);
int attention_window_tc(const WindowDesc& d, cudaStream_t s);
bool attention_window_bwd_tc_supported(const WindowDesc& d);
size_t attention_window_bwd_tc_parts(int dh);
int attention_window_bwd_tc(const WindowDesc& d, cudaStream_t s);
size_t attention_window_bwd_workspace(int T, int Hq, int Hkv, int dh, int dtype);
int attention_window_bwd(const WindowDesc& d, cudaStream_t s);
int attention_window_bwd_launches(const WindowDesc& d);

}  // namespace nsb
