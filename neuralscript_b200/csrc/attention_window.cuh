// What the kernels of attention with a window share: which rows a block has,
// which keys a query sees, and which tiles of keys (of queries) a tile needs.
#pragma once
#include "attention_cache.h"

namespace nsb {

// Rows [first, first + rows) of a sequence of n rows that starts at row0 of
// the packed buffer; n = 0: no such tile.
struct Rows {
    long long row0;
    int n, first;
};

// The tile-th tile of `rows` rows, counted over all sequences. Offsets outside
// [0, T], or falling ones, are cut to it and reported. Called by whole warps;
// every warp finds it by itself.
__device__ __forceinline__ Rows find_rows(const WindowDesc& d, int tile, int rows) {
    if (!d.offsets) return Rows{0, d.T, tile * rows};
    const int lane = threadIdx.x & 31;
    for (int b0 = 0; b0 < d.B; b0 += 32) {
        int lo = 0, n = 0;
        if (b0 + lane < d.B) {
            const int x = d.offsets[b0 + lane], y = d.offsets[b0 + lane + 1];
            lo = min(max(x, 0), d.T);
            n = min(max(y, lo), d.T) - lo;
            if (x < 0 || y < x || y > d.T) atomicCAS(d.err, 0, kErrBadIndex);
        }
        const int own = (n + rows - 1) / rows;
        int sum = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += u;
        }
        const unsigned past = __ballot_sync(0xffffffffu, sum > tile);
        if (past) {
            const int src = __ffs(past) - 1;
            return Rows{__shfl_sync(0xffffffffu, lo, src), __shfl_sync(0xffffffffu, n, src),
                        (tile - __shfl_sync(0xffffffffu, sum - own, src)) * rows};
        }
        tile -= __shfl_sync(0xffffffffu, sum, 31);
    }
    return Rows{0, 0, 0};
}

__device__ __forceinline__ bool sees(const WindowDesc& d, int i, int j) {
    return j <= i && (d.window == 0 || i - j < d.window || j < d.sinks);
}

// Tiles of `size` keys that queries [q0, q1) see any of: those of the first
// `sinks` keys, then those from the first query's window to the last query.
struct KeyTiles {
    int front, skip, count;
    __device__ __forceinline__ KeyTiles(const WindowDesc& d, int q0, int q1, int size) {
        const int end = (q1 + size - 1) / size;
        const int lo = d.window && q0 >= d.window ? (q0 - d.window + 1) / size : 0;
        front = min(min(lo, end), d.sinks / size + (d.sinks % size != 0));
        skip = lo - front;
        count = end - skip;
    }
    __device__ __forceinline__ int at(int x) const { return x < front ? x : x + skip; }
};

// Whether queries [q0, q1) see few keys: two tiles of 128, or a window and first
// tokens of 64 together. D = rowdot(dout, out) from an `out` in bf16 is off by up
// to 2^-9 |dout| |out|, and with it every dS of the row by P times that. Where rows
// see few keys, dS itself is small (one key: 0) and that is most of its error, so
// there a pass before sums dS: as the weights P add up to 1, the sum over a row of
// P (dP - D) is what D is short of. Error of dq against 64 bits, in the norm, with
// and without, 700 rows on the tensor cores: a window of 2 and 1 first token 2.4e-3
// and 3.2e-3 (on the fp32 units 1.7e-3 and 2.7e-3), 9 and 4 2.4e-3 and 2.5e-3, 50
// and 3 2.37e-3 and 2.42e-3; 100 and 28 2.38e-3 and 2.40e-3, where the pass would
// take 23 of 167 us (8192 rows of 16 heads of 64).
constexpr int kFewTiles = 2;
constexpr int kFewKeys = 64;
__device__ __forceinline__ bool few_keys(const WindowDesc& d, int q0, int q1) {
    return KeyTiles(d, q0, q1, 128).count <= kFewTiles || (d.window && (long long)d.window + d.sinks <= kFewKeys);
}

// End of the tiles of `size` queries that see any of the keys [k0, k0 + size).
__device__ __forceinline__ int query_tiles_end(const WindowDesc& d, int k0, int n, int size) {
    const int end = (n + size - 1) / size;
    if (d.window == 0 || k0 < d.sinks) return end;
    const long long past = (long long)k0 + size - 1 + d.window;  // first query that no longer sees the last key
    return (int)min((long long)end, (past + size - 1) / size);
}

}  // namespace nsb
