// Rotary positions and the write of keys and values into a paged cache.
//
// A pair (x0, x1) of a head's columns, the i-th of n, becomes
//   (x0 cos a - x1 sin a, x1 cos a + x0 sin a),  a = pos * freq[i],
// with pos one of up to four coordinates of the token. The gradient turns
// back by the same angle. A position of 2^31 times a frequency leaves fp32
// no digit behind the point, so the angle is formed in 64 bits in units of a
// whole turn; what is left after the whole turns is within half a turn and
// goes to sincospif in fp32.
//
// Memory-bound: every value is read and written once. A token's angles are
// the same for all of its heads: a block computes them once for a few tokens
// (64 bits, sine and cosine: some 60 instructions a pair) into shared memory
// and its threads then stream the heads, two 16-byte pieces a thread, the
// two halves of its pairs. kv_append is the same kernel with three tensors at
// once (queries, keys, values), whose keys and values go to the cache's
// places.
//
// Bound by HBM, with the issue slots close behind (64 %): 16384 rows of 20 heads
// of 128 columns in bf16, 29.8 us a pass, 5.6 TB/s (a measured copy: 6.5); 9001 x
// 12 x 80 in fp32, 14.6 us, 4.7 TB/s: 1126 blocks are one round, so that all form
// their angles first and HBM waits. Appending 32 tokens: 3.1 us, a launch (fp32
// 3.2); 8000 tokens of 8 heads of 64: 8.1 us, 4.1 TB/s: one round of blocks and 122
// more, whose chain (place of the token, angles, heads) passes by itself; in fp32,
// twice the bytes, 10.6 us, 6.2 TB/s.
#include <cuda_bf16.h>

#include <type_traits>

#include "attention_cache.h"
#include "gemm.h"

namespace nsb {

namespace {

constexpr int kTurnThreads = 256;
constexpr int kTurnTokens = 8;  // most tokens of a block
constexpr int kTurnMaxRow = 1 << 26;  // columns of a token, all heads

struct TurnJob {
    const void* src;
    long long src_row, src_head;
    void* dst;
    long long dst_row, dst_head, dst_page;  // with pages: row = place in a page
    int first;                              // heads of the jobs before
    int turn, paged;
};

// Division of numbers below 2^31 by d: m = ceil(2^p / d) with p = 31 + ceil(log2 d)
// gives floor(x m / 2^p) = floor(x / d), since m d - 2^p < d <= 2^(p - 31).
struct Divisor {
    uint32_t d, m, shift;
    Divisor(uint32_t by = 1) : d(by), m(0), shift(0) {
        int log = 0;
        while ((1ull << log) < by) log++;
        if (log) {  // (by 1: m 0)
            m = (uint32_t)(((1ull << (31 + log)) + by - 1) / by);
            shift = log - 1;
        }
    }
    __device__ __forceinline__ int of(int x) const { return m ? (int)(__umulhi((uint32_t)x, m) >> shift) : x; }
};

struct TurnArgs {
    Turn r;
    TurnJob job[3];
    int jobs, T, dh, heads, tokens;
    Divisor by_each, by_units, by_n;  // units a token, units a head, pairs
    const int *seq, *at, *table;
    long long ld_table;
    int B, width, pages, page;
    int* err;
};

template <int BYTES>
struct Piece;
template <>
struct Piece<16> {
    using type = uint4;
};
template <>
struct Piece<8> {
    using type = uint2;
};
template <>
struct Piece<4> {
    using type = uint32_t;
};
template <>
struct Piece<2> {
    using type = uint16_t;
};

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f(float& d, float v) { d = v; }
__device__ __forceinline__ void from_f(__nv_bfloat16& d, float v) { d = __float2bfloat16_rn(v); }

// The pieces of a unit turned: pair e is (x0[e], x1[e]), or with SIDE pairs lie
// side by side, through both pieces.
template <int P, bool SIDE>
__device__ __forceinline__ void turn_pairs(float* x0, float* x1, const float2* w, int pieces) {
#pragma unroll
    for (int e = 0; e < P; e++) {
        float& p0 = SIDE && P > 1 ? (2 * e < P ? x0 : x1)[2 * e % P] : x0[e];
        float& p1 = SIDE && P > 1 ? (2 * e < P ? x0 : x1)[(2 * e + 1) % P] : x1[e];
        const float2 c = w[e / 2 * 2 * pieces + e % 2];
        const float f0 = p0, f1 = p1;
        p0 = f0 * c.x - f1 * c.y;
        p1 = f1 * c.x + f0 * c.y;
    }
}

// P values a piece; a thread's unit is two pieces of one head. Cosine and sine
// of two neighbouring pairs lie together, those of all pieces' first two pairs
// before those of the next two: neighbouring threads read neighbouring 16
// bytes (pair by pair they met each bank four times, which bound the kernel:
// 34 us a pass over 16384 x 20 x 128 in place of 31). ONE: there is one job
// (known when compiled, with divisions by multiplication: 31 to 30 us).
template <typename T, int P, bool SIDE, bool ONE>
__global__ void __launch_bounds__(kTurnThreads) turn_kernel(const __grid_constant__ TurnArgs a) {
    using V = typename Piece<P * sizeof(T)>::type;
    extern __shared__ __align__(16) float2 cs[];  // [tokens][n] cosine and sine
    __shared__ int s_page[kTurnTokens], s_place[kTurnTokens];
    const long long t0 = (long long)blockIdx.x * a.tokens;
    const int tokens = (int)min((long long)a.tokens, a.T - t0);
    const int n = a.r.n;

    if (!ONE && (int)threadIdx.x < tokens) {
        const long long t = t0 + threadIdx.x;
        const int b = a.seq[t];
        int page = -1, place = 0;
        if (b >= 0) {
            const int at = a.at[t];
            const int p = at >= 0 ? at / a.page : -1;
            if (b < a.B && p >= 0 && p < a.width) page = a.table[(long long)b * a.ld_table + p];
            if (page < 0 || page >= a.pages) {  // no such place: the token is left out
                page = -1;
                atomicCAS(a.err, 0, kErrBadIndex);
            }
            place = at - p * a.page;
        }
        s_page[threadIdx.x] = page;
        s_place[threadIdx.x] = place;
    }
    const int units = a.dh / (2 * P), turned = n / P, each = a.heads * units;
    for (int e = threadIdx.x; e < tokens * n; e += kTurnThreads) {
        const int t = a.by_n.of(e), i = e - t * n;
        int axis = 0;
        while (axis + 1 < a.r.axes && i >= a.r.end[axis]) axis++;
        const double turns = (double)a.r.pos[axis * a.r.ld_pos + t0 + t] * ((double)a.r.freq[i] * 0.15915494309189533577);
        float s, c;
        sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
        const int piece = i / P, in = i - piece * P;
        cs[t * n + (P > 1 ? (in / 2 * turned + piece) * 2 + in % 2 : i)] = make_float2(c * a.r.scale, s * a.r.scale * a.r.sign);
    }
    __syncthreads();

    for (int u = threadIdx.x; u < tokens * each; u += kTurnThreads) {
        const int t = a.by_each.of(u), in = u - t * each;
        int head = a.by_units.of(in);
        const int piece = in - head * units;
        const TurnJob& j = a.job[ONE ? 0 : head >= a.job[2].first ? 2 : head >= a.job[1].first ? 1 : 0];
        head -= j.first;
        if (!ONE && s_page[t] < 0) continue;
        const bool turn = j.turn && piece < turned;
        int o0 = piece * 2 * P, o1 = o0 + P;
        if (turn && !SIDE) {
            o0 = piece * P;
            o1 = o0 + n;
        }
        const T* src = (const T*)j.src + (t0 + t) * j.src_row + head * j.src_head;
        T* dst = (T*)j.dst + head * j.dst_head +
                 (!ONE && j.paged ? s_page[t] * j.dst_page + s_place[t] * j.dst_row : (t0 + t) * j.dst_row);
        V v0 = *reinterpret_cast<const V*>(src + o0), v1 = *reinterpret_cast<const V*>(src + o1);
        if (turn) {
            T* x0 = reinterpret_cast<T*>(&v0);
            T* x1 = reinterpret_cast<T*>(&v1);
            float f0[P], f1[P];
#pragma unroll
            for (int e = 0; e < P; e++) f0[e] = to_f(x0[e]), f1[e] = to_f(x1[e]);
            turn_pairs<P, SIDE>(f0, f1, cs + t * n + piece * (P > 1 ? 2 : 1), turned);
            if constexpr (P > 1 && sizeof(T) == 2) {
#pragma unroll
                for (int e = 0; e < P; e += 2) {
                    reinterpret_cast<__nv_bfloat162*>(x0)[e / 2] = __floats2bfloat162_rn(f0[e], f0[e + 1]);
                    reinterpret_cast<__nv_bfloat162*>(x1)[e / 2] = __floats2bfloat162_rn(f1[e], f1[e + 1]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < P; e++) from_f(x0[e], f0[e]), from_f(x1[e], f1[e]);
            }
        }
        *reinterpret_cast<V*>(dst + o0) = v0;
        *reinterpret_cast<V*>(dst + o1) = v1;
    }
}

bool turn_ok(const Turn& t, int dh, int T) {
    if (t.n < 0 || 2 * t.n > dh || !(t.scale == t.scale)) return false;
    if (t.n == 0) return true;
    if (t.axes < 1 || t.axes > kMaxAxes || !t.freq || (T && !t.pos) || (t.axes > 1 && t.ld_pos < T)) return false;
    int last = 0;
    for (int i = 0; i < t.axes; i++) {
        if (t.end[i] < last) return false;
        last = t.end[i];
    }
    return last == t.n;
}

// Whether addresses and strides of a tensor are multiples of `bytes`.
bool even(const void* p, long long a, long long b, long long c, int size, int bytes) {
    return reinterpret_cast<uintptr_t>(p) % bytes == 0 && a * size % bytes == 0 && b * size % bytes == 0 &&
           c * size % bytes == 0;
}

// Tokens a block: several where a token has few units, so that the angles are
// shared out over all threads, but never so many that SMs stay without a block.
int launch(TurnArgs& a, int dtype, cudaStream_t s) {
    const int size = dtype == kBF16 ? 2 : 4;
    for (int j = a.jobs; j < 3; j++) a.job[j].first = 0x7fffffff;
    auto fits = [&](int P) {
        if (a.dh % (2 * P) || a.r.n % P) return false;
        for (int j = 0; j < a.jobs; j++) {
            const TurnJob& t = a.job[j];
            if (!even(t.src, t.src_row, t.src_head, 0, size, P * size) ||
                !even(t.dst, t.dst_row, t.dst_head, t.dst_page, size, P * size))
                return false;
        }
        return true;
    };
    auto go = [&](auto zero, auto width) {
        using T = decltype(zero);
        constexpr int P = decltype(width)::value;
        const long long each = (long long)a.heads * (a.dh / (2 * P));
        a.tokens = 1;
        while (a.tokens < kTurnTokens && a.tokens * each < 4 * kTurnThreads && a.T / (2 * a.tokens) >= 4 * num_sms())
            a.tokens *= 2;
        a.by_each = Divisor((uint32_t)each);
        a.by_units = Divisor(a.dh / (2 * P));
        a.by_n = Divisor(a.r.n ? a.r.n : 1);
        const auto f = a.seq ? (a.r.interleaved ? turn_kernel<T, P, true, false> : turn_kernel<T, P, false, false>)
                             : (a.r.interleaved ? turn_kernel<T, P, true, true> : turn_kernel<T, P, false, true>);
        f<<<(unsigned)(((long long)a.T + a.tokens - 1) / a.tokens), kTurnThreads, (size_t)a.tokens * a.r.n * sizeof(float2), s>>>(a);
        return cudaGetLastError() == cudaSuccess ? 0 : -5;
    };
    using std::integral_constant;
    if ((long long)a.heads * a.dh > kTurnMaxRow) return -2;
    if (dtype == kBF16) {
        if (fits(8)) return go(__nv_bfloat16(), integral_constant<int, 8>());
        if (fits(4)) return go(__nv_bfloat16(), integral_constant<int, 4>());
        return go(__nv_bfloat16(), integral_constant<int, 1>());
    }
    if (fits(4)) return go(0.f, integral_constant<int, 4>());
    return go(0.f, integral_constant<int, 1>());
}

TurnJob job(const Heads& src, const Heads& dst, int first, int turn) {
    return TurnJob{src.p, src.row, src.head, dst.p, dst.row, dst.head, 0, first, turn, 0};
}
TurnJob job(const Heads& src, const Pages& dst, int first, int turn) {
    return TurnJob{src.p, src.row, src.head, dst.p, dst.slot, dst.head, dst.page, first, turn, 1};
}

}  // namespace

int rope(const Turn& t, int dtype, const Heads& x, const Heads& y, int T, int H, int dh, cudaStream_t s) {
    if (T < 0 || H <= 0 || dh <= 0 || dh > kTurnMaxHead || (dh & 1) || (dtype != kF32 && dtype != kBF16)) return -1;
    if (t.n == 0 || !turn_ok(t, dh, T)) return -1;
    if (T == 0) return 0;
    if (!x.p || !y.p) return -1;
    TurnArgs a = {};
    a.r = t;
    a.job[0] = job(x, y, 0, 1);
    a.jobs = 1;
    a.T = T;
    a.dh = dh;
    a.heads = H;
    return launch(a, dtype, s);
}

int kv_append(const AppendDesc& d, cudaStream_t s) {
    if (d.T < 0 || d.Hkv <= 0 || d.dh <= 0 || d.dh > kTurnMaxHead || (d.dh & 1) || (d.dtype != kF32 && d.dtype != kBF16))
        return -1;
    if ((2LL * d.Hkv + (d.q.p ? d.Hq : 0)) * d.dh > kTurnMaxRow) return -2;
    if (d.B < 0 || d.width < 0 || d.ld_table < d.width || d.pages < 0 || d.page <= 0 || !turn_ok(d.turn, d.dh, d.T)) return -1;
    if ((d.q.p == nullptr) != (d.q_out.p == nullptr) || (d.q.p && d.Hq <= 0)) return -1;
    if (d.T == 0) return 0;
    if (!d.k.p || !d.v.p || !d.seq || !d.at || (d.B && d.width && !d.table) || (d.pages && (!d.kc.p || !d.vc.p)))
        return -1;
    if (!d.err) return -5;
    TurnArgs a = {};
    a.r = d.turn;
    int first = 0;
    a.job[a.jobs++] = job(d.k, d.kc, first, 1);
    first += d.Hkv;
    a.job[a.jobs++] = job(d.v, d.vc, first, 0);
    first += d.Hkv;
    if (d.q.p) {
        a.job[a.jobs++] = job(d.q, d.q_out, first, 1);
        first += d.Hq;
    }
    a.heads = first;
    a.T = d.T;
    a.dh = d.dh;
    a.seq = d.seq;
    a.at = d.at;
    a.table = d.table;
    a.ld_table = d.ld_table;
    a.B = d.B;
    a.width = d.width;
    a.pages = d.pages;
    a.page = d.page;
    a.err = d.err;
    return launch(a, d.dtype, s);
}

}  // namespace nsb
