// Group normalisation with an activation on fields over the sphere, forward and backward.
//
// x (B, C, nlat, nlon), planes or channels last, G groups of C / G channels, a_k = weight of latitude row k:
//     mu = sum a x / sum a,  v = sum a (x - mu)^2 / sum a      (over the C / G channels and all grid points of a group)
//     xh = (x - mu) r,  r = (v + eps)^(-1/2),  z = w_c xh + b_c,  y = act(z)
// With g = dy act'(z), h = w_c g and q = a / sum a:
//     db_c = sum g,  dw_c = sum g xh,  dx = r (h - q (sum h + xh sum h xh)).
// A few operations per element: float32 is bound by memory, 16-bit fields by it and by the arithmetic of their 8 values a vector.  x (and dy) are read
// from HBM twice, since a pass goes over the whole field before the next one begins.
//
// Two or three launches a direction: sums of chunks, their joining (in the second pass itself where that is little), the second pass.  The
// work is cut into units (a sample, channels last; a plane, otherwise), units into chunks of pixels, a CTA each.  A chunk is read as one flat stream of
// 16-byte vectors: with C' interleaved channels (C, or 1 for planes) and V values a vector, a thread that steps by a multiple of lcm(C', V)
// values meets the same channels in every vector ("slots"), whatever C' is, and keeps their sums and parameters in registers.  The second
// pass takes the last pieces of all chunks first, since what the first has read last may still be in L2: of the 266 MB of 721x1440x64 float32 the counters
// find 9 MB there, of the 133 MB of bf16 19 MB (backward, with twice as much read, nothing).
//
// All times below are device times on a B200 with a cold L2 (fields in HBM, copied at 6.56 TB/s).
//
// Sums for the variance are taken about a centre c per slot, (W, c, S1, S2) = (sum a, c, sum a (x - c), sum a (x - c)^2).  c begins as a value
// of the field (in a row that counts) and is moved to the mean so far after 1, 2, 4, 8, ... rounds; fields whose level is far above their spread
// (pressures), that have a value far out, or whose rows weigh very differently lose nothing.  Chunks are joined in float64 as (W, K, mean - K, M2).
//
// What is held in float32: the sums of a thread and of the threads of a chunk (up to 2,000 terms one after the other; float64 would take twice the registers,
// of which these loops are short), the slope and the activation, exponentials and reciprocals by the approximate instructions (2^-22).  Against 64 bits, 721x1440x64 and
// 256x512x32 float32, root mean square: y 8e-8, dx 1.1e-7, dweight and dbias 1.2e-7 to 4e-7 of their own size (float64 sums: 8e-8 all).

#include "common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <initializer_list>
#include <map>
#include <mutex>
#include <numeric>

namespace shtb200 {

namespace {

// ------------------------------------------------------------------------------------------------
// pairs of float32: sm_100a multiplies and adds two at a time
// ------------------------------------------------------------------------------------------------
struct F2 {
    unsigned long long v;
};
__device__ __forceinline__ F2 f2(float x, float y) {
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ F2 f2(float x) { return f2(x, x); }
__device__ __forceinline__ float2 split(F2 a) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
    return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
    F2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 sub2(F2 a, F2 b) {
    F2 r;
    asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float rcp_fast(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// ------------------------------------------------------------------------------------------------
// activations, two values at a time
// ------------------------------------------------------------------------------------------------
// Normal distribution function of -|z|:  Phi(-a) = e^(-a^2 / 2) R(a),  R(a) = t P(t) with t = 1 / (1 + 0.3 a): the polynomial P of
// degree 7 is the minimax fit of R(a) / t in relative error over 0 <= a <= 13.5 (1.3e-7; computed by reweighted least squares
// against the scaled complementary error function).  gelu(z) = max(z, 0) - a Phi(-a) then keeps its relative accuracy in the tail, up to the rounding of
// z^2: 2e-6 at z = -6.  Values that are rounded to 16 bits behind it take degree 4 and t = 1 / (1 + 0.375 a), 2.9e-5: an eighth of float16's smallest
// half step.
struct Tail {
    F2 e, r, na;  // e^(-a^2 / 2), R(a), -a
};
template <typename T> __device__ __forceinline__ Tail normal_tail(F2 z) {
    Tail k;
    k.na.v = z.v | 0x8000000080000000ull;
    const float2 d = split(fma2(k.na, f2(sizeof(T) == 2 ? -0.375f : -0.3f), f2(1.f)));
    const F2 t = f2(rcp_fast(d.x), rcp_fast(d.y));
    F2 p;
    if constexpr (sizeof(T) == 2) {
        p = fma2(t, f2(-0.090985179f), f2(0.20104314f));
        p = fma2(t, p, f2(0.082974225f));
        p = fma2(t, p, f2(0.15792f));
        p = fma2(t, p, f2(0.14904104f));
    } else {
        p = fma2(t, f2(0.035931703f), f2(-0.15827584f));
        p = fma2(t, p, f2(0.20820633f));
        p = fma2(t, p, f2(-0.05539357f));
        p = fma2(t, p, f2(0.12946904f));
        p = fma2(t, p, f2(0.099637546f));
        p = fma2(t, p, f2(0.12079835f));
        p = fma2(t, p, f2(0.11962639f));
    }
    k.r = mul2(t, p);
    const float2 x = split(mul2(mul2(z, f2(-0.72134752f)), z));
    k.e = f2(exp2_fast(x.x), exp2_fast(x.y));
    return k;
}
__device__ __forceinline__ F2 logistic(F2 z) {
    const float2 x = split(mul2(z, f2(-1.44269504f)));
    const float2 d = split(add2(f2(exp2_fast(x.x), exp2_fast(x.y)), f2(1.f)));
    return f2(rcp_fast(d.x), rcp_fast(d.y));
}

template <typename T, int ACT> __device__ __forceinline__ F2 act_value(F2 z) {
    if constexpr (ACT == SHTB200_ACT_RELU) {
        const float2 v = split(z);
        return f2(v.x <= 0.f ? 0.f : v.x, v.y <= 0.f ? 0.f : v.y);  // (a NaN stays one)
    } else if constexpr (ACT == SHTB200_ACT_SILU) {
        return mul2(z, logistic(z));
    } else if constexpr (ACT == SHTB200_ACT_GELU) {
        const Tail k = normal_tail<T>(z);
        const float2 v = split(z);
        return fma2(mul2(k.na, k.e), k.r, f2(fmaxf(v.x, 0.f), fmaxf(v.y, 0.f)));
    }
    return z;
}
// The slope takes kSlopeScale z, which costs nothing where z is made from a scale and a shift, and comes divided by it again (OVER) where a scale
// follows.  gelu'(z) = Phi(z) + z phi(z) = 1/2 + sign(z) (1/2 - e^(-a^2 / 2) (R(a) - a / sqrt(2 pi))), here with e^(-a^2 / 2) = 2^(-zs^2) and
// R fitted (as above) in absolute error weighted by e^(-a^2 / 2): degree 5 with t = 1 / (1 + 0.28 a), 2.2e-7 over all z in float32 arithmetic.  Absolute,
// since a slope is one term among those of size 1 in dx and in the sums; in the tail it is 7e-6 at z = -5, where the error is 0.7 % of it.
template <int ACT> constexpr float kSlopeScale = ACT == SHTB200_ACT_GELU ? 0.84932180f : ACT == SHTB200_ACT_SILU ? 1.44269504f : 1.f;
template <int ACT, bool OVER> __device__ __forceinline__ F2 act_slope(F2 zs) {
    constexpr float F = OVER ? 1.f / kSlopeScale<ACT> : 1.f;
    if constexpr (ACT == SHTB200_ACT_RELU) {
        const float2 v = split(zs);
        return f2(v.x <= 0.f ? 0.f : 1.f, v.y <= 0.f ? 0.f : 1.f);
    } else if constexpr (ACT == SHTB200_ACT_SILU) {
        constexpr float kLn2 = 0.69314718f * F;
        const float2 x = split(zs);
        const float2 d = split(add2(f2(exp2_fast(-x.x), exp2_fast(-x.y)), f2(1.f)));
        const F2 s = f2(rcp_fast(d.x), rcp_fast(d.y));
        return fma2(mul2(zs, s), fma2(s, f2(-kLn2), f2(kLn2)), OVER ? mul2(s, f2(F)) : s);
    } else if constexpr (ACT == SHTB200_ACT_GELU) {
        F2 na;
        na.v = zs.v | 0x8000000080000000ull;
        const float2 d = split(fma2(na, f2(-0.3296748f), f2(1.f)));
        const F2 t = f2(rcp_fast(d.x), rcp_fast(d.y));
        F2 r = fma2(t, f2(0.101911396f * F), f2(-0.37383756f * F));
        r = fma2(t, r, f2(0.21076515f * F));
        r = fma2(t, r, f2(-0.24760479f * F));
        r = fma2(t, r, f2(-0.07608968f * F));
        r = fma2(t, r, f2(-0.11514454f * F));
        r = fma2(na, f2(-0.46971864f * F), mul2(t, r));  // a / sqrt(2 pi) - R(a)
        const float2 x = split(mul2(zs, zs));
        F2 h = fma2(f2(exp2_fast(-x.x), exp2_fast(-x.y)), r, f2(0.5f * F));
        h.v ^= zs.v & 0x8000000080000000ull;
        return add2(h, f2(0.5f * F));
    }
    return f2(1.f);
}

// ------------------------------------------------------------------------------------------------
// vectors of 16 bytes
// ------------------------------------------------------------------------------------------------
template <typename T> constexpr int kV = 16 / (int)sizeof(T);  // values of a vector
template <typename T> constexpr int kP = kV<T> / 2;            // pairs of a vector

__device__ __forceinline__ void unpack(uint4 u, F2 (&p)[2], float) {
    p[0] = f2(__uint_as_float(u.x), __uint_as_float(u.y));
    p[1] = f2(__uint_as_float(u.z), __uint_as_float(u.w));
}
__device__ __forceinline__ void unpack(uint4 u, F2 (&p)[4], __nv_bfloat16) {
    const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = f2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
}
__device__ __forceinline__ void unpack(uint4 u, F2 (&p)[4], __half) {
    const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 v = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        p[i] = f2(v.x, v.y);
    }
}
__device__ __forceinline__ uint4 pack(const F2 (&p)[2], float) {
    const float2 a = split(p[0]), b = split(p[1]);
    return make_uint4(__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x), __float_as_uint(b.y));
}
__device__ __forceinline__ uint4 pack(const F2 (&p)[4], __nv_bfloat16) {
    uint4 u;
    unsigned *w = &u.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 v = split(p[i]);
        const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
        w[i] = *reinterpret_cast<const unsigned *>(&h);
    }
    return u;
}
__device__ __forceinline__ uint4 pack(const F2 (&p)[4], __half) {
    uint4 u;
    unsigned *w = &u.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 v = split(p[i]);
        const __half2 h = __floats2half2_rn(v.x, v.y);
        w[i] = *reinterpret_cast<const unsigned *>(&h);
    }
    return u;
}
__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void store_f(float *p, float v) { *p = v; }
__device__ __forceinline__ void store_f(__half *p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void store_f(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }

// The scale and shift parameters are a handful of values: their type is a run-time switch.
__device__ __forceinline__ float load_param(const void *p, int dtype, int i, float none) {
    if (!p) return none;
    if (dtype == SHTB200_F32) return reinterpret_cast<const float *>(p)[i];
    if (dtype == SHTB200_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(p)[i]);
    return __half2float(reinterpret_cast<const __half *>(p)[i]);
}
__device__ __forceinline__ void store_param(void *p, int dtype, int i, float v) {
    if (!p) return;
    if (dtype == SHTB200_F32) reinterpret_cast<float *>(p)[i] = v;
    else if (dtype == SHTB200_BF16) reinterpret_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
    else reinterpret_cast<__half *>(p)[i] = __float2half_rn(v);
}

// ------------------------------------------------------------------------------------------------
// geometry
// ------------------------------------------------------------------------------------------------
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCols = 128;  // columns of vectors a CTA covers at a time

struct GnArgs {
    const void *x, *dy;
    void *out;
    const float *lat;  // nullptr: 1 everywhere
    const void *weight, *bias;
    void *dweight, *dbias;
    float4 *stats;     // (B, G): mean, its low part, r, 1 / sum a
    float4 *part;      // forward: (unit, chunk, group of the unit): (W, K, mean - K, M2)
    float2 *bpart;     // backward: (unit, chunk, channel of the unit): (sum g, sum g xh)
    double2 *csum;     // backward, not direct: (B, C): the same over all chunks
    long long hw;
    int B, C, G, cg, nlat, nlon, cl, pdtype;
    float eps;
    int cu, gu, cgu;   // channels, groups of a unit, channels of a group inside a unit: (C, G, cg) channels last, (1, 1, 1) for planes
    int chunks, chunk_px, tasks;  // of a unit for the sums; chunks of all units
    int pieces, piece_px;         // of a chunk, for the second pass
    int cols, dup;                // lcm(cu, V) / V: vectors after which the channels repeat; how often each occurs in them
    int win_cols, windows, reps;  // columns a CTA covers at a time, how many windows that takes, vectors of a column it takes side by side
    int step_px, step_rows, step_cols;  // from a thread's vector to its next, in pixels, and as rows and columns of the grid
    int lanes;                    // that join the slots of a group
    int direct;        // the partial results of a group are joined by every CTA that needs them; else by a launch in between
};

// A chunk of a unit: n values from `base` on; `head` of them lie before the first aligned vector, then `vecs` vectors, then the tail.
struct Chunk {
    int unit, chunk, b, c;  // (c: the channel of a plane)
    long long base;  // first value
    int px0;         // its pixel
    int n, head, vecs;
};
// Piece `piece` of chunk `task`, pieces of `piece_px` pixels (the whole chunk: piece 0 of chunk_px); n <= 0 where a chunk has fewer.
template <typename T> __device__ __forceinline__ Chunk make_chunk(const GnArgs &a, int task, int piece, int piece_px) {
    Chunk k;
    k.unit = (int)((unsigned)task / (unsigned)a.chunks);
    k.chunk = task - k.unit * a.chunks;
    k.b = a.cl ? k.unit : (int)((unsigned)k.unit / (unsigned)a.C);
    k.c = a.cl ? 0 : k.unit - k.b * a.C;
    const int in = piece * piece_px;
    k.px0 = k.chunk * a.chunk_px + in;
    const int px = (int)min((long long)min(piece_px, a.chunk_px - in), a.hw - k.px0);
    k.base = ((long long)k.unit * a.hw + k.px0) * a.cu;
    k.n = px * a.cu;
    const unsigned mis = (unsigned)((uintptr_t)(reinterpret_cast<const T *>(a.x) + k.base) & 15u);
    k.head = min(k.n, (int)(((16u - mis) & 15u) / (unsigned)sizeof(T)));
    k.vecs = (k.n - k.head) / kV<T>;
    return k;
}

// The second pass takes the last pieces of all chunks first, then the ones before: the sums have read their chunks side by side, so that is what L2
// holds.
template <typename T> __device__ __forceinline__ Chunk second_pass_chunk(const GnArgs &a, int block) {
    const int back = (int)((unsigned)block / (unsigned)a.tasks);
    return make_chunk<T>(a, block - back * a.tasks, a.pieces - 1 - back, a.piece_px);
}

// A thread's share of a window of a chunk: vectors first, first + step, ... (count of them); the channel (of the unit) of slot 0.
struct Share {
    int first, step, count, ch0, rep, col;
};
template <typename T, bool PLANES> __device__ __forceinline__ Share make_share(const GnArgs &a, const Chunk &k, int window) {
    Share s;
    if constexpr (PLANES) {  // a contiguous stretch for every warp, so that a thread stays in a row for a while
        const int per = (k.vecs + kThreads - 1) / kThreads * 32, lo = (int)(threadIdx.x >> 5) * per, hi = min(lo + per, k.vecs);
        s.rep = threadIdx.x;
        s.col = s.ch0 = 0;
        s.first = lo + (int)(threadIdx.x & 31);
        s.step = 32;
        s.count = s.first < hi ? (hi - s.first + 31) / 32 : 0;
    } else {
        s.rep = a.win_cols == 1 ? (int)threadIdx.x : (int)(threadIdx.x / (unsigned)a.win_cols);
        s.col = (int)threadIdx.x - s.rep * a.win_cols;
        const int c = window * a.win_cols + s.col;
        s.first = c + s.rep * a.cols;
        s.step = a.reps * a.cols;
        s.count = (s.rep < a.reps && c < a.cols && s.first < k.vecs) ? (int)((unsigned)(k.vecs - s.first + s.step - 1) / (unsigned)s.step) : 0;
        s.ch0 = (int)((unsigned)(c * kV<T> + k.head) % (unsigned)a.cu);
    }
    return s;
}

// Latitude weight of the vectors of a share.  A vector lies in one row, but for those across a row's end.
struct Rows {
    int row, col, over;  // of slot 0; pixels from slot 0 to the last slot
};
template <typename T> __device__ __forceinline__ Rows make_rows(const GnArgs &a, const Chunk &k, const Share &s, int n) {
    Rows r;
    const unsigned e = (unsigned)k.head + ((unsigned)s.first + (unsigned)n * (unsigned)s.step) * kV<T>;
    const unsigned px = (unsigned)k.px0 + (a.cu == 1 ? e : e / (unsigned)a.cu);
    r.row = (int)(px / (unsigned)a.nlon);
    r.col = (int)px - r.row * a.nlon;
    r.over = a.cu == 1 ? kV<T> - 1 : (int)((unsigned)(s.ch0 + kV<T> - 1) / (unsigned)a.cu);
    return r;
}
__device__ __forceinline__ void advance(const GnArgs &a, Rows &r) {
    r.row += a.step_rows;
    r.col += a.step_cols;
    if (r.col >= a.nlon) {
        r.col -= a.nlon;
        ++r.row;
    }
}
// Weights of the U vectors of a whole round, r and w moved on to the next one.  False, and nothing moved, where the vectors have to be taken one at
// a time.
// Planes look every vector's weight up, unless one lies across a row's end: a warp's round spans a third of a row of 1440 16-bit values, so a
// branch for rounds within a row is taken both ways too often (721x1440x64 bf16, forward / backward: 86 / 135 us, with the branch 92 / 151; 721x1440x73
// float32 forward 161, with it 159).
// Channels last a round spans a few points: those within a row share a weight, the others go one at a time (361x720x256 bf16: 92 / 138 us,
// looked up 94 / 142).
template <int U, bool PLANES> __device__ __forceinline__ bool round_weights(const GnArgs &a, int have, Rows &r, float &w, float (&wu)[U]) {
    if (have < U) return false;
    if (!a.lat || (!PLANES && r.col + U * a.step_px + r.over < a.nlon)) {  // all in one row, the next one too
#pragma unroll
        for (int u = 0; u < U; ++u) wu[u] = w;
        r.col += U * a.step_px;
        return true;
    }
    if constexpr (PLANES) {
        Rows q = r;
        float v = w;
        bool across = false;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            wu[u] = v;
            across |= q.col + q.over >= a.nlon;
            advance(a, q);
            v = __ldg(a.lat + min(q.row, a.nlat - 1));
        }
        if (across) return false;
        r = q;
        w = v;
        return true;
    }
    return false;
}
// weights of the slots of a vector across a row's end
template <typename T> __device__ __forceinline__ void mixed_weights(const float *lat, int nlon, int cu, int ch, int row, int col, float (&w)[kV<T>]) {
#pragma unroll
    for (int i = 0; i < kV<T>; ++i) {
        while (col >= nlon) {
            col -= nlon;
            ++row;
        }
        w[i] = __ldg(lat + row);
        if (++ch == cu) {
            ch = 0;
            ++col;
        }
    }
}
// value i of the head and tail of a chunk (fewer than 2 V values): its index in the chunk, -1 beyond
template <typename T> __device__ __forceinline__ int ragged(const Chunk &k, int i) {
    const int tail = k.head + k.vecs * kV<T>;
    if (i < k.head) return i;
    i += tail - k.head;
    return i < k.n ? i : -1;
}
__device__ __forceinline__ float weight_at(const GnArgs &a, const Chunk &k, int e) { return a.lat ? __ldg(a.lat + (k.px0 + e / a.cu) / a.nlon) : 1.f; }

// Weight, bias and group (of the unit) of the V slots from channel ch on.  The loads go out together.
template <int V, bool PLANES> __device__ __forceinline__ void slot_params(const GnArgs &a, const Chunk &k, int ch, float (&w)[V], float (&b)[V], int (&g)[V]) {
    if constexpr (PLANES) {
        const float w0 = load_param(a.weight, a.pdtype, k.c, 1.f), b0 = load_param(a.bias, a.pdtype, k.c, 0.f);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            w[i] = w0;
            b[i] = b0;
            g[i] = 0;
        }
        return;
    }
    int c[V], group = (int)((unsigned)ch / (unsigned)a.cgu), in = ch - group * a.cgu;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        c[i] = ch;
        g[i] = group;
        w[i] = 1.f;
        b[i] = 0.f;
        ++ch;
        if (++in == a.cgu) {
            in = 0;
            ++group;
        }
        if (ch == a.cu) ch = group = in = 0;
    }
    if (a.pdtype == SHTB200_F32) {
        if (a.weight)
#pragma unroll
            for (int i = 0; i < V; ++i) w[i] = __ldg(reinterpret_cast<const float *>(a.weight) + c[i]);
        if (a.bias)
#pragma unroll
            for (int i = 0; i < V; ++i) b[i] = __ldg(reinterpret_cast<const float *>(a.bias) + c[i]);
    } else {
        unsigned short hw[V], hb[V];
        if (a.weight)
#pragma unroll
            for (int i = 0; i < V; ++i) hw[i] = __ldg(reinterpret_cast<const unsigned short *>(a.weight) + c[i]);
        if (a.bias)
#pragma unroll
            for (int i = 0; i < V; ++i) hb[i] = __ldg(reinterpret_cast<const unsigned short *>(a.bias) + c[i]);
        const bool bf = a.pdtype == SHTB200_BF16;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (a.weight) w[i] = bf ? __uint_as_float((unsigned)hw[i] << 16) : __half2float(__ushort_as_half(hw[i]));
            if (a.bias) b[i] = bf ? __uint_as_float((unsigned)hb[i] << 16) : __half2float(__ushort_as_half(hb[i]));
        }
    }
}

// ------------------------------------------------------------------------------------------------
// joining of moments
// ------------------------------------------------------------------------------------------------
struct Moments {  // (sum of weights, K, mean - K, M2); K is the mean rounded: a K far out (the value at a pole) would round mean - K
    float W, K, m, M2;
};
__device__ __forceinline__ void normalise(Moments &a) {
    const float K = a.K + a.m;
    a.m = (a.K - K) + a.m;
    a.K = K;
}
__device__ __forceinline__ Moments moments(float W, float c, float S1, float S2) {
    const float m = W > 0.f ? __fdividef(S1, W) : 0.f;
    Moments r{W, c, m, fmaxf(fmaf(-S1, m, S2), S2 * 0.f)};  // (rounding may leave less than nothing; a NaN or infinity has to stay)
    normalise(r);
    return r;
}
__device__ __forceinline__ void join(Moments &a, const Moments &b) {
    if (b.W == 0.f) return;
    if (a.W == 0.f) {
        a = b;
        return;
    }
    // (from the mean of the part that weighs more: the other's may be far from it, and the rounding of f would move the mean by as much of that)
    const bool swap = b.W > a.W;
    const Moments heavy = swap ? b : a, light = swap ? a : b;
    const float W = a.W + b.W, f = __fdividef(light.W, W), d = (light.K - heavy.K) + (light.m - heavy.m);
    a = {W, heavy.K, fmaf(d, f, heavy.m), heavy.M2 + fmaf(d * d, heavy.W * f, light.M2)};
    normalise(a);
}

__device__ __forceinline__ double warp_sum(double v) {
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ double2 warp_sum(double2 v) { return make_double2(warp_sum(v.x), warp_sum(v.y)); }

// Partial results joined in float64, about the mean of the first that has any weight (fields whose level is far above their spread lose nothing, and no
// division is needed on the way; a part of rows that do not count has no mean): thread `i` of `of` takes every of-th, four loads at a time.
struct Sums64 {
    double c, W, s, q;
    __device__ __forceinline__ void add(const float4 &v) {
        if (v.x != 0.f) {
            const double d = ((double)v.y - c) + v.z, wd = v.x * d;
            W += v.x;
            s += wd;
            q += v.w + wd * d;
        }
    }
    __device__ __forceinline__ void gather(const float4 *p, int n, long long stride, int i, int of) {
        float4 v[4], v0 = __ldcg(p);
        auto fetch = [&] {
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = i + u * of < n ? __ldcg(p + (i + u * of) * stride) : make_float4(0.f, 0.f, 0.f, 0.f);
        };
        fetch();
        for (int from = 0; v0.x == 0.f && from < n; from += 32) {  // (the same part for every warp and CTA)
            const int at = from + (int)(threadIdx.x & 31);
            const float here = at < n ? __ldcg(p + at * stride).x : 0.f;
            if (const unsigned some = __ballot_sync(0xffffffffu, here != 0.f)) v0 = __ldcg(p + (from + __ffs(some) - 1) * stride);
        }
        c = (double)v0.y + v0.z;
        W = s = q = 0.;
        while (i < n) {
#pragma unroll
            for (int u = 0; u < 4; ++u) add(v[u]);
            i += 4 * of;
            fetch();
        }
        W = warp_sum(W);
        s = warp_sum(s);
        q = warp_sum(q);
    }
    // (float64 to the end: c is the mean of the first part, which may be ten thousand spreads from the mean of all.  1 / W in float32 left the variance
    // of a 721x1440 field whose first row is that far out 2.4e-3 off.)
    __device__ __forceinline__ float4 stats(const GnArgs &a) const {
        const double inv = 1. / W, m = s * inv, mean = c + m;
        const float hi = (float)mean, var = (float)((q - s * m) * inv);
        return make_float4(hi, (float)(mean - hi), 1.f / sqrtf(fmaxf(var, var * 0.f) + a.eps), (float)inv);
    }
};

// Sums over the threads of a column, M pairs of each: pair i of column c at tot[i * kMaxCols + c].
template <int M> __device__ __forceinline__ void column_sums(const GnArgs &a, const Share &s, F2 (&v)[M], F2 *red, F2 *tot) {
    int rep = s.rep, c = s.col, n = a.reps;
    if (a.windows == 1 && a.cols <= 32 && (a.cols & (a.cols - 1)) == 0) {  // whole columns in a warp: lanes first
        for (int o = 16; o >= a.cols; o >>= 1)
#pragma unroll
            for (int i = 0; i < M; ++i) {
                F2 u;
                u.v = __shfl_xor_sync(0xffffffffu, v[i].v, o);
                v[i] = add2(v[i], u);
            }
        c = threadIdx.x & 31;
        rep = c < a.cols ? (int)(threadIdx.x >> 5) : kThreads;
        n = kWarps;
    }
    if (rep < n)
#pragma unroll
        for (int i = 0; i < M; ++i) red[i * kThreads + rep * a.win_cols + c] = v[i];
    __syncthreads();
    for (int o = threadIdx.x; o < M * a.win_cols; o += kThreads) {
        const int i = (int)((unsigned)o / (unsigned)a.win_cols), col = o - i * a.win_cols;
        const F2 *p = red + i * kThreads + col;
        F2 t = p[0];
        for (int r = 1; r < n; ++r) t = add2(t, p[r * a.win_cols]);
        tot[i * kMaxCols + col] = t;
    }
    __syncthreads();
}
__device__ __forceinline__ float half_of(const F2 *tot, int pair, int col, int h) { return reinterpret_cast<const float *>(tot + pair * kMaxCols + col)[h]; }

// A thread's vectors on their way: rounds of U vectors (of each tensor), R rounds ahead, through a ring of its own in shared memory.  Nobody
// else reads it, so no barrier is needed; and what is in flight does not cost registers.
template <int TENSORS, int U, int R> struct Feed {
    static constexpr size_t bytes = (size_t)TENSORS * U * R * kThreads * 16;
    uint32_t ring;                 // the thread's vector 0
    const char *at[TENSORS];
    long long step;
    int left, slot;                // vectors to be sent for; the round at hand
    __device__ __forceinline__ void send(int to) {
        if (left >= U) {
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int t = 0; t < TENSORS; ++t) {
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(ring + 16u * kThreads * (uint32_t)((to * U + u) * TENSORS + t)), "l"(at[t]) : "memory");
                    at[t] += step;
                }
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (u < left)
#pragma unroll
                    for (int t = 0; t < TENSORS; ++t) {
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(ring + 16u * kThreads * (uint32_t)((to * U + u) * TENSORS + t)), "l"(at[t]) : "memory");
                        at[t] += step;
                    }
        }
        left -= U;
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    __device__ __forceinline__ void start(void *shared, const void *x, const void *y, int count, int step_vectors) {
        ring = (uint32_t)__cvta_generic_to_shared(shared) + 16u * threadIdx.x;
        at[0] = reinterpret_cast<const char *>(x);
        if constexpr (TENSORS == 2) at[1] = reinterpret_cast<const char *>(y);
        step = 16LL * step_vectors;
        left = count;
        slot = 0;
#pragma unroll
        for (int i = 0; i < R; ++i) send(i);
    }
    __device__ __forceinline__ void wait() { asm volatile("cp.async.wait_group %0;" ::"n"(R - 1) : "memory"); }
    __device__ __forceinline__ uint4 get(int u, int t) const {
        uint4 v;
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                     : "r"(ring + 16u * kThreads * (uint32_t)((slot * U + u) * TENSORS + t))
                     : "memory");
        return v;
    }
    __device__ __forceinline__ void next() {  // after the last get() of a round
        send(slot);
        if (++slot == R) slot = 0;
    }
};

// What follows a launch waits here for it; what precedes it in the kernel overlaps its end.
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_begin() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// ------------------------------------------------------------------------------------------------
// forward
// ------------------------------------------------------------------------------------------------
// q: (S1, S2) of the slots' pairs
template <typename T> __device__ __forceinline__ void accumulate(const F2 (&v)[kP<T>], const F2 (&c)[kP<T>], F2 (&q)[2 * kP<T>], const F2 (&w)[kP<T>]) {
#pragma unroll
    for (int p = 0; p < kP<T>; ++p) {
        const F2 d = sub2(v[p], c[p]), wd = mul2(d, w[p]);
        q[p] = add2(q[p], wd);
        q[kP<T> + p] = fma2(wd, d, q[kP<T> + p]);
    }
}
__device__ __forceinline__ F2 reciprocal(F2 a) {
    const float2 v = split(a);
    return f2(v.x > 0.f ? __fdividef(1.f, v.x) : 0.f, v.y > 0.f ? __fdividef(1.f, v.y) : 0.f);  // (0 while all rows so far have weight 0)
}
// sums about c + delta from those about c
__device__ __forceinline__ void recentre(F2 W, F2 delta, F2 &S1, F2 &S2) {
    const F2 t = mul2(W, delta);
    S2 = sub2(S2, mul2(delta, sub2(add2(S1, S1), t)));
    S1 = sub2(S1, t);
}

// Slots that a vector (of weights w) outweighs so far take their value in it as the centre.  True while some have met no row that counts.
template <typename T>
__device__ __forceinline__ bool centre_on(uint4 raw, const F2 (&w)[kP<T>], float W, const F2 (*extra)[kThreads], F2 (&c)[kP<T>], F2 (&q)[2 * kP<T>]) {
    F2 v[kP<T>];
    unpack(raw, v, T());
    bool open = false;
#pragma unroll
    for (int p = 0; p < kP<T>; ++p) {
        const F2 Wp = add2(extra[p][threadIdx.x], f2(W));
        const float2 so_far = split(Wp), now = split(w[p]), x = split(v[p]), d = split(sub2(v[p], c[p])), old = split(c[p]);
        const bool b0 = now.x > so_far.x, b1 = now.y > so_far.y;
        recentre(Wp, f2(b0 ? d.x : 0.f, b1 ? d.y : 0.f), q[p], q[kP<T> + p]);
        c[p] = f2(b0 ? x.x : old.x, b1 ? x.y : old.y);
        open |= (so_far.x == 0.f && now.x == 0.f) || (so_far.y == 0.f && now.y == 0.f);
    }
    return open;
}

constexpr int kUnroll = 2;
template <typename T> constexpr int kStatsCtas = sizeof(T) == 4 ? 4 : 3;  // on an SM: 8 slots a thread spill at 4 (73 channels bf16 122 us, at 3 103); 4 slots do not
using StatsFeed = Feed<1, kUnroll, 3>;  // (721x1440x73 bf16 channels last, forward: 103 us with 3 rounds, 104 with 2, 115 with 5)

// Sums of a chunk.  Bound by reading x in float32.  With 16-bit values a vector has twice the arithmetic: at 24 warps an SM 61 % of the issue slots are
// taken, and warps wait for a result of their own, or at the barriers at the end of a chunk, where few threads join its sums; of 73 channels three rows of 73
// threads have vectors, so an eighth warp waits there from the start.  (Without the weights' multiplications it is no faster.)
// 721x1440x73 float32 planes, with the pass below: 161 us, 5.7 TB/s over two reads and a write.

template <typename T, bool PLANES> __global__ void __launch_bounds__(kThreads, kStatsCtas<T>) gn_stats_kernel(const __grid_constant__ GnArgs a) {
    constexpr int V = kV<T>, P = kP<T>, U = kUnroll;
    __shared__ __align__(16) F2 red[(PLANES ? 1 : 2) * P * kThreads];
    __shared__ __align__(16) F2 tot[PLANES ? kWarps * 2 : 4 * P * kMaxCols];  // of the columns: W, W (mean - centre), S1, S2
    __shared__ __align__(16) F2 centre[PLANES ? 1 : P * kMaxCols];
    // weights of a slot in the vectors that lie across rows, beside those that all slots share: rare, and registers are short
    F2(*extra)[kThreads] = reinterpret_cast<F2(*)[kThreads]>(red);
    extern __shared__ __align__(16) unsigned char gn_smem[];
    Moments *acc = reinterpret_cast<Moments *>(gn_smem + StatsFeed::bytes);
    const Chunk k = make_chunk<T>(a, blockIdx.x, 0, a.chunk_px);
    const T *x = reinterpret_cast<const T *>(a.x) + k.base;
    const uint4 *xv = reinterpret_cast<const uint4 *>(x + k.head);
    float4 *out = a.part + ((long long)k.unit * a.chunks + k.chunk) * a.gu;
    if (!PLANES)
        for (int g = threadIdx.x; g < a.gu; g += kThreads) acc[g] = {0.f, 0.f, 0.f, 0.f};
    wait_for_previous();
    let_next_begin();
    for (int win = 0; win < (PLANES ? 1 : a.windows); ++win) {
        const Share s = make_share<T, PLANES>(a, k, win);
        F2 c[P], q[2 * P];
        float W = 0.f;
#pragma unroll
        for (int p = 0; p < P; ++p) {
            c[p] = q[p] = q[P + p] = f2(0.f);
            extra[p][threadIdx.x] = f2(0.f);
        }
        StatsFeed feed;
        feed.start(gn_smem, xv + s.first, nullptr, s.count, s.step);
        if (s.count) {
            bool open = true;  // some slots have met no row that counts
            Rows r{0, 0, 0};
            float w = 1.f;
            if (a.lat) {
                r = make_rows<T>(a, k, s, 0);
                w = __ldg(a.lat + r.row);
            }
            for (int j = 0; j < s.count; j += U) {
                const int have = min(U, s.count - j);
                uint4 raw[U];
                feed.wait();
#pragma unroll
                for (int u = 0; u < U; ++u) raw[u] = feed.get(u, 0);
                feed.next();
                float wu[U];
                // The first centre: of the first round that counts, the vector that counts most (a value at the pole, far out, is none for rows of a
                // hundred times its weight, and one in a row that does not count is none at all).
                if (round_weights<U, PLANES>(a, have, r, w, wu)) {
                    if (open || wu[U - 1] > W) {
                        const bool last = wu[U - 1] >= wu[0];
                        const float most = last ? wu[U - 1] : wu[0];
                        F2 wp[P];
#pragma unroll
                        for (int p = 0; p < P; ++p) wp[p] = f2(most);
                        open = centre_on<T>(last ? raw[U - 1] : raw[0], wp, W, extra, c, q);
                    }
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        F2 v[P], wp[P];
                        unpack(raw[u], v, T());
#pragma unroll
                        for (int p = 0; p < P; ++p) wp[p] = f2(wu[u]);
                        accumulate<T>(v, c, q, wp);
                        W += wu[u];
                    }
                } else {
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (u < have) {
                            F2 v[P], wp[P];
#pragma unroll
                            for (int p = 0; p < P; ++p) wp[p] = f2(w);
                            const bool mixed = a.lat && r.col + r.over >= a.nlon;
                            if (mixed) {
                                float ws[V];
                                mixed_weights<T>(a.lat, a.nlon, a.cu, s.ch0, r.row, r.col, ws);
#pragma unroll
                                for (int p = 0; p < P; ++p) wp[p] = f2(ws[2 * p], ws[2 * p + 1]);
                            }
                            if (open || mixed || w > W) open = centre_on<T>(raw[u], wp, W, extra, c, q);
                            if (mixed)
#pragma unroll
                                for (int p = 0; p < P; ++p) extra[p][threadIdx.x] = add2(extra[p][threadIdx.x], wp[p]);
                            else
                                W += w;
                            unpack(raw[u], v, T());
                            accumulate<T>(v, c, q, wp);
                            if (a.lat) {
                                advance(a, r);
                                w = __ldg(a.lat + min(r.row, a.nlat - 1));
                            }
                        }
                }
                const int round = j / U;
                if ((round & (round + 1)) == 0) {
#pragma unroll
                    for (int p = 0; p < P; ++p) {
                        const F2 Wp = add2(extra[p][threadIdx.x], f2(W)), to = fma2(q[p], reciprocal(Wp), c[p]), delta = sub2(to, c[p]);
                        recentre(Wp, delta, q[p], q[P + p]);
                        c[p] = to;
                    }
                }
            }
        }
        // All threads of a column about their common mean, then added (planes: all slots of all threads).  The mean of one thread would not do as the
        // centre of all: it may hold little but a value at the pole, far out, whose weight is a ten thousandth of the others'.
        // (It is taken relative to the first thread's, so that the mean of a constant is that constant.)
        F2 z[P];  // W
#pragma unroll
        for (int p = 0; p < P; ++p) z[p] = add2(extra[p][threadIdx.x], f2(W));
        if constexpr (PLANES) {
            F2 *first = tot, *second = tot + kWarps;  // (W, mean) and (S1, S2) of every warp
            const int warp = threadIdx.x >> 5;
            auto slots = [](const F2 *v) {
                F2 t = v[0];
#pragma unroll
                for (int p = 1; p < P; ++p) t = add2(t, v[p]);
                const float2 h = split(t);
                return h.x + h.y;
            };
            auto lanes = [](float v) {
                for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
                return v;
            };
            F2 t[P];
            const float w = lanes(slots(z)), inv = w > 0.f ? __fdividef(1.f, w) : 0.f;
            const float lane0 = __shfl_sync(0xffffffffu, split(z[0]).x > 0.f ? split(c[0]).x : 0.f, 0);
#pragma unroll
            for (int p = 0; p < P; ++p) t[p] = fma2(mul2(z[p], f2(inv)), sub2(c[p], f2(lane0)), mul2(q[p], f2(inv)));
            const float mean = lane0 + lanes(slots(t));
            if ((threadIdx.x & 31) == 0) first[warp] = f2(w, mean);
            __syncthreads();
            float all = 0.f, off = 0.f;
            for (int n = 0; n < kWarps; ++n) all += split(first[n]).x;
            const float part = all > 0.f ? __fdividef(1.f, all) : 0.f, warp0 = split(first[0]).x > 0.f ? split(first[0]).y : 0.f;
            for (int n = 0; n < kWarps; ++n) off = fmaf(split(first[n]).x * part, split(first[n]).y - warp0, off);
            const float c0 = warp0 + off;
            if (s.count)
#pragma unroll
                for (int p = 0; p < P; ++p) recentre(z[p], sub2(f2(c0), c[p]), q[p], q[P + p]);
            const float S1 = lanes(slots(q)), S2 = lanes(slots(q + P));
            if ((threadIdx.x & 31) == 0) second[warp] = f2(S1, S2);
            __syncthreads();
            if (threadIdx.x == 0) {
                F2 v = second[0];
                for (int n = 1; n < kWarps; ++n) v = add2(v, second[n]);
                Moments m = moments(all, c0, split(v).x, split(v).y);
                for (int i = 0; i < 2 * V; ++i) {  // the values outside the vectors
                    const int e = ragged<T>(k, i);
                    if (e < 0) break;
                    join(m, Moments{weight_at(a, k, e), to_f(x[e]), 0.f, 0.f});
                }
                out[0] = make_float4(m.W, m.K, m.m, m.M2);
            }
        } else {
            F2 t[2 * P];
#pragma unroll
            for (int p = 0; p < P; ++p) {
                const float2 counted = split(z[p]), v = split(c[p]);
                if (s.rep == 0) centre[p * kMaxCols + s.col] = f2(counted.x > 0.f ? v.x : 0.f, counted.y > 0.f ? v.y : 0.f);
            }
            __syncthreads();  // (the columns are added where `extra` was, too)
#pragma unroll
            for (int p = 0; p < P; ++p) {
                t[p] = z[p];
                t[P + p] = fma2(z[p], sub2(c[p], centre[p * kMaxCols + s.col]), q[p]);
            }
            column_sums(a, s, t, red, tot);
            if (s.count)
#pragma unroll
                for (int p = 0; p < P; ++p) {
                    const F2 c0 = fma2(tot[(P + p) * kMaxCols + s.col], reciprocal(tot[p * kMaxCols + s.col]), centre[p * kMaxCols + s.col]);
                    recentre(z[p], sub2(c0, c[p]), q[p], q[P + p]);
                }
            column_sums(a, s, q, red, tot + 2 * P * kMaxCols);
            // groups: a few lanes each go through its channels' slots in this window
            const int period = a.cols * V, slots = a.cgu * a.dup, shift = k.head % a.cu, L = a.lanes;
            const int sub = threadIdx.x & (L - 1), lo = win * a.win_cols * V, hi = min(lo + a.win_cols * V, period);
            for (int g0 = 0; g0 < a.gu; g0 += kThreads / L) {
                const int g = g0 + (int)threadIdx.x / L;
                Moments m{0.f, 0.f, 0.f, 0.f};
                if (g < a.gu)
                    for (int i = sub; i < slots; i += L) {
                        const int again = (int)((unsigned)i / (unsigned)a.cgu);
                        int e = g * a.cgu + (i - again * a.cgu) - shift;  // value of the period that has this channel
                        if (e < 0) e += a.cu;
                        e += again * a.cu;
                        if (e >= lo && e < hi) {
                            const int col = (e - lo) / V, i2 = (e - lo) % V;
                            const float Wc = half_of(tot, i2 / 2, col, i2 & 1), inv = Wc > 0.f ? __fdividef(1.f, Wc) : 0.f;
                            const float c0 = fmaf(half_of(tot, P + i2 / 2, col, i2 & 1), inv, half_of(centre, i2 / 2, col, i2 & 1));  // (as above, to the bit)
                            join(m, moments(Wc, c0, half_of(tot, 2 * P + i2 / 2, col, i2 & 1), half_of(tot, 3 * P + i2 / 2, col, i2 & 1)));
                        }
                    }
                for (int o = L / 2; o; o >>= 1) {
                    Moments b;
                    b.W = __shfl_down_sync(0xffffffffu, m.W, o, L);
                    b.K = __shfl_down_sync(0xffffffffu, m.K, o, L);
                    b.m = __shfl_down_sync(0xffffffffu, m.m, o, L);
                    b.M2 = __shfl_down_sync(0xffffffffu, m.M2, o, L);
                    join(m, b);
                }
                if (g < a.gu && sub == 0) {
                    Moments t = acc[g];
                    join(t, m);
                    if (win == 0)  // the values outside the vectors, one at a time
                        for (int i = 0; i < 2 * V; ++i) {
                            const int e = ragged<T>(k, i);
                            if (e < 0) break;
                            if ((e % a.cu) / a.cgu == g) join(t, Moments{weight_at(a, k, e), to_f(x[e]), 0.f, 0.f});
                        }
                    acc[g] = t;
                    if (win == a.windows - 1) out[g] = make_float4(t.W, t.K, t.m, t.M2);
                }
            }
            if (a.windows > 1) __syncthreads();
        }
    }
}

// The partial results of a group: n of them, stride apart.
__device__ __forceinline__ void group_parts(const GnArgs &a, int b, int g, const float4 **p, int *n, int *stride) {
    *p = a.cl ? a.part + (long long)b * a.chunks * a.G + g : a.part + ((long long)b * a.C + g * a.cg) * a.chunks;
    *n = a.cl ? a.chunks : a.cg * a.chunks;
    *stride = a.cl ? a.G : 1;
}

// Statistics of the groups of a chunk's unit, into shared memory.  Where they are joined here (the same order in every CTA), no launch in between is
// needed.
__device__ __forceinline__ void unit_stats(const GnArgs &a, const Chunk &k, float4 *st) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g0 = a.cl ? 0 : (int)((unsigned)k.c / (unsigned)a.cg);  // first group of the unit
    if (a.direct) {
        for (int i = warp; i < a.gu; i += kWarps) {
            const float4 *p;
            int n, stride;
            group_parts(a, k.b, g0 + i, &p, &n, &stride);
            Sums64 m;
            m.gather(p, n, stride, lane, 32);
            if (lane == 0) {
                st[i] = m.stats(a);
                if (k.px0 == 0 && (a.cl || k.c == g0 * a.cg)) a.stats[k.b * a.G + g0 + i] = st[i];
            }
        }
    } else {
        for (int i = threadIdx.x; i < a.gu; i += kThreads) st[i] = __ldcg(a.stats + (long long)k.b * a.G + g0 + i);
    }
    __syncthreads();
}
// ... joined once: a CTA for every group of a sample
__global__ void __launch_bounds__(kThreads) gn_finish_stats_kernel(const __grid_constant__ GnArgs a) {
    __shared__ double red[kWarps * 3];
    const int warp = threadIdx.x >> 5, b = blockIdx.x / a.G, g = blockIdx.x - b * a.G;
    wait_for_previous();
    Sums64 m;
    const float4 *p;
    int n, stride;
    group_parts(a, b, g, &p, &n, &stride);
    m.gather(p, n, stride, threadIdx.x, kThreads);
    if ((threadIdx.x & 31) == 0) {
        red[warp * 3] = m.W;
        red[warp * 3 + 1] = m.s;
        red[warp * 3 + 2] = m.q;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kWarps; ++w) {
            m.W += red[w * 3];
            m.s += red[w * 3 + 1];
            m.q += red[w * 3 + 2];
        }
        a.stats[blockIdx.x] = m.stats(a);
    }
    let_next_begin();
}

template <typename T, bool PLANES> constexpr int kApplyCtas = sizeof(T) == 2 && !PLANES ? 3 : 4;  // on an SM: 8 slots of different channels keep
// more parameters than 4 CTAs leave registers for (721x1440x73 bf16 forward 106 us, at 3 103; 361x720x256 92 both; float32 gains from 4: 16x128x256x32 42 us, at 3 43)
constexpr int kApplyUnroll = 2;
using ApplyFeed = Feed<1, kApplyUnroll, 4>;  // (721x1440x73 float32 forward: 161 us with 4 rounds, 163 with 2, 158 with 6)

// z = (x - m) sc + sh, the difference first, in every type: with the mean in the shift, the shift is rounded at |m| r, and where a group is constant or
// nearly so r is up to eps^(-1/2) (a constant bf16 field of 101,376 came out 0.55 off, of 16-bit values exact as they are).  It costs 16-bit values a
// subtraction and the registers of m: 361x720x256 bf16 channels last with gelu, forward / backward, 92 / 138 us, folded 89 / 135; 721x1440x64 planes 86 / 135, folded 85 / 134.

// y of a piece.  Bound by the write of y and the read of what L2 no longer holds of x; with 16-bit values and an activation by
// its arithmetic too (721x1440x64 bf16 planes forward: 86 us with gelu and latitude weights, 72 without either).
template <typename T, int ACT, bool PLANES> __global__ void __launch_bounds__(kThreads, kApplyCtas<T, PLANES>) gn_apply_kernel(const __grid_constant__ GnArgs a) {
    constexpr int V = kV<T>, P = kP<T>, U = kApplyUnroll;
    extern __shared__ __align__(16) unsigned char gn_smem[];
    float4 *st = reinterpret_cast<float4 *>(gn_smem + ApplyFeed::bytes);
    const Chunk k = second_pass_chunk<T>(a, blockIdx.x);
    if (k.n <= 0) return;
    const T *x = reinterpret_cast<const T *>(a.x) + k.base;
    T *y = reinterpret_cast<T *>(a.out) + k.base;
    const uint4 *xv = reinterpret_cast<const uint4 *>(x + k.head);
    uint4 *yv = reinterpret_cast<uint4 *>(y + k.head);
    for (int win = 0; win < (PLANES ? 1 : a.windows); ++win) {
        const Share s = make_share<T, PLANES>(a, k, win);
        ApplyFeed feed;
        feed.start(gn_smem, xv + s.first, nullptr, s.count, s.step);  // (x was complete before the sums)
        F2 m[P], sc[P], sh[P];
        {
            float w[V], b[V];
            int g[V];
            slot_params<V, PLANES>(a, k, s.ch0, w, b, g);
            if (win == 0) {
                wait_for_previous();
                let_next_begin();
                unit_stats(a, k, st);
            }
#pragma unroll
            for (int p = 0; p < P; ++p) {
                const float4 u = st[g[2 * p]], v = st[g[2 * p + 1]];
                sc[p] = mul2(f2(u.z, v.z), f2(w[2 * p], w[2 * p + 1]));
                sh[p] = fma2(f2(-u.y, -v.y), sc[p], f2(b[2 * p], b[2 * p + 1]));
                m[p] = f2(u.x, v.x);
            }
        }
        const long long step = s.step;
        uint4 *to = yv + s.first;
        auto one = [&](uint4 raw) {
            F2 v[P];
            unpack(raw, v, T());
#pragma unroll
            for (int p = 0; p < P; ++p) v[p] = act_value<T, ACT>(fma2(sub2(v[p], m[p]), sc[p], sh[p]));
            return pack(v, T());
        };
        for (int j = 0; j < s.count; j += U) {
            feed.wait();
            uint4 raw[U];
#pragma unroll
            for (int u = 0; u < U; ++u) raw[u] = feed.get(u, 0);
            feed.next();
            if (j + U <= s.count) {
#pragma unroll
                for (int u = 0; u < U; ++u) to[u * step] = one(raw[u]);
            } else {
#pragma unroll
                for (int u = 0; u < U - 1; ++u)
                    if (j + u < s.count) to[u * step] = one(raw[u]);
            }
            to += U * step;
        }
    }
    if ((int)threadIdx.x < 2 * V) {
        const int e = ragged<T>(k, threadIdx.x);
        if (e >= 0) {
            const int ch = e % a.cu, c = a.cl ? ch : k.c;
            const float4 v = st[ch / a.cgu];
            const float sc = v.z * load_param(a.weight, a.pdtype, c, 1.f), sh = fmaf(-v.y, sc, load_param(a.bias, a.pdtype, c, 0.f));
            store_f(y + e, split(act_value<T, ACT>(f2(fmaf(to_f(x[e]) - v.x, sc, sh)))).x);
        }
    }
}

// ------------------------------------------------------------------------------------------------
// backward
// ------------------------------------------------------------------------------------------------
constexpr int kUnrollB = 2;
// On an SM: what a thread keeps of 8 slots and the activation's constants spills at 3 (361x720x256 bf16 167 us, at 2 138).  Planes have one channel's
// parameters and would take 3 without an activation, not with one (721x1440x64 bf16: none 121 us, at 2 127; gelu 139, at 2 135; float32 gelu 231, at 2 226).
constexpr int kBackwardCtas = 2;
using BackwardFeed = Feed<2, kUnrollB, 2>;  // (deeper was slower: 721x1440x73 bf16 155 us with 2 rounds, 165 with 3, 170 with 4; 721x1440x64 bf16 planes 135 with 2 and 3)

__device__ __forceinline__ void load_stats(const GnArgs &a, const Chunk &k, float4 *st) {
    if (a.cl)
        for (int g = threadIdx.x; g < a.G; g += kThreads) st[g] = __ldg(a.stats + (long long)k.b * a.G + g);
    else if (threadIdx.x == 0) st[0] = __ldg(a.stats + k.b * a.G + (int)((unsigned)k.c / (unsigned)a.cg));
}
// one value outside the vectors: (g, x - m)
template <typename T, int ACT> __device__ __forceinline__ float2 ragged_slope(const GnArgs &a, const Chunk &k, const float4 *st, float x, float dy, int ch) {
    const int c = a.cl ? ch : k.c;
    const float4 v = st[ch / a.cgu];
    const float sc = v.z * load_param(a.weight, a.pdtype, c, 1.f), sh = fmaf(-v.y, sc, load_param(a.bias, a.pdtype, c, 0.f)), d = x - v.x;
    return make_float2(dy * split(act_slope<ACT, false>(f2(kSlopeScale<ACT> * fmaf(d, sc, sh)))).x, d);
}

// (sum g, sum g xh) of the channels of a chunk: the slope is evaluated here and again in the second pass, since storing g would cost a write and a
// read of the field.  721x1440x64 float32 planes, with the pass below: 226 us, 5.9 TB/s over four reads and a write; with 16-bit values
// the registers that 8 slots take leave 16 warps an SM, which wait for their own results and at the barriers of a chunk's end (73 channels bf16: 155 us, 4.9 TB/s, 49 % of the issue slots).
template <typename T, int ACT, bool PLANES> __global__ void __launch_bounds__(kThreads, kBackwardCtas) gn_sums_kernel(const __grid_constant__ GnArgs a) {
    constexpr int V = kV<T>, P = kP<T>, U = kUnrollB;
    __shared__ __align__(16) F2 red[PLANES ? kWarps : 2 * P * kThreads];
    __shared__ __align__(16) F2 tot[PLANES ? 1 : 2 * P * kMaxCols];
    extern __shared__ __align__(16) unsigned char gn_smem[];
    float4 *st = reinterpret_cast<float4 *>(gn_smem + BackwardFeed::bytes);
    float2 *acc = reinterpret_cast<float2 *>(st + a.gu);
    const Chunk k = make_chunk<T>(a, blockIdx.x, 0, a.chunk_px);
    const T *x = reinterpret_cast<const T *>(a.x) + k.base, *dy = reinterpret_cast<const T *>(a.dy) + k.base;
    const uint4 *xv = reinterpret_cast<const uint4 *>(x + k.head), *dv = reinterpret_cast<const uint4 *>(dy + k.head);
    float2 *out = a.bpart + ((long long)k.unit * a.chunks + k.chunk) * a.cu;
    wait_for_previous();
    let_next_begin();
    load_stats(a, k, st);
    if (!PLANES)
        for (int c = threadIdx.x; c < a.cu; c += kThreads) acc[c] = make_float2(0.f, 0.f);
    __syncthreads();
    for (int win = 0; win < (PLANES ? 1 : a.windows); ++win) {
        const Share s = make_share<T, PLANES>(a, k, win);
        BackwardFeed feed;
        feed.start(gn_smem, xv + s.first, dv + s.first, s.count, s.step);
        F2 q[2 * P], m[P], sc[P], sh[P];  // q: sum g, sum g (x - m)
        {
            float w[V], b[V];
            int g[V];
            slot_params<V, PLANES>(a, k, s.ch0, w, b, g);
#pragma unroll
            for (int p = 0; p < P; ++p) {
                const float4 u = st[g[2 * p]], v = st[g[2 * p + 1]];
                m[p] = f2(u.x, v.x);
                sc[p] = mul2(f2(u.z * kSlopeScale<ACT>, v.z * kSlopeScale<ACT>), f2(w[2 * p], w[2 * p + 1]));
                sh[p] = fma2(f2(-u.y, -v.y), sc[p], f2(b[2 * p] * kSlopeScale<ACT>, b[2 * p + 1] * kSlopeScale<ACT>));
                q[p] = q[P + p] = f2(0.f);
            }
        }
        auto one = [&](uint4 rx, uint4 rd) {
            F2 v[P], d[P];
            unpack(rx, v, T());
            unpack(rd, d, T());
#pragma unroll
            for (int p = 0; p < P; ++p) {
                const F2 e = sub2(v[p], m[p]), g = mul2(d[p], act_slope<ACT, false>(fma2(e, sc[p], sh[p])));
                q[p] = add2(q[p], g);
                q[P + p] = fma2(g, e, q[P + p]);
            }
        };
        for (int j = 0; j < s.count; j += U) {
            feed.wait();
            uint4 rx[U], rd[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                rx[u] = feed.get(u, 0);
                rd[u] = feed.get(u, 1);
            }
            feed.next();
            one(rx[0], rd[0]);
            if (j + 1 < s.count) one(rx[1], rd[1]);
        }
        if constexpr (PLANES) {
            float v[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                F2 t = q[i * P];
#pragma unroll
                for (int p = 1; p < P; ++p) t = add2(t, q[i * P + p]);
                const float2 h = split(t);
                v[i] = h.x + h.y;
                for (int o = 16; o; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
            }
            float2 *w = reinterpret_cast<float2 *>(red);
            if ((threadIdx.x & 31) == 0) w[threadIdx.x >> 5] = make_float2(v[0], v[1]);
            __syncthreads();
            if (threadIdx.x == 0) {
                float2 t = w[0];
                for (int n = 1; n < kWarps; ++n) {
                    t.x += w[n].x;
                    t.y += w[n].y;
                }
                for (int i = 0; i < 2 * V; ++i) {
                    const int e = ragged<T>(k, i);
                    if (e < 0) break;
                    const float2 g = ragged_slope<T, ACT>(a, k, st, to_f(x[e]), to_f(dy[e]), 0);
                    t.x += g.x;
                    t.y = fmaf(g.x, g.y, t.y);
                }
                out[0] = make_float2(t.x, st[0].z * fmaf(-st[0].y, t.x, t.y));  // sum g (x - m) -> sum g xh
            }
        } else {
            column_sums(a, s, q, red, tot);
            const int period = a.cols * V, lo = win * a.win_cols * V, hi = min(lo + a.win_cols * V, period), shift = k.head % a.cu;
            for (int c = threadIdx.x; c < a.cu; c += kThreads) {
                float2 t = acc[c];
                for (int e = c >= shift ? c - shift : c - shift + a.cu; e < hi; e += a.cu)
                    if (e >= lo) {
                        const int col = (e - lo) / V, i = (e - lo) % V;
                        t.x += half_of(tot, i / 2, col, i & 1);
                        t.y += half_of(tot, P + i / 2, col, i & 1);
                    }
                if (win == 0)
                    for (int i = 0; i < 2 * V; ++i) {
                        const int e = ragged<T>(k, i);
                        if (e < 0) break;
                        if (e % a.cu == c) {
                            const float2 g = ragged_slope<T, ACT>(a, k, st, to_f(x[e]), to_f(dy[e]), c);
                            t.x += g.x;
                            t.y = fmaf(g.x, g.y, t.y);
                        }
                    }
                acc[c] = t;
                if (win == a.windows - 1) {
                    const float4 v = st[c / a.cgu];
                    out[c] = make_float2(t.x, v.z * fmaf(-v.y, t.x, t.y));
                }
            }
            if (a.windows > 1) __syncthreads();
        }
    }
}

// (sum h, sum h xh) of the groups of a chunk's unit
__device__ void group_sums(const GnArgs &a, const Chunk &k, float2 *gsum) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (a.cl || !a.direct) {
        const int g0 = a.cl ? 0 : (int)((unsigned)k.c / (unsigned)a.cg);  // first group of the unit
        for (int j = warp; j < a.gu; j += kWarps) {
            const int g = g0 + j;
            double2 t = make_double2(0., 0.);
            if (a.direct) {
                for (int i = lane; i < a.cg * a.chunks; i += 32) {
                    const int n = (int)((unsigned)i / (unsigned)a.cg), c = g * a.cg + (i - n * a.cg);
                    const double w = load_param(a.weight, a.pdtype, c, 1.f);
                    const float2 v = __ldcg(a.bpart + ((long long)k.b * a.chunks + n) * a.C + c);
                    t.x += w * v.x;
                    t.y += w * v.y;
                }
            } else {
                for (int i = lane; i < a.cg; i += 32) {
                    const int c = g * a.cg + i;
                    const double w = load_param(a.weight, a.pdtype, c, 1.f);
                    const double2 v = __ldcg(a.csum + (long long)k.b * a.C + c);
                    t.x += w * v.x;
                    t.y += w * v.y;
                }
            }
            t = warp_sum(t);
            if (lane == 0) gsum[j] = make_float2((float)t.x, (float)t.y);
        }
    } else if (warp == 0) {
        const int first = k.c - (int)((unsigned)k.c % (unsigned)a.cg);  // first channel of the group
        const float2 *p = a.bpart + ((long long)k.b * a.C + first) * a.chunks;
        double2 t = make_double2(0., 0.);
        const int n = a.cg * a.chunks;
        for (int i = lane; i < n; i += 128) {
            float2 v[4];
            float w[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int e = min(i + 32 * u, n - 1);
                v[u] = __ldcg(p + e);
                w[u] = i + 32 * u < n ? load_param(a.weight, a.pdtype, first + (a.cg == 1 ? 0 : (int)((unsigned)e / (unsigned)a.chunks)), 1.f) : 0.f;
            }
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (i + 32 * u < n) {
                    t.x += (double)w[u] * v[u].x;
                    t.y += (double)w[u] * v[u].y;
                }
        }
        t = warp_sum(t);
        if (lane == 0) gsum[0] = make_float2((float)t.x, (float)t.y);
    }
}
// ... the sums of the channels joined once: a CTA for 4 channels of a sample (32 bytes of every chunk), the chunks dealt to 64 lanes a channel
constexpr int kFinishChannels = 4;
__global__ void __launch_bounds__(kThreads) gn_finish_sums_kernel(const __grid_constant__ GnArgs a) {
    __shared__ double2 red[kWarps * kFinishChannels];
    const int blocks = (a.C + kFinishChannels - 1) / kFinishChannels, b = blockIdx.x / blocks;
    const int i = threadIdx.x % kFinishChannels, first = threadIdx.x / kFinishChannels, c = (blockIdx.x - b * blocks) * kFinishChannels + i;
    constexpr int kRows = kThreads / kFinishChannels;
    wait_for_previous();
    double2 v = make_double2(0., 0.);
    if (c < a.C)
        for (int n = first; n < a.chunks; n += 8 * kRows) {
            float2 p[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) p[u] = n + u * kRows < a.chunks ? __ldcg(a.bpart + (a.cl ? ((long long)b * a.chunks + n + u * kRows) * a.C + c : ((long long)b * a.C + c) * a.chunks + n + u * kRows)) : make_float2(0.f, 0.f);
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                v.x += p[u].x;
                v.y += p[u].y;
            }
        }
    for (int o = 16; o >= kFinishChannels; o >>= 1) {
        v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
        v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
    if ((threadIdx.x & 31) < kFinishChannels) red[(threadIdx.x >> 5) * kFinishChannels + i] = v;
    __syncthreads();
    if (threadIdx.x < kFinishChannels && c < a.C) {
        for (int w = 1; w < kWarps; ++w) {
            v.x += red[w * kFinishChannels + i].x;
            v.y += red[w * kFinishChannels + i].y;
        }
        a.csum[(long long)b * a.C + c] = v;
    }
    let_next_begin();
}

// The parameters' gradients, one warp a channel, over all samples.
__device__ __forceinline__ void parameter_gradients(const GnArgs &a, int block) {
    const int lane = threadIdx.x & 31, c = block * kWarps + (int)(threadIdx.x >> 5);
    if (c >= a.C) return;
    double2 v = make_double2(0., 0.);
    if (!a.direct) {
        for (int b = lane; b < a.B; b += 32) {
            const double2 p = __ldcg(a.csum + (long long)b * a.C + c);
            v.x += p.x;
            v.y += p.y;
        }
    } else {
        for (long long n = lane; n < (long long)a.B * a.chunks; n += 32) {
            const long long b = n / a.chunks, i = n - b * a.chunks;
            const float2 p = __ldcg(a.bpart + (a.cl ? n * a.C + c : (b * a.C + c) * a.chunks + i));
            v.x += p.x;
            v.y += p.y;
        }
    }
    v = warp_sum(v);
    if (lane == 0) {
        store_param(a.dbias, a.pdtype, c, (float)v.x);
        store_param(a.dweight, a.pdtype, c, (float)v.y);
    }
}

// dx = sc g - a (alpha + (x - m) beta),  alpha = r (sum h - lo r sum h xh) / sum a,  beta = r^2 sum h xh / sum a
__device__ __forceinline__ float2 group_terms(const float4 &v, const float2 &t) { return make_float2(-v.z * fmaf(-v.y * v.z, t.y, t.x) * v.w, -v.z * v.z * t.y * v.w); }

// dx of a piece.  The last CTAs of the grid compute the parameters' gradients: no launch of their own.
template <typename T, int ACT, bool PLANES> __global__ void __launch_bounds__(kThreads, kBackwardCtas) gn_dx_kernel(const __grid_constant__ GnArgs a) {
    constexpr int V = kV<T>, P = kP<T>, U = kUnrollB;
    const int tasks = a.out ? a.tasks * a.pieces : 0;
    if ((int)blockIdx.x >= tasks) {
        wait_for_previous();
        parameter_gradients(a, (int)blockIdx.x - tasks);
        return;
    }
    extern __shared__ __align__(16) unsigned char gn_smem[];
    float4 *st = reinterpret_cast<float4 *>(gn_smem + BackwardFeed::bytes);
    float2 *gsum = reinterpret_cast<float2 *>(st + a.gu);
    const Chunk k = second_pass_chunk<T>(a, blockIdx.x);
    if (k.n <= 0) return;
    const T *x = reinterpret_cast<const T *>(a.x) + k.base, *dy = reinterpret_cast<const T *>(a.dy) + k.base;
    T *dx = reinterpret_cast<T *>(a.out) + k.base;
    const uint4 *xv = reinterpret_cast<const uint4 *>(x + k.head), *dv = reinterpret_cast<const uint4 *>(dy + k.head);
    uint4 *ov = reinterpret_cast<uint4 *>(dx + k.head);
    for (int win = 0; win < (PLANES ? 1 : a.windows); ++win) {
        const Share s = make_share<T, PLANES>(a, k, win);
        BackwardFeed feed;
        feed.start(gn_smem, xv + s.first, dv + s.first, s.count, s.step);  // (x and dy were complete before the sums)
        if (win == 0) {
            wait_for_previous();
            let_next_begin();
            load_stats(a, k, st);
            group_sums(a, k, gsum);
            __syncthreads();
        }
        F2 m[P], sc[P], sh[P], al[P], be[P];
        {
            float w[V], b[V];
            int g[V];
            slot_params<V, PLANES>(a, k, s.ch0, w, b, g);
#pragma unroll
            for (int p = 0; p < P; ++p) {
                const float4 u = st[g[2 * p]], v = st[g[2 * p + 1]];
                const float2 tu = group_terms(u, gsum[g[2 * p]]), tv = group_terms(v, gsum[g[2 * p + 1]]);
                sc[p] = mul2(f2(u.z * kSlopeScale<ACT>, v.z * kSlopeScale<ACT>), f2(w[2 * p], w[2 * p + 1]));
                sh[p] = fma2(f2(-u.y, -v.y), sc[p], f2(b[2 * p] * kSlopeScale<ACT>, b[2 * p + 1] * kSlopeScale<ACT>));
                al[p] = f2(tu.x, tv.x);
                be[p] = f2(tu.y, tv.y);
                m[p] = f2(u.x, v.x);
            }
        }
        if (!s.count) continue;
        const long long step = s.step;
        uint4 *to = ov + s.first;
        Rows r{0, 0, 0};
        float w = 1.f;
        if (a.lat) {
            r = make_rows<T>(a, k, s, 0);
            w = __ldg(a.lat + r.row);
        }
        auto one = [&](uint4 rx, uint4 rd, const F2 (&wt)[P]) {
            F2 v[P], d[P];
            unpack(rx, v, T());
            unpack(rd, d, T());
#pragma unroll
            for (int p = 0; p < P; ++p) {
                const F2 e = sub2(v[p], m[p]), g = mul2(d[p], act_slope<ACT, true>(fma2(e, sc[p], sh[p])));
                v[p] = fma2(wt[p], fma2(e, be[p], al[p]), mul2(sc[p], g));
            }
            return pack(v, T());
        };
        for (int j = 0; j < s.count; j += U) {
            const int have = min(U, s.count - j);
            uint4 rx[U], rd[U];
            feed.wait();
#pragma unroll
            for (int u = 0; u < U; ++u) {
                rx[u] = feed.get(u, 0);
                rd[u] = feed.get(u, 1);
            }
            feed.next();
            F2 wt[P];
            float wu[U];
            if (round_weights<U, PLANES>(a, have, r, w, wu)) {
#pragma unroll
                for (int u = 0; u < U; ++u) {
#pragma unroll
                    for (int p = 0; p < P; ++p) wt[p] = f2(wu[u]);
                    to[u * step] = one(rx[u], rd[u], wt);
                }
            } else {
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (u < have) {
#pragma unroll
                        for (int p = 0; p < P; ++p) wt[p] = f2(w);
                        if (a.lat && r.col + r.over >= a.nlon) {
                            float ws[V];
                            mixed_weights<T>(a.lat, a.nlon, a.cu, s.ch0, r.row, r.col, ws);
#pragma unroll
                            for (int p = 0; p < P; ++p) wt[p] = f2(ws[2 * p], ws[2 * p + 1]);
                        }
                        to[u * step] = one(rx[u], rd[u], wt);
                        if (a.lat) {
                            advance(a, r);
                            w = __ldg(a.lat + min(r.row, a.nlat - 1));
                        }
                    }
            }
            to += U * step;
        }
    }
    if ((int)threadIdx.x < 2 * V) {
        const int e = ragged<T>(k, threadIdx.x);
        if (e >= 0) {
            const int ch = e % a.cu, g = ch / a.cgu;
            const float2 t = group_terms(st[g], gsum[g]), u = ragged_slope<T, ACT>(a, k, st, to_f(x[e]), to_f(dy[e]), ch);
            const float sc = st[g].z * load_param(a.weight, a.pdtype, a.cl ? ch : k.c, 1.f);
            store_f(dx + e, fmaf(weight_at(a, k, e), fmaf(u.y, t.y, t.x), sc * u.x));
        }
    }
}

// ------------------------------------------------------------------------------------------------
// host
// ------------------------------------------------------------------------------------------------
constexpr int kMaxChannels = SHTB200_GROUP_NORM_MAX_CHANNELS;  // what a CTA keeps per channel or group has to fit into its shared memory
// Partial results of a group up to which every CTA joins them itself, a warp a group, instead of a launch in between.  (256x512x32 float32,
// forward: 29 us with the launch, 39 without, which a limit of 512 would choose; 16x128x256x32: 42 us without, 43 with, which 32 would.)
constexpr int kDirect = 128;

int value_bytes(int dtype) { return dtype == SHTB200_F32 ? 4 : 2; }
size_t up256(size_t b) { return (b + 255) / 256 * 256; }

struct Launch {
    GnArgs a{};
    size_t part = 0, csum = 0;  // bytes of workspace
    size_t total() const { return part + csum; }
};

// Pieces of a chunk for the second pass: small ones follow what L2 holds more closely, large ones pay a CTA's start less often.  Forward, 721x1440x73
// float32: 161 us, with whole chunks 166; 721x1440x64 bf16 planes 86 and 100; 361x720x256 bf16: 92 us, with pieces of half the size 94 (backward, where they
// are twice as large: 138 us, with half the size 145).
constexpr long long kPieceBytes = 128 << 10;
constexpr int kMaxPieces = 4;

Launch geometry(const GroupNormDesc &d, bool backward) {
    Launch l;
    GnArgs &a = l.a;
    const int V = 16 / value_bytes(d.dtype);
    a.hw = (long long)d.nlat * d.nlon;
    a.B = d.batch;
    a.C = d.channels;
    a.G = d.groups;
    a.cg = a.C / a.G;
    a.nlat = d.nlat;
    a.nlon = d.nlon;
    a.cl = d.channels_last;
    a.pdtype = d.param_dtype;
    a.eps = d.eps;
    a.cu = a.cl ? a.C : 1;
    a.gu = a.cl ? a.G : 1;
    a.cgu = a.cl ? a.cg : 1;
    // columns
    a.cols = a.cu / std::gcd(a.cu, V);
    a.dup = a.cols * V / a.cu;
    a.windows = ceil_div(a.cols, kMaxCols);
    a.win_cols = ceil_div(a.cols, a.windows);
    a.reps = kThreads / a.win_cols;
    for (a.lanes = 1; a.lanes < 32 && a.lanes < a.cgu * a.dup;) a.lanes *= 2;
    const long long step_px = a.cu == 1 ? 32 * V : (long long)a.reps * a.cols * V / a.cu;
    a.step_px = (int)step_px;
    a.step_rows = (int)(step_px / a.nlon);
    a.step_cols = (int)(step_px % a.nlon);
    // Chunks for the sums: one for every CTA that 148 SMs hold, but none under 16 KB, what a CTA does besides costing some microseconds (128x256x32 bf16
    // forward and backward: 16.0 and 16.4 us, with 4 KB 19.6 and 18.4, with 64 KB 18.2 and 20.7).
    const int units = a.cl ? a.B : a.B * a.C, ctas = 148 * (backward ? kBackwardCtas : V == 4 ? kStatsCtas<float> : kStatsCtas<__half>);
    const long long unit_vecs = a.hw * a.cu / V, most = std::max<long long>(1, std::min<long long>(a.hw, unit_vecs / (kThreads * 4)));
    const long long n = std::min<long long>(most, std::max(1, ctas / units));
    a.chunk_px = (int)((a.hw + n - 1) / n);
    if (a.chunk_px >= 256) a.chunk_px = (a.chunk_px + 31) / 32 * 32;  // (chunks of an aligned field begin aligned)
    a.chunks = (int)((a.hw + a.chunk_px - 1) / a.chunk_px);
    a.tasks = units * a.chunks;
    // pieces of them for the second pass
    a.pieces = (int)std::max<long long>(1, std::min<long long>(kMaxPieces, (long long)a.chunk_px * a.cu * value_bytes(d.dtype) / (backward ? 2 * kPieceBytes : kPieceBytes)));
    a.piece_px = ceil_div(a.chunk_px, a.pieces);
    if (a.piece_px >= 256) a.piece_px = (a.piece_px + 31) / 32 * 32;
    a.direct = a.gu <= kWarps && (long long)a.chunks * (backward || !a.cl ? a.cg : 1) <= kDirect;
    l.part = up256((size_t)a.tasks * (backward ? a.cu * sizeof(float2) : a.gu * sizeof(float4)));
    if (backward && !a.direct) l.csum = up256((size_t)a.B * a.C * sizeof(double2));
    return l;
}

// Once for every kernel and device (and size, where it grows): dynamic shared memory beyond the default.
int allow_smem(const void *kernel, size_t smem) {
    static std::mutex mutex;
    static std::map<std::pair<const void *, int>, size_t> allowed;
    int dev = 0;
    SHT_CUDA_CHECK(cudaGetDevice(&dev));
    std::lock_guard<std::mutex> lock(mutex);
    size_t &have = allowed[{kernel, dev}];
    if (have >= smem) return SHTB200_OK;
    SHT_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    have = smem;
    return SHTB200_OK;
}

// A launch that may begin while the one before it ends (the kernels wait for its results themselves).
int launch(const void *kernel, int grid, size_t smem, const GnArgs &a, cudaStream_t st) {
    int rc = allow_smem(kernel, smem);
    if (rc) return rc;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    void *args[] = {const_cast<GnArgs *>(&a)};
    SHT_CUDA_CHECK(cudaLaunchKernelExC(&cfg, kernel, args));
    return SHTB200_OK;
}

// the kernel of a descriptor's type, activation and layout
enum Which { kStats, kApply, kSums, kDx };
template <typename T, int ACT, bool PLANES> const void *kernel_of(Which w) {
    switch (w) {
        case kStats: return (const void *)gn_stats_kernel<T, PLANES>;
        case kApply: return (const void *)gn_apply_kernel<T, ACT, PLANES>;
        case kSums: return (const void *)gn_sums_kernel<T, ACT, PLANES>;
        default: return (const void *)gn_dx_kernel<T, ACT, PLANES>;
    }
}
template <typename T, int ACT> const void *kernel_of(Which w, bool planes) { return planes ? kernel_of<T, ACT, true>(w) : kernel_of<T, ACT, false>(w); }
template <typename T> const void *kernel_of(Which w, bool planes, int act) {
    switch (act) {
        case SHTB200_ACT_RELU: return kernel_of<T, SHTB200_ACT_RELU>(w, planes);
        case SHTB200_ACT_SILU: return kernel_of<T, SHTB200_ACT_SILU>(w, planes);
        case SHTB200_ACT_GELU: return kernel_of<T, SHTB200_ACT_GELU>(w, planes);
        default: return kernel_of<T, SHTB200_ACT_NONE>(w, planes);
    }
}
const void *kernel_of(Which w, const GroupNormDesc &d, const GnArgs &a) {
    const bool planes = a.cu == 1;
    return d.dtype == SHTB200_F32 ? kernel_of<float>(w, planes, d.activation) : d.dtype == SHTB200_BF16 ? kernel_of<__nv_bfloat16>(w, planes, d.activation) : kernel_of<__half>(w, planes, d.activation);
}

int check_desc(const GroupNormDesc *d) {
    if (!d) return fail(SHTB200_EINVAL, "group norm descriptor is null");
    if (d->batch < 0 || d->channels < 1 || d->groups < 1 || d->nlat < 1 || d->nlon < 1) return fail(SHTB200_EINVAL, "bad group norm shape");
    if (d->channels % d->groups) return fail(SHTB200_EINVAL, "channels must be divisible by groups");
    if (d->dtype < SHTB200_F32 || d->dtype > SHTB200_F16 || d->param_dtype < SHTB200_F32 || d->param_dtype > SHTB200_F16) return fail(SHTB200_EINVAL, "unknown element type");
    if (d->activation < SHTB200_ACT_NONE || d->activation > SHTB200_ACT_GELU) return fail(SHTB200_EINVAL, "unknown activation");
    if (!(d->eps >= 0.f)) return fail(SHTB200_EINVAL, "eps must be >= 0");
    if (d->channels > kMaxChannels) return fail(SHTB200_EINVAL, "at most " + std::to_string(kMaxChannels) + " channels");
    // a chunk's values are counted in 32 bits
    if ((long long)d->batch * d->channels > (1LL << 24) || (long long)d->nlat * d->nlon > (1LL << 30) || (long long)d->nlat * d->nlon * (d->channels_last ? d->channels : 1) > (1LL << 36))
        return fail(SHTB200_EINVAL, "group norm shape too large");
    return SHTB200_OK;
}

int plan(const GroupNormDesc *d, bool backward, const void *ws, size_t ws_bytes, const void *stats, Launch *l) {
    *l = geometry(*d, backward);
    if (!ws || ws_bytes < l->total()) return fail(SHTB200_EWORKSPACE, "workspace too small: need " + std::to_string(l->total()) + " bytes");
    if (((uintptr_t)ws & 255) != 0) return fail(SHTB200_EINVAL, "workspace must be 256-byte aligned");
    if (((uintptr_t)stats & 15) != 0) return fail(SHTB200_EINVAL, "the statistics must be 16-byte aligned");
    if ((long long)l->a.chunk_px * l->a.cu > (1 << 30) || (long long)l->a.tasks * l->a.pieces > (1 << 30)) return fail(SHTB200_EINVAL, "group norm shape too large");
    return SHTB200_OK;
}
// every value lies on a multiple of its size (vectors begin a whole number of values behind the first)
int check_values(const GroupNormDesc &d, std::initializer_list<const void *> fields, std::initializer_list<const void *> params, const float *lat) {
    uintptr_t f = 0, p = 0;
    for (const void *t : fields) f |= (uintptr_t)t;
    for (const void *t : params) p |= (uintptr_t)t;
    if (f % value_bytes(d.dtype) || p % value_bytes(d.param_dtype) || (uintptr_t)lat % sizeof(float)) return fail(SHTB200_EINVAL, "a tensor is not aligned to its element type");
    return SHTB200_OK;
}
// vectors are aligned in all tensors or in none
bool aligned_alike(const void *p, const void *q) { return !p || !q || (((uintptr_t)p ^ (uintptr_t)q) & 15) == 0; }

}  // namespace

size_t group_norm_workspace(const GroupNormDesc *d, bool backward) {
    if (check_desc(d)) return 0;
    if (d->batch == 0) return 256;
    return std::max<size_t>(geometry(*d, backward).total(), 256);
}

int group_norm_forward(const GroupNormDesc *d, const void *x, const float *lat, const void *weight, const void *bias, void *y, void *stats, void *ws, size_t ws_bytes,
                       cudaStream_t st) {
    int rc = check_desc(d);
    if (rc) return rc;
    if (d->batch == 0) return SHTB200_OK;
    if (!x || !y || !stats) return fail(SHTB200_EINVAL, "null pointer");
    if ((rc = check_values(*d, {x, y}, {weight, bias}, lat))) return rc;
    if (!aligned_alike(x, y)) return fail(SHTB200_EINVAL, "x and y must have the same address modulo 16");
    Launch l;
    if ((rc = plan(d, false, ws, ws_bytes, stats, &l))) return rc;
    GnArgs &a = l.a;
    a.x = x;
    a.out = y;
    a.lat = lat;
    a.weight = weight;
    a.bias = bias;
    a.stats = reinterpret_cast<float4 *>(stats);
    a.part = reinterpret_cast<float4 *>(ws);
    if ((rc = launch(kernel_of(kStats, *d, a), a.tasks, StatsFeed::bytes + (a.cu > 1 ? sizeof(Moments) * a.gu : 0), a, st))) return rc;
    if (!a.direct && (rc = launch((const void *)gn_finish_stats_kernel, a.B * a.G, 0, a, st))) return rc;
    return launch(kernel_of(kApply, *d, a), a.tasks * a.pieces, ApplyFeed::bytes + sizeof(float4) * a.gu, a, st);
}

int group_norm_backward(const GroupNormDesc *d, const void *dy, const void *x, const float *lat, const void *weight, const void *bias, const void *stats, void *dx, void *dweight,
                        void *dbias, void *ws, size_t ws_bytes, cudaStream_t st) {
    int rc = check_desc(d);
    if (rc) return rc;
    if (d->batch == 0) return fail(SHTB200_EINVAL, "an empty batch has no gradient to compute");
    if (!x || !dy || !stats) return fail(SHTB200_EINVAL, "null pointer");
    if ((rc = check_values(*d, {x, dy, dx}, {weight, bias, dweight, dbias}, lat))) return rc;
    if (!aligned_alike(x, dy) || !aligned_alike(x, dx)) return fail(SHTB200_EINVAL, "x, dy and dx must have the same address modulo 16");
    Launch l;
    if ((rc = plan(d, true, ws, ws_bytes, stats, &l))) return rc;
    GnArgs &a = l.a;
    a.x = x;
    a.dy = dy;
    a.out = dx;
    a.lat = lat;
    a.weight = weight;
    a.bias = bias;
    a.dweight = dweight;
    a.dbias = dbias;
    a.stats = reinterpret_cast<float4 *>(const_cast<void *>(stats));
    a.bpart = reinterpret_cast<float2 *>(ws);
    a.csum = reinterpret_cast<double2 *>(reinterpret_cast<char *>(ws) + l.part);
    const int grads = dweight || dbias ? ceil_div(a.C, kWarps) : 0;
    if (!dx && !grads) return SHTB200_OK;
    const size_t smem = BackwardFeed::bytes + sizeof(float4) * a.gu + sizeof(float2) * std::max(a.cu, a.gu);
    if ((rc = launch(kernel_of(kSums, *d, a), a.tasks, smem, a, st))) return rc;
    if (!a.direct && (rc = launch((const void *)gn_finish_sums_kernel, a.B * ceil_div(a.C, kFinishChannels), 0, a, st))) return rc;
    return launch(kernel_of(kDx, *d, a), (dx ? a.tasks * a.pieces : 0) + grads, smem, a, st);
}

}  // namespace shtb200
