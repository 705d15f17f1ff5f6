// Group normalisation with an activation on fields over the sphere, forward and backward.
//
// x (B, C, nlat, nlon), planes or channels last, G groups of C / G channels, a_k = weight of latitude row k:
//     mu = sum a x / sum a,  v = sum a (x - mu)^2 / sum a      (over the C / G channels and all grid points of a group)
//     xh = (x - mu) r,  r = (v + eps)^(-1/2),  z = w_c xh + b_c,  y = act(z)
// With g = dy act'(z), h = w_c g and q = a / sum a:
//     db_c = sum g,  dw_c = sum g xh,  dx = r (h - q (sum h + xh sum h xh)).
// A few operations per element: all of it is bound by memory, x (and dy) being read twice unless the second read finds them in L2.
//
// One cooperative launch a direction.  The work is cut into units (a sample, channels last; a plane, otherwise), units into chunks of
// pixels, and units are taken in batches that fit into L2: while a batch is normalised, the sums of the next one are taken, so that its
// second read does not go to memory.  A chunk is read as one flat stream of 16-byte vectors: with C' interleaved channels (C, or 1 for
// planes) and V values a vector, a thread that steps by a multiple of lcm(C', V) values meets the same channels in every
// vector ("slots"), whatever C' is, and keeps their sums and parameters in registers.
//
// Sums for the variance are taken about a centre c per slot, (W, c, S1, S2) = (sum a, c, sum a (x - c), sum a (x - c)^2).  c begins as a value
// of the field and is moved to the mean so far after 1, 2, 4, 8, ... rounds; fields whose level is far above their spread (pressures) or
// that have a value far out lose nothing.  Chunks are joined in float64 as (W, K, mean - K, M2).

#include "common.cuh"

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <numeric>

namespace cg = cooperative_groups;

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
// against the scaled complementary error function).  gelu(z) = max(z, 0) - a Phi(-a) then keeps its relative accuracy in both tails.
struct Tail {
    F2 e, r, na;  // e^(-a^2 / 2), R(a), -a
};
__device__ __forceinline__ Tail normal_tail(F2 z) {
    Tail k;
    k.na.v = z.v | 0x8000000080000000ull;
    const float2 d = split(fma2(k.na, f2(-0.3f), f2(1.f)));
    const F2 t = f2(rcp_fast(d.x), rcp_fast(d.y));
    F2 p = fma2(t, f2(0.035931703f), f2(-0.15827584f));
    p = fma2(t, p, f2(0.20820633f));
    p = fma2(t, p, f2(-0.05539357f));
    p = fma2(t, p, f2(0.12946904f));
    p = fma2(t, p, f2(0.099637546f));
    p = fma2(t, p, f2(0.12079835f));
    p = fma2(t, p, f2(0.11962639f));
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

template <int ACT> __device__ __forceinline__ F2 act_value(F2 z) {
    if constexpr (ACT == SHTB200_ACT_RELU) {
        const float2 v = split(z);
        return f2(v.x <= 0.f ? 0.f : v.x, v.y <= 0.f ? 0.f : v.y);  // (a NaN stays one)
    } else if constexpr (ACT == SHTB200_ACT_SILU) {
        return mul2(z, logistic(z));
    } else if constexpr (ACT == SHTB200_ACT_GELU) {
        const Tail k = normal_tail(z);
        const float2 v = split(z);
        return fma2(k.na, mul2(k.e, k.r), f2(fmaxf(v.x, 0.f), fmaxf(v.y, 0.f)));
    }
    return z;
}
template <int ACT> __device__ __forceinline__ F2 act_slope(F2 z) {
    if constexpr (ACT == SHTB200_ACT_RELU) {
        const float2 v = split(z);
        return f2(v.x <= 0.f ? 0.f : 1.f, v.y <= 0.f ? 0.f : 1.f);
    } else if constexpr (ACT == SHTB200_ACT_SILU) {
        const F2 s = logistic(z);
        return fma2(mul2(z, s), fma2(s, f2(-1.f), f2(1.f)), s);
    } else if constexpr (ACT == SHTB200_ACT_GELU) {
        const Tail k = normal_tail(z);
        const F2 s = mul2(k.e, fma2(k.na, f2(0.39894228f), k.r));  // the slope at -a; at a it is one less this
        const float2 m = split(s), p = split(fma2(s, f2(-1.f), f2(1.f))), v = split(z);
        return f2(v.x > 0.f ? p.x : m.x, v.y > 0.f ? p.y : m.y);
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
constexpr int kCtasPerSm = 2;

struct GnArgs {
    const void *x, *dy;
    void *out;
    const float *lat;  // nullptr: 1 everywhere
    const void *weight, *bias;
    void *dweight, *dbias;
    float4 *stats;     // (B, G): mean, its low part, r, 1 / sum a
    float4 *part;      // forward: (unit, chunk, group of the unit): (W, K, mean - K, M2)
    float2 *bpart;     // backward: (unit, chunk, channel of the unit): (sum g, sum g xh)
    double2 *csum;     // backward, channels last: (B, C): the same over all chunks
    long long hw;
    int B, C, G, cg, nlat, nlon, cl, pdtype;
    float eps;
    int cu, gu, cgu;   // channels, groups of a unit, channels of a group inside a unit: (C, G, cg) channels last, (1, 1, 1) for planes
    int units;         // B or B C
    int batch_units, batches;
    int chunks;        // of a unit
    int chunk_px;
    int cols;          // lcm(cu, V) / V: vectors after which the channels repeat
    int win_cols, windows, reps;  // columns a CTA covers at a time, how many windows that takes, vectors of a column it has in flight
    int step_rows, step_cols;     // reps columns further in pixels, as rows and columns of the grid
    int sync;          // 0: every group lies in one chunk
};

// A chunk of a unit: n values from `base` on; `head` of them lie before the first aligned vector, then `vecs` vectors, then the tail.
struct Chunk {
    int unit, chunk, b;
    long long base;  // first value
    int px0;         // its pixel
    int n, head, vecs;
};
template <typename T> __device__ __forceinline__ Chunk make_chunk(const GnArgs &a, int first_unit, int task, const void *align) {
    Chunk k;
    k.unit = first_unit + task / a.chunks;
    k.chunk = task % a.chunks;
    k.b = a.cl ? k.unit : k.unit / a.C;
    k.px0 = k.chunk * a.chunk_px;
    const int px = (int)min((long long)a.chunk_px, a.hw - k.px0);
    k.base = ((long long)k.unit * a.hw + k.px0) * a.cu;
    k.n = px * a.cu;
    const unsigned mis = (unsigned)((uintptr_t)(reinterpret_cast<const T *>(align) + k.base) & 15u);
    k.head = min(k.n, (int)((16u - mis) & 15u) / (int)sizeof(T));
    k.vecs = (k.n - k.head) / kV<T>;
    return k;
}

// A thread's share of a window of a chunk: vectors first, first + step, ... (count of them); the channel (of the unit) of slot 0.
struct Share {
    int first, step, count, ch0, rep, col;
};
template <typename T> __device__ __forceinline__ Share make_share(const GnArgs &a, const Chunk &k, int window) {
    Share s;
    const int cols = min(a.win_cols, a.cols - window * a.win_cols);
    s.rep = (int)threadIdx.x / a.win_cols;
    s.col = (int)threadIdx.x - s.rep * a.win_cols;
    const int c = window * a.win_cols + s.col;
    s.first = c + s.rep * a.cols;
    s.step = a.reps * a.cols;
    s.count = (s.rep < a.reps && s.col < cols && s.first < k.vecs) ? (k.vecs - s.first + s.step - 1) / s.step : 0;
    s.ch0 = a.cu == 1 ? 0 : (int)(((long long)c * kV<T> + k.head) % a.cu);
    return s;
}

// Latitude weight of the vectors of a share.  A vector lies in one row, but for those across a row's end.
struct Rows {
    int row, col, over;  // of slot 0; pixels from slot 0 to the last slot
};
template <typename T> __device__ __forceinline__ Rows make_rows(const GnArgs &a, const Chunk &k, const Share &s, int j) {
    Rows r;
    const long long e = (long long)k.head + ((long long)s.first + (long long)j * s.step) * kV<T>;
    const int px = k.px0 + (a.cu == 1 ? (int)e : (int)(e / a.cu));
    r.row = px / a.nlon;
    r.col = px - r.row * a.nlon;
    r.over = a.cu == 1 ? kV<T> - 1 : (s.ch0 + kV<T> - 1) / a.cu;
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
__device__ __forceinline__ void retreat(const GnArgs &a, Rows &r) {
    r.row -= a.step_rows;
    r.col -= a.step_cols;
    if (r.col < 0) {
        r.col += a.nlon;
        --r.row;
    }
}
// weights of the slots of a vector across a row's end
template <typename T> __device__ __noinline__ void mixed_weights(const float *lat, int nlon, int cu, int ch0, int row, int col, float *w) {
    for (int i = 0; i < kV<T>; ++i) {
        const int px = col + (ch0 + i) / cu;
        w[i] = lat[row + px / nlon];
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

// ------------------------------------------------------------------------------------------------
// joining of moments
// ------------------------------------------------------------------------------------------------
struct Moments {  // (sum of weights, K, mean - K, M2)
    float W, K, m, M2;
};
__device__ __forceinline__ void join(Moments &a, const Moments &b) {
    if (b.W == 0.f) return;
    if (a.W == 0.f) {
        a = b;
        return;
    }
    const float W = a.W + b.W, f = __fdividef(b.W, W), d = (b.K - a.K) + (b.m - a.m);
    a.m = fmaf(d, f, a.m);
    a.M2 += fmaf(d * d, a.W * f, b.M2);
    a.W = W;
}
struct Moments64 {
    double W, mean, M2;
};
__device__ __forceinline__ void join(Moments64 &a, const Moments64 &b) {
    if (b.W == 0.) return;
    const double W = a.W + b.W, f = b.W / W, d = b.mean - a.mean;
    a.mean += d * f;
    a.M2 += b.M2 + d * d * a.W * f;
    a.W = W;
}
__device__ __forceinline__ Moments64 widen(float4 v) { return {v.x, (double)v.y + v.z, v.w}; }

__device__ __forceinline__ float4 finished(const GnArgs &a, const Moments64 &m) {
    const float hi = (float)m.mean;
    return make_float4(hi, (float)(m.mean - hi), (float)(1. / sqrt(m.M2 / m.W + (double)a.eps)), (float)(1. / m.W));
}

// `n` partial results `stride` apart, joined by one warp; the result is lane 0's
__device__ __forceinline__ Moments64 join_parts(const float4 *p, int n, long long stride) {
    const int lane = threadIdx.x & 31;
    Moments64 m{0., 0., 0.};
    for (int i = lane; i < n; i += 32) {
        const Moments64 b = widen(__ldcg(p + i * stride));
        if (m.W == 0.) m = b;
        else join(m, b);
    }
    for (int o = 16; o; o >>= 1) {
        Moments64 b;
        b.W = __shfl_down_sync(0xffffffffu, m.W, o);
        b.mean = __shfl_down_sync(0xffffffffu, m.mean, o);
        b.M2 = __shfl_down_sync(0xffffffffu, m.M2, o);
        if (m.W == 0.) m = b;
        else join(m, b);
    }
    return m;
}

// ------------------------------------------------------------------------------------------------
// forward: sums of a chunk
// ------------------------------------------------------------------------------------------------
constexpr int kUnroll = 4;

template <typename T> __device__ __forceinline__ void accumulate(const F2 (&v)[kP<T>], const F2 (&c)[kP<T>], F2 (&S1)[kP<T>], F2 (&S2)[kP<T>], const F2 (&w)[kP<T>]) {
#pragma unroll
    for (int p = 0; p < kP<T>; ++p) {
        const F2 d = sub2(v[p], c[p]), wd = mul2(d, w[p]);
        S1[p] = add2(S1[p], wd);
        S2[p] = fma2(wd, d, S2[p]);
    }
}
// sums about c + delta from those about c
__device__ __forceinline__ void recentre(F2 W, F2 delta, F2 &S1, F2 &S2) {
    const F2 t = mul2(W, delta);
    S2 = sub2(S2, mul2(delta, sub2(add2(S1, S1), t)));
    S1 = sub2(S1, t);
}

template <typename T>
__device__ void chunk_moments(const GnArgs &a, const Chunk &k, float *red, Moments *acc) {
    constexpr int V = kV<T>, P = kP<T>;
    const T *x = reinterpret_cast<const T *>(a.x) + k.base;
    const uint4 *xv = reinterpret_cast<const uint4 *>(x + k.head);
    for (int g = threadIdx.x; g < a.gu; g += kThreads) acc[g] = {0.f, 0.f, 0.f, 0.f};
    for (int win = 0; win < a.windows; ++win) {
        const Share s = make_share<T>(a, k, win);
        F2 c[P], S1[P], S2[P], dW[P];
        float W = 0.f;
#pragma unroll
        for (int p = 0; p < P; ++p) c[p] = S1[p] = S2[p] = dW[p] = f2(0.f);
        if (s.count) {
            Rows r = make_rows<T>(a, k, s, 0);
            for (int j = 0; j < s.count; j += kUnroll) {
                uint4 raw[kUnroll];
#pragma unroll
                for (int u = 0; u < kUnroll; ++u)
                    if (j + u < s.count) raw[u] = __ldg(xv + s.first + (long long)(j + u) * s.step);
                if (j == 0) {
                    // of the first round, the vector that counts most: a value at the pole, far out, is then no centre for rows of a hundred times its weight
                    if (a.lat && 2 * r.row < a.nlat) {
#pragma unroll
                        for (int u = 0; u < kUnroll; ++u)
                            if (u < s.count) unpack(raw[u], c, T());
                    } else {
                        unpack(raw[0], c, T());
                    }
                }
#pragma unroll
                for (int u = 0; u < kUnroll; ++u) {
                    if (j + u >= s.count) break;
                    F2 v[P];
                    unpack(raw[u], v, T());
                    float w = 1.f;
                    if (a.lat) {
                        w = __ldg(a.lat + r.row);
                        if (r.col + r.over >= a.nlon) {
                            float ws[V];
                            mixed_weights<T>(a.lat, a.nlon, a.cu, s.ch0, r.row, r.col, ws);
                            F2 wp[P];
#pragma unroll
                            for (int p = 0; p < P; ++p) {
                                wp[p] = f2(ws[2 * p], ws[2 * p + 1]);
                                dW[p] = add2(dW[p], sub2(wp[p], f2(w)));
                            }
                            accumulate<T>(v, c, S1, S2, wp);
                            W += w;
                            advance(a, r);
                            continue;
                        }
                        advance(a, r);
                    }
                    F2 wp[P];
#pragma unroll
                    for (int p = 0; p < P; ++p) wp[p] = f2(w);
                    accumulate<T>(v, c, S1, S2, wp);
                    W += w;
                }
                const int round = j / kUnroll;
                if ((round & (round + 1)) == 0) {
                    const F2 inv = f2(__fdividef(1.f, W));
#pragma unroll
                    for (int p = 0; p < P; ++p) {
                        const F2 to = fma2(S1[p], inv, c[p]), delta = sub2(to, c[p]);
                        recentre(add2(f2(W), dW[p]), delta, S1[p], S2[p]);
                        c[p] = to;
                    }
                }
            }
        }
        // all threads of a column: about the centre of its first thread, then added in a tree
        __syncthreads();  // (the last window's readers are done)
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const float2 v = split(c[p]);
            if (s.rep == 0) {
                red[(2 * p) * kThreads + threadIdx.x] = v.x;
                red[(2 * p + 1) * kThreads + threadIdx.x] = v.y;
            }
        }
        __syncthreads();
        F2 c0[P];
#pragma unroll
        for (int p = 0; p < P; ++p) {
            c0[p] = f2(red[(2 * p) * kThreads + s.col], red[(2 * p + 1) * kThreads + s.col]);
            dW[p] = add2(dW[p], f2(W));
            if (s.count) recentre(dW[p], sub2(c0[p], c[p]), S1[p], S2[p]);
        }
        __syncthreads();
        for (int n = a.reps; n > 1;) {
            const int h = (n + 1) / 2;
            if (s.rep >= h && s.rep < n) {
#pragma unroll
                for (int p = 0; p < P; ++p) {
                    const float2 w = split(dW[p]), u = split(S1[p]), q = split(S2[p]);
                    const int t = (s.rep - h) * a.win_cols + s.col;
                    red[(6 * p) * kThreads + t] = w.x;
                    red[(6 * p + 1) * kThreads + t] = w.y;
                    red[(6 * p + 2) * kThreads + t] = u.x;
                    red[(6 * p + 3) * kThreads + t] = u.y;
                    red[(6 * p + 4) * kThreads + t] = q.x;
                    red[(6 * p + 5) * kThreads + t] = q.y;
                }
            }
            __syncthreads();
            if (s.rep < n - h) {
                const int t = threadIdx.x;
#pragma unroll
                for (int p = 0; p < P; ++p) {
                    dW[p] = add2(dW[p], f2(red[(6 * p) * kThreads + t], red[(6 * p + 1) * kThreads + t]));
                    S1[p] = add2(S1[p], f2(red[(6 * p + 2) * kThreads + t], red[(6 * p + 3) * kThreads + t]));
                    S2[p] = add2(S2[p], f2(red[(6 * p + 4) * kThreads + t], red[(6 * p + 5) * kThreads + t]));
                }
            }
            __syncthreads();
            n = h;
        }
        // slots -> moments, in memory as [slot] of the window
        Moments *slot = reinterpret_cast<Moments *>(red);
        if (s.rep == 0 && s.col < a.win_cols) {
#pragma unroll
            for (int p = 0; p < P; ++p) {
                const float2 w = split(dW[p]), u = split(S1[p]), q = split(S2[p]), cc = split(c0[p]);
                const float m0 = w.x > 0.f ? u.x / w.x : 0.f, m1 = w.y > 0.f ? u.y / w.y : 0.f;
                slot[s.col * V + 2 * p] = {w.x, cc.x, m0, fmaxf(fmaf(-u.x, m0, q.x), q.x * 0.f)};
                slot[s.col * V + 2 * p + 1] = {w.y, cc.y, m1, fmaxf(fmaf(-u.y, m1, q.y), q.y * 0.f)};
            }
        }
        __syncthreads();
        // groups: L lanes a group go through its channels' slots in this window
        const int period = a.cols * V, dup = period / a.cu, n = a.cgu * dup;
        int L = 1;
        while (L < 32 && L < n) L *= 2;
        const int sub = threadIdx.x % L, lo = win * a.win_cols * V, hi = min(lo + a.win_cols * V, period);
        for (int g0 = 0; g0 < a.gu; g0 += kThreads / L) {
            const int g = g0 + (int)threadIdx.x / L;
            Moments m{0.f, 0.f, 0.f, 0.f};
            if (g < a.gu)
                for (int i = sub; i < n; i += L) {
                    const int ch = g * a.cgu + i / dup;
                    int e = (ch - k.head % a.cu + a.cu) % a.cu + (i % dup) * a.cu;  // value of the period that has this channel
                    if (e >= lo && e < hi) join(m, slot[e - lo]);
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
            }
        }
    }
    __syncthreads();
    float4 *out = a.part + ((long long)k.unit * a.chunks + k.chunk) * a.gu;
    for (int g = threadIdx.x; g < a.gu; g += kThreads) out[g] = make_float4(acc[g].W, acc[g].K, acc[g].m, acc[g].M2);
    __syncthreads();
}

// Statistics of the group a plane belongs to, joined by every CTA that needs them (the same order everywhere): a second
// wait for the whole grid would cost more.
__device__ __forceinline__ float4 plane_stats(const GnArgs &a, const Chunk &k, float4 *shared) {
    const int g = (k.unit % a.C) / a.cg, first = k.b * a.C + g * a.cg;
    if (threadIdx.x < 32) {
        const Moments64 m = join_parts(a.part + (long long)first * a.chunks, a.cg * a.chunks, 1);
        if (threadIdx.x == 0) {
            *shared = finished(a, m);
            if (k.unit == first && k.chunk == 0) a.stats[k.b * a.G + g] = *shared;
        }
    }
    __syncthreads();
    const float4 st = *shared;
    __syncthreads();
    return st;
}

template <typename T, int ACT>
__device__ void chunk_apply(const GnArgs &a, const Chunk &k, float4 *shared) {
    constexpr int V = kV<T>, P = kP<T>;
    const T *x = reinterpret_cast<const T *>(a.x) + k.base;
    T *y = reinterpret_cast<T *>(a.out) + k.base;
    float4 pst = make_float4(0.f, 0.f, 0.f, 0.f);
    if (!a.cl) pst = plane_stats(a, k, shared);
    auto params = [&](int ch, float &m, float &sc, float &sh) {
        const int c = a.cl ? ch : k.unit % a.C;
        const float4 st = a.cl ? __ldcg(a.stats + k.b * a.G + ch / a.cg) : pst;
        sc = st.z * load_param(a.weight, a.pdtype, c, 1.f);
        m = st.x;
        sh = fmaf(-st.y, sc, load_param(a.bias, a.pdtype, c, 0.f));
    };
    const uint4 *xv = reinterpret_cast<const uint4 *>(x + k.head);
    T *yh = y + k.head;
    const bool aligned = ((uintptr_t)yh & 15) == 0;
    for (int win = 0; win < a.windows; ++win) {
        const Share s = make_share<T>(a, k, win);
        if (!s.count) continue;
        F2 m[P], sc[P], sh[P];
        int ch = s.ch0;
#pragma unroll
        for (int p = 0; p < P; ++p) {
            float v[2][3];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                params(ch, v[h][0], v[h][1], v[h][2]);
                if (++ch >= a.cu) ch = 0;
            }
            m[p] = f2(v[0][0], v[1][0]);
            sc[p] = f2(v[0][1], v[1][1]);
            sh[p] = f2(v[0][2], v[1][2]);
        }
        // from the end: what the sums have read last is nearest
        for (int j = s.count - 1; j >= 0; j -= kUnroll) {
            uint4 raw[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u)
                if (j - u >= 0) raw[u] = __ldg(xv + s.first + (long long)(j - u) * s.step);
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                if (j - u < 0) break;
                F2 v[P];
                unpack(raw[u], v, T());
#pragma unroll
                for (int p = 0; p < P; ++p) v[p] = act_value<ACT>(fma2(sub2(v[p], m[p]), sc[p], sh[p]));
                const long long at = s.first + (long long)(j - u) * s.step;
                if (aligned) reinterpret_cast<uint4 *>(yh)[at] = pack(v, T());
                else
#pragma unroll
                    for (int p = 0; p < P; ++p) {
                        const float2 w = split(v[p]);
                        store_f(yh + at * V + 2 * p, w.x);
                        store_f(yh + at * V + 2 * p + 1, w.y);
                    }
            }
        }
    }
    if ((int)threadIdx.x < 2 * V) {
        const int e = ragged<T>(k, threadIdx.x);
        if (e >= 0) {
            float m, sc, sh;
            params(e % a.cu, m, sc, sh);
            store_f(y + e, split(act_value<ACT>(f2(fmaf(to_f(x[e]) - m, sc, sh)))).x);
        }
    }
}

__device__ __forceinline__ int batch_tasks(const GnArgs &a, int batch) { return min(a.batch_units, a.units - batch * a.batch_units) * a.chunks; }

template <typename T, int ACT>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) gn_forward_kernel(const GnArgs a) {
    extern __shared__ Moments acc[];
    __shared__ __align__(16) float red[8 * kP<T> * kThreads];  // (a window's moments: kThreads columns of V slots of 16 bytes)
    __shared__ float4 shared;
    cg::grid_group grid = cg::this_grid();
    auto moments = [&](int batch) {
        for (int t = blockIdx.x; t < batch_tasks(a, batch); t += gridDim.x) chunk_moments<T>(a, make_chunk<T>(a, batch * a.batch_units, t, a.x), red, acc);
    };
    moments(0);
    for (int i = 0; i < a.batches; ++i) {
        if (a.sync) grid.sync();
        if (a.cl) {  // one warp a group
            const int lo = i * a.batch_units * a.G, hi = min(lo + a.batch_units * a.G, a.B * a.G);
            for (int t = lo + blockIdx.x * kWarps + (int)(threadIdx.x >> 5); t < hi; t += gridDim.x * kWarps) {
                const Moments64 m = join_parts(a.part + ((long long)(t / a.G) * a.chunks) * a.G + t % a.G, a.chunks, a.G);
                if ((threadIdx.x & 31) == 0) a.stats[t] = finished(a, m);
            }
            grid.sync();
        }
        if (i + 1 < a.batches) moments(i + 1);
        for (int t = blockIdx.x; t < batch_tasks(a, i); t += gridDim.x) chunk_apply<T, ACT>(a, make_chunk<T>(a, i * a.batch_units, t, a.x), &shared);
    }
}

// ------------------------------------------------------------------------------------------------
// backward
// ------------------------------------------------------------------------------------------------
constexpr int kUnrollB = 2;

struct SlotIn {  // what a slot needs to find z, and g from it
    float m, sc, sh, r, lo;
};
__device__ __forceinline__ SlotIn slot_in(const GnArgs &a, const Chunk &k, int ch) {
    const int c = a.cl ? ch : k.unit % a.C;
    const float4 st = __ldcg(a.stats + k.b * a.G + c / a.cg);
    SlotIn s;
    s.m = st.x;
    s.sc = st.z * load_param(a.weight, a.pdtype, c, 1.f);
    s.sh = fmaf(-st.y, s.sc, load_param(a.bias, a.pdtype, c, 0.f));
    s.r = st.z;
    s.lo = st.y;
    return s;
}

template <typename T> __device__ __forceinline__ uint4 load_any(const T *p, bool aligned) {
    if (aligned) return __ldg(reinterpret_cast<const uint4 *>(p));
    uint4 u;
    T *w = reinterpret_cast<T *>(&u);
#pragma unroll
    for (int i = 0; i < kV<T>; ++i) w[i] = p[i];
    return u;
}

template <typename T, int ACT>
__device__ void chunk_sums(const GnArgs &a, const Chunk &k, float *red, float2 *acc) {
    constexpr int V = kV<T>, P = kP<T>;
    const T *x = reinterpret_cast<const T *>(a.x) + k.base, *dy = reinterpret_cast<const T *>(a.dy) + k.base;
    const uint4 *xv = reinterpret_cast<const uint4 *>(x + k.head);
    const T *dh = dy + k.head;
    const bool aligned = ((uintptr_t)dh & 15) == 0;
    __syncthreads();  // (the memory of acc serves as gsum as well)
    for (int c = threadIdx.x; c < a.cu; c += kThreads) acc[c] = make_float2(0.f, 0.f);
    for (int win = 0; win < a.windows; ++win) {
        const Share s = make_share<T>(a, k, win);
        F2 S1[P], S2[P];
#pragma unroll
        for (int p = 0; p < P; ++p) S1[p] = S2[p] = f2(0.f);
        if (s.count) {
            F2 m[P], sc[P], sh[P], r[P], lo[P];
            int ch = s.ch0;
#pragma unroll
            for (int p = 0; p < P; ++p) {
                const SlotIn u = slot_in(a, k, ch);
                if (++ch >= a.cu) ch = 0;
                const SlotIn v = slot_in(a, k, ch);
                if (++ch >= a.cu) ch = 0;
                m[p] = f2(u.m, v.m);
                sc[p] = f2(u.sc, v.sc);
                sh[p] = f2(u.sh, v.sh);
                r[p] = f2(u.r, v.r);
                lo[p] = f2(u.lo, v.lo);
            }
            for (int j = 0; j < s.count; j += kUnrollB) {
                uint4 rx[kUnrollB], rd[kUnrollB];
#pragma unroll
                for (int u = 0; u < kUnrollB; ++u)
                    if (j + u < s.count) {
                        const long long at = s.first + (long long)(j + u) * s.step;
                        rx[u] = __ldg(xv + at);
                        rd[u] = load_any<T>(dh + at * V, aligned);
                    }
#pragma unroll
                for (int u = 0; u < kUnrollB; ++u) {
                    if (j + u >= s.count) break;
                    F2 v[P], d[P];
                    unpack(rx[u], v, T());
                    unpack(rd[u], d, T());
#pragma unroll
                    for (int p = 0; p < P; ++p) {
                        const F2 e = sub2(v[p], m[p]), g = mul2(d[p], act_slope<ACT>(fma2(e, sc[p], sh[p])));
                        S1[p] = add2(S1[p], g);
                        S2[p] = fma2(g, e, S2[p]);
                    }
                }
            }
#pragma unroll
            for (int p = 0; p < P; ++p) S2[p] = mul2(r[p], sub2(S2[p], mul2(lo[p], S1[p])));  // sum g (x - m) -> sum g xh
        }
        __syncthreads();
        for (int n = a.reps; n > 1;) {
            const int h = (n + 1) / 2;
            if (s.rep >= h && s.rep < n) {
#pragma unroll
                for (int p = 0; p < P; ++p) {
                    const float2 u = split(S1[p]), q = split(S2[p]);
                    const int t = (s.rep - h) * a.win_cols + s.col;
                    red[(4 * p) * kThreads + t] = u.x;
                    red[(4 * p + 1) * kThreads + t] = u.y;
                    red[(4 * p + 2) * kThreads + t] = q.x;
                    red[(4 * p + 3) * kThreads + t] = q.y;
                }
            }
            __syncthreads();
            if (s.rep < n - h) {
                const int t = threadIdx.x;
#pragma unroll
                for (int p = 0; p < P; ++p) {
                    S1[p] = add2(S1[p], f2(red[(4 * p) * kThreads + t], red[(4 * p + 1) * kThreads + t]));
                    S2[p] = add2(S2[p], f2(red[(4 * p + 2) * kThreads + t], red[(4 * p + 3) * kThreads + t]));
                }
            }
            __syncthreads();
            n = h;
        }
        float2 *slot = reinterpret_cast<float2 *>(red);
        if (s.rep == 0 && s.col < a.win_cols) {
#pragma unroll
            for (int p = 0; p < P; ++p) {
                const float2 u = split(S1[p]), q = split(S2[p]);
                slot[s.col * V + 2 * p] = make_float2(u.x, q.x);
                slot[s.col * V + 2 * p + 1] = make_float2(u.y, q.y);
            }
        }
        __syncthreads();
        const int period = a.cols * V, lo = win * a.win_cols * V, hi = min(lo + a.win_cols * V, period);
        for (int c = threadIdx.x; c < a.cu; c += kThreads) {
            float2 t = acc[c];
            for (int e = (c - k.head % a.cu + a.cu) % a.cu; e < hi; e += a.cu)
                if (e >= lo) {
                    t.x += slot[e - lo].x;
                    t.y += slot[e - lo].y;
                }
            if (win == 0)
                for (int i = 0; i < 2 * V; ++i) {
                    const int e = ragged<T>(k, i);
                    if (e < 0) break;
                    if (e % a.cu == c) {
                        const SlotIn q = slot_in(a, k, c);
                        const float d = to_f(x[e]) - q.m, g = to_f(dy[e]) * split(act_slope<ACT>(f2(fmaf(d, q.sc, q.sh)))).x;
                        t.x += g;
                        t.y = fmaf(g, q.r * (d - q.lo), t.y);
                    }
                }
            acc[c] = t;
        }
    }
    __syncthreads();
    float2 *out = a.bpart + ((long long)k.unit * a.chunks + k.chunk) * a.cu;
    for (int c = threadIdx.x; c < a.cu; c += kThreads) out[c] = acc[c];
    __syncthreads();
}

__device__ __forceinline__ double2 warp_sum(double2 v) {
    for (int o = 16; o; o >>= 1) {
        v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
        v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
    return v;
}

// (sum h, sum h xh) of the groups of a chunk's unit
__device__ void group_sums(const GnArgs &a, const Chunk &k, float2 *gsum) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    __syncthreads();
    if (a.cl) {
        for (int g = warp; g < a.G; g += kWarps) {
            double2 t = make_double2(0., 0.);
            for (int i = lane; i < a.cg; i += 32) {
                const int c = g * a.cg + i;
                const double w = load_param(a.weight, a.pdtype, c, 1.f);
                const double2 v = __ldcg(a.csum + (long long)k.b * a.C + c);
                t.x += w * v.x;
                t.y += w * v.y;
            }
            t = warp_sum(t);
            if (lane == 0) gsum[g] = make_float2((float)t.x, (float)t.y);
        }
    } else if (warp == 0) {
        const int first = (k.unit % a.C) / a.cg * a.cg;  // first channel of the group
        const float2 *p = a.bpart + ((long long)k.b * a.C + first) * a.chunks;
        double2 t = make_double2(0., 0.);
        for (int i = lane; i < a.cg * a.chunks; i += 32) {
            const double w = load_param(a.weight, a.pdtype, first + i / a.chunks, 1.f);
            const float2 v = __ldcg(p + i);
            t.x += w * v.x;
            t.y += w * v.y;
        }
        t = warp_sum(t);
        if (lane == 0) gsum[0] = make_float2((float)t.x, (float)t.y);
    }
    __syncthreads();
}

// dx = sc g - a (alpha + (x - m) beta),  alpha = r (sum h - lo r sum h xh) / sum a,  beta = r^2 sum h xh / sum a
template <typename T, int ACT>
__device__ void chunk_dx(const GnArgs &a, const Chunk &k, float2 *gsum) {
    constexpr int V = kV<T>, P = kP<T>;
    const T *x = reinterpret_cast<const T *>(a.x) + k.base, *dy = reinterpret_cast<const T *>(a.dy) + k.base;
    T *dx = reinterpret_cast<T *>(a.out) + k.base;
    group_sums(a, k, gsum);
    auto params = [&](int ch, SlotIn &s, float &alpha, float &beta) {
        s = slot_in(a, k, ch);
        const int c = a.cl ? ch : k.unit % a.C;
        const float inv = __ldcg(a.stats + k.b * a.G + c / a.cg).w;
        const float2 g = gsum[a.cl ? ch / a.cg : 0];
        beta = s.r * s.r * g.y * inv;
        alpha = s.r * (g.x - s.lo * s.r * g.y) * inv;
    };
    const uint4 *xv = reinterpret_cast<const uint4 *>(x + k.head);
    const T *dh = dy + k.head;
    T *oh = dx + k.head;
    const bool aligned = ((uintptr_t)dh & 15) == 0, out_aligned = ((uintptr_t)oh & 15) == 0;
    for (int win = 0; win < a.windows; ++win) {
        const Share s = make_share<T>(a, k, win);
        if (!s.count) continue;
        F2 m[P], sc[P], sh[P], al[P], be[P];
        int ch = s.ch0;
#pragma unroll
        for (int p = 0; p < P; ++p) {
            SlotIn u, v;
            float a0, b0, a1, b1;
            params(ch, u, a0, b0);
            if (++ch >= a.cu) ch = 0;
            params(ch, v, a1, b1);
            if (++ch >= a.cu) ch = 0;
            m[p] = f2(u.m, v.m);
            sc[p] = f2(u.sc, v.sc);
            sh[p] = f2(u.sh, v.sh);
            al[p] = f2(-a0, -a1);
            be[p] = f2(-b0, -b1);
        }
        Rows r = make_rows<T>(a, k, s, s.count - 1);
        for (int j = s.count - 1; j >= 0; j -= kUnrollB) {
            uint4 rx[kUnrollB], rd[kUnrollB];
#pragma unroll
            for (int u = 0; u < kUnrollB; ++u)
                if (j - u >= 0) {
                    const long long at = s.first + (long long)(j - u) * s.step;
                    rx[u] = __ldg(xv + at);
                    rd[u] = load_any<T>(dh + at * V, aligned);
                }
#pragma unroll
            for (int u = 0; u < kUnrollB; ++u) {
                if (j - u < 0) break;
                F2 v[P], d[P], w[P];
                unpack(rx[u], v, T());
                unpack(rd[u], d, T());
                const float w0 = a.lat ? __ldg(a.lat + r.row) : 1.f;
#pragma unroll
                for (int p = 0; p < P; ++p) w[p] = f2(w0);
                if (a.lat && r.col + r.over >= a.nlon) {
                    float ws[V];
                    mixed_weights<T>(a.lat, a.nlon, a.cu, s.ch0, r.row, r.col, ws);
#pragma unroll
                    for (int p = 0; p < P; ++p) w[p] = f2(ws[2 * p], ws[2 * p + 1]);
                }
                retreat(a, r);
#pragma unroll
                for (int p = 0; p < P; ++p) {
                    const F2 e = sub2(v[p], m[p]), g = mul2(d[p], act_slope<ACT>(fma2(e, sc[p], sh[p])));
                    v[p] = fma2(w[p], fma2(e, be[p], al[p]), mul2(sc[p], g));
                }
                const long long at = s.first + (long long)(j - u) * s.step;
                if (out_aligned) reinterpret_cast<uint4 *>(oh)[at] = pack(v, T());
                else
#pragma unroll
                    for (int p = 0; p < P; ++p) {
                        const float2 o = split(v[p]);
                        store_f(oh + at * V + 2 * p, o.x);
                        store_f(oh + at * V + 2 * p + 1, o.y);
                    }
            }
        }
    }
    if ((int)threadIdx.x < 2 * V) {
        const int e = ragged<T>(k, threadIdx.x);
        if (e >= 0) {
            SlotIn s;
            float alpha, beta;
            params(e % a.cu, s, alpha, beta);
            const float d = to_f(x[e]) - s.m, g = to_f(dy[e]) * split(act_slope<ACT>(f2(fmaf(d, s.sc, s.sh)))).x;
            store_f(dx + e, fmaf(-weight_at(a, k, e), fmaf(d, beta, alpha), s.sc * g));
        }
    }
}

template <typename T, int ACT>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) gn_backward_kernel(const GnArgs a) {
    extern __shared__ float2 bacc[];
    __shared__ __align__(16) float red[4 * kP<T> * kThreads];
    cg::grid_group grid = cg::this_grid();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    auto sums = [&](int batch) {
        for (int t = blockIdx.x; t < batch_tasks(a, batch); t += gridDim.x) chunk_sums<T, ACT>(a, make_chunk<T>(a, batch * a.batch_units, t, a.x), red, bacc);
    };
    sums(0);
    for (int i = 0; i < a.batches; ++i) {
        grid.sync();
        if (a.cl) {  // 32 channels of a sample: a lane each, the chunks dealt to the warps
            const int blocks = (a.C + 31) / 32, lo = i * a.batch_units, hi = min(lo + a.batch_units, a.B);
            double2 *wsum = reinterpret_cast<double2 *>(red);
            for (int t = blockIdx.x; t < (hi - lo) * blocks; t += gridDim.x) {
                const int b = lo + t / blocks, c = (t % blocks) * 32 + lane;
                double2 v = make_double2(0., 0.);
                if (c < a.C)
                    for (int n = warp; n < a.chunks; n += kWarps) {
                        const float2 p = __ldcg(a.bpart + ((long long)b * a.chunks + n) * a.C + c);
                        v.x += p.x;
                        v.y += p.y;
                    }
                __syncthreads();
                wsum[threadIdx.x] = v;
                __syncthreads();
                if (warp == 0 && c < a.C) {
                    for (int w = 1; w < kWarps; ++w) {
                        v.x += wsum[w * 32 + lane].x;
                        v.y += wsum[w * 32 + lane].y;
                    }
                    a.csum[(long long)b * a.C + c] = v;
                }
                __syncthreads();
            }
            grid.sync();
        }
        if (i + 1 < a.batches) sums(i + 1);
        if (a.out)
            for (int t = blockIdx.x; t < batch_tasks(a, i); t += gridDim.x) chunk_dx<T, ACT>(a, make_chunk<T>(a, i * a.batch_units, t, a.x), bacc);
    }
    // the parameters' gradients: one warp a channel, over all samples (every sum of the last batch was complete before its dx)
    if (a.dweight || a.dbias)
        for (int c = blockIdx.x * kWarps + warp; c < a.C; c += gridDim.x * kWarps) {
            double2 v = make_double2(0., 0.);
            if (a.cl) {
                for (int b = lane; b < a.B; b += 32) {
                    const double2 p = __ldcg(a.csum + (long long)b * a.C + c);
                    v.x += p.x;
                    v.y += p.y;
                }
            } else {
                for (long long n = lane; n < (long long)a.B * a.chunks; n += 32) {
                    const long long b = n / a.chunks;
                    const float2 p = __ldcg(a.bpart + (b * a.C + c) * a.chunks + (n - b * a.chunks));
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
}

// ------------------------------------------------------------------------------------------------
// host
// ------------------------------------------------------------------------------------------------
constexpr size_t kStaticSmem = 33 << 10;  // at most, of either kernel
constexpr int kMaxWaves = 4;              // chunks a CTA takes one after the other, at most, where a unit is cut
constexpr int kMaxChannels = 8192;        // what a CTA keeps per channel or group has to fit into its shared memory
constexpr long long kResident = 48 << 20; // bytes that a second read may be expected to find in L2 (126 MB, the written values among them)
constexpr long long kBatch = 24 << 20;    // bytes of a batch where the whole is more

// How much of the last wave is filled.
double filled(long long tasks, int grid) { return (double)tasks / (double)((tasks + grid - 1) / grid * grid); }

int sm_count() {
    int dev = 0, n = 148;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) n = 148;
    cudaGetLastError();
    return n;
}

int value_bytes(int dtype) { return dtype == SHTB200_F32 ? 4 : 2; }
size_t up256(size_t b) { return (b + 255) / 256 * 256; }

struct Launch {
    GnArgs a{};
    int grid = 0;
    long long max_chunks = 0;  // of a unit, whatever the number of SMs the grid is limited to
    size_t smem = 0;
};

Launch geometry(const GroupNormDesc &d, bool backward, int sms, int sms_used) {
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
    a.units = a.cl ? a.B : a.B * a.C;
    // batches: whole groups of planes, or whole samples
    const int least_units = a.cl ? 1 : a.cg;
    const long long unit_bytes = a.hw * a.cu * value_bytes(d.dtype) * (backward ? 2 : 1);
    a.batch_units = a.units;
    if (unit_bytes * a.units > kResident) {
        const long long fit = std::max<long long>(1, kBatch / (unit_bytes * least_units));
        a.batch_units = (int)std::min<long long>(a.units, fit * least_units);
        const int n = ceil_div(a.units, a.batch_units);  // evenly
        a.batch_units = ceil_div(ceil_div(a.units, n), least_units) * least_units;
    }
    a.batches = ceil_div(a.units, a.batch_units);
    // chunks
    const int full = sms * kCtasPerSm, grid = std::max(1, sms_used * kCtasPerSm);
    const long long values = a.hw * a.cu, most = std::max<long long>(1, std::min<long long>(a.hw, values / (kThreads * V)));
    l.max_chunks = std::min<long long>(most, std::max(1, kMaxWaves * full / a.batch_units));
    long long chunks = 1;
    double best = 0.;
    for (int w = 1; w <= kMaxWaves; ++w) {
        const long long c = std::min<long long>(most, std::max(1, w * grid / a.batch_units));
        const double f = filled(c * a.batch_units, grid);
        if (f > best + 0.03) {
            best = f;
            chunks = c;
        }
    }
    a.chunk_px = (int)((a.hw + chunks - 1) / chunks);
    if (a.chunk_px >= 256) a.chunk_px = (a.chunk_px + 31) / 32 * 32;  // (chunks of an aligned field begin aligned)
    a.chunks = (int)((a.hw + a.chunk_px - 1) / a.chunk_px);
    a.sync = !(!a.cl && a.chunks == 1 && a.cg == 1);
    // columns
    a.cols = a.cu / std::gcd(a.cu, V);
    a.windows = ceil_div(a.cols, kThreads);
    a.win_cols = ceil_div(a.cols, a.windows);
    a.reps = kThreads / a.win_cols;
    const long long step_px = (long long)a.reps * a.cols * V / a.cu;
    a.step_rows = (int)(step_px / a.nlon);
    a.step_cols = (int)(step_px % a.nlon);
    l.smem = backward ? sizeof(float2) * std::max(a.cu, a.gu) : sizeof(Moments) * a.gu;
    const long long tasks = (long long)a.batch_units * a.chunks;
    const int per_sm = std::max<int>(1, std::min<int>(kCtasPerSm, (int)((224 << 10) / (l.smem + kStaticSmem + 1024))));
    l.grid = (int)std::max<long long>(1, std::min<long long>(tasks, sms_used * per_sm));
    return l;
}

struct GnWs {
    size_t part = 0, csum = 0;
    size_t total() const { return part + csum; }
};
GnWs ws_sizes(const GroupNormDesc &d, const Launch &l, bool backward) {
    GnWs w;
    const size_t parts = (size_t)l.a.units * (size_t)l.max_chunks;
    w.part = up256(backward ? parts * l.a.cu * sizeof(float2) : parts * l.a.gu * sizeof(float4));
    if (backward && l.a.cl) w.csum = up256((size_t)d.batch * d.channels * sizeof(double2));
    return w;
}

int launch(const void *kernel, const Launch &l, cudaStream_t st) {
    if (l.smem + kStaticSmem > (48 << 10)) SHT_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)l.smem));
    void *args[] = {const_cast<GnArgs *>(&l.a)};
    SHT_CUDA_CHECK(cudaLaunchCooperativeKernel(kernel, dim3(l.grid), dim3(kThreads), args, l.smem, st));
    return SHTB200_OK;
}

template <typename T> const void *forward_kernel(int act) {
    switch (act) {
        case SHTB200_ACT_RELU: return (const void *)gn_forward_kernel<T, SHTB200_ACT_RELU>;
        case SHTB200_ACT_SILU: return (const void *)gn_forward_kernel<T, SHTB200_ACT_SILU>;
        case SHTB200_ACT_GELU: return (const void *)gn_forward_kernel<T, SHTB200_ACT_GELU>;
        default: return (const void *)gn_forward_kernel<T, SHTB200_ACT_NONE>;
    }
}
template <typename T> const void *backward_kernel(int act) {
    switch (act) {
        case SHTB200_ACT_RELU: return (const void *)gn_backward_kernel<T, SHTB200_ACT_RELU>;
        case SHTB200_ACT_SILU: return (const void *)gn_backward_kernel<T, SHTB200_ACT_SILU>;
        case SHTB200_ACT_GELU: return (const void *)gn_backward_kernel<T, SHTB200_ACT_GELU>;
        default: return (const void *)gn_backward_kernel<T, SHTB200_ACT_NONE>;
    }
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

int check_call(const GroupNormDesc *d, const Launch &l, bool backward, const void *ws, size_t ws_bytes, const void *stats) {
    const GnWs w = ws_sizes(*d, l, backward);
    if (!ws || ws_bytes < w.total()) return fail(SHTB200_EWORKSPACE, "workspace too small: need " + std::to_string(w.total()) + " bytes");
    if (((uintptr_t)ws & 255) != 0) return fail(SHTB200_EINVAL, "workspace must be 256-byte aligned");
    if (((uintptr_t)stats & 15) != 0) return fail(SHTB200_EINVAL, "the statistics must be 16-byte aligned");
    if ((long long)l.a.chunk_px * l.a.cu > 0x7fffffff - 64) return fail(SHTB200_EINVAL, "group norm shape too large");
    return SHTB200_OK;
}

}  // namespace

size_t group_norm_workspace(const GroupNormDesc *d, bool backward) {
    if (check_desc(d)) return 0;
    const int sms = sm_count();
    return d->batch == 0 ? 256 : std::max<size_t>(ws_sizes(*d, geometry(*d, backward, sms, sms), backward).total(), 256);
}

int group_norm_forward(const GroupNormDesc *d, const void *x, const float *lat, const void *weight, const void *bias, void *y, void *stats, void *ws, size_t ws_bytes,
                       cudaStream_t st) {
    int rc = check_desc(d);
    if (rc) return rc;
    if (d->batch == 0) return SHTB200_OK;
    if (!x || !y || !stats) return fail(SHTB200_EINVAL, "null pointer");
    const int sms = sm_count();
    Launch l = geometry(*d, false, sms, effective_sms(sms));
    if ((rc = check_call(d, l, false, ws, ws_bytes, stats))) return rc;
    GnArgs &a = l.a;
    a.x = x;
    a.out = y;
    a.lat = lat;
    a.weight = weight;
    a.bias = bias;
    a.stats = reinterpret_cast<float4 *>(stats);
    a.part = reinterpret_cast<float4 *>(ws);
    return launch(d->dtype == SHTB200_F32    ? forward_kernel<float>(d->activation)
                  : d->dtype == SHTB200_BF16 ? forward_kernel<__nv_bfloat16>(d->activation)
                                             : forward_kernel<__half>(d->activation),
                  l, st);
}

int group_norm_backward(const GroupNormDesc *d, const void *dy, const void *x, const float *lat, const void *weight, const void *bias, const void *stats, void *dx, void *dweight,
                        void *dbias, void *ws, size_t ws_bytes, cudaStream_t st) {
    int rc = check_desc(d);
    if (rc) return rc;
    if (d->batch == 0) return fail(SHTB200_EINVAL, "an empty batch has no gradient to compute");
    if (!x || !dy || !stats) return fail(SHTB200_EINVAL, "null pointer");
    const int sms = sm_count();
    Launch l = geometry(*d, true, sms, effective_sms(sms));
    if ((rc = check_call(d, l, true, ws, ws_bytes, stats))) return rc;
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
    a.csum = reinterpret_cast<double2 *>(reinterpret_cast<char *>(ws) + ws_sizes(*d, l, true).part);
    return launch(d->dtype == SHTB200_F32    ? backward_kernel<float>(d->activation)
                  : d->dtype == SHTB200_BF16 ? backward_kernel<__nv_bfloat16>(d->activation)
                                             : backward_kernel<__half>(d->activation),
                  l, st);
}

}  // namespace shtb200
