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
// pixels.  A chunk is read as one flat stream of 16-byte vectors: with C' interleaved channels (C, or 1 for planes) and V values a vector, a thread
// that steps by a multiple of lcm(C', V) values meets the same channels in every vector ("slots"), whatever C' is, and keeps their sums and
// parameters in registers.  The stream comes through a ring of tiles in shared memory, filled by bulk asynchronous copies: enough is in
// flight whatever the registers allow, and what the ring holds when the sums are done is normalised without being read again.  Two orders:
//   - one batch: sums forward, result backward from the last tile, so that the ring and then L2 serve the second pass first;
//   - batches of whole groups of which the ring holds two: every value is read from memory once, the sums of a batch are taken while the one
//     before is normalised.
//
// Sums for the variance are taken about a centre c per slot, (W, c, S1, S2) = (sum a, c, sum a (x - c), sum a (x - c)^2).  c begins as a value
// of the field and is moved to the mean so far after 1, 2, 4, 8, ... rounds; fields whose level is far above their spread (pressures) or
// that have a value far out lose nothing.  Chunks are joined in float64 as (W, K, mean - K, M2).

#include "common.cuh"
#include "tc_ptx.cuh"

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
constexpr int kMaxCols = 128;       // columns of vectors a CTA covers at a time
constexpr int kMaxStages = 30;      // of the ring
constexpr int kTileVectors = 4;     // vectors a thread has in a tile (x and dy together): 16 KiB
constexpr int kCounterPitch = 8;    // (counters of different teams do not share a sector)

struct GnArgs {
    const void *x, *dy;
    void *out;
    const float *lat;  // nullptr: 1 everywhere
    const void *weight, *bias;
    void *dweight, *dbias;
    float4 *stats;     // (B, G): mean, its low part, r, 1 / sum a
    float4 *part;      // forward: (unit, chunk, group of the unit): (W, K, mean - K, M2)
    float2 *bpart;     // backward: (unit, chunk, channel of the unit): (sum g, sum g xh)
    double2 *csum;     // backward, channels last, not direct: (B, C): the same over all chunks
    unsigned *arrived; // a counter for every team
    long long hw;
    int B, C, G, cg, nlat, nlon, cl, pdtype;
    float eps;
    int cu, gu, cgu;   // channels, groups of a unit, channels of a group inside a unit: (C, G, cg) channels last, (1, 1, 1) for planes
    int jobs, job_units;          // a sample; a group of planes
    int teams, team;              // teams of `team` CTAs
    int chunks, chunk_px;         // of a unit
    int tasks;                    // of a job: job_units * chunks
    int cols, dup;                // lcm(cu, V) / V: vectors after which the channels repeat; how often each occurs in them
    int win_cols, windows, reps;  // columns a CTA covers at a time, how many windows that takes, vectors of a column it takes side by side
    int step_rows, step_cols;     // reps periods further in pixels, as rows and columns of the grid
    int lanes;                    // that join the slots of a group
    int stages, tile_bytes;       // of the ring; one tensor's part of a tile
    int direct;        // the partial results of a group are joined by every CTA that needs them; else once, before a second wait for the team
};

// A chunk of a unit: n values from `base` on; `head` of them lie before the first aligned vector, then `vecs` vectors, then the tail.
struct Chunk {
    int unit, chunk, b, c;  // (c: the channel of a plane)
    long long base;  // first value
    int px0;         // its pixel
    int n, head, vecs;
    int tiles;       // of a window
};
template <typename T, int U> __device__ __forceinline__ Chunk make_chunk(const GnArgs &a, int job, int task) {
    Chunk k;
    const int u = a.chunks == 1 ? task : (int)((unsigned)task / (unsigned)a.chunks);
    k.unit = job * a.job_units + u;
    k.chunk = task - u * a.chunks;
    k.b = a.cl ? k.unit : (int)((unsigned)k.unit / (unsigned)a.C);
    k.c = a.cl ? 0 : k.unit - k.b * a.C;
    k.px0 = k.chunk * a.chunk_px;
    const int px = (int)min((long long)a.chunk_px, a.hw - k.px0);
    k.base = ((long long)k.unit * a.hw + k.px0) * a.cu;
    k.n = px * a.cu;
    const unsigned mis = (unsigned)((uintptr_t)(reinterpret_cast<const T *>(a.x) + k.base) & 15u);
    k.head = min(k.n, (int)(((16u - mis) & 15u) / (unsigned)sizeof(T)));
    k.vecs = (k.n - k.head) / kV<T>;
    const unsigned periods = a.cols == 1 ? (unsigned)k.vecs : (unsigned)(k.vecs + a.cols - 1) / (unsigned)a.cols, per = (unsigned)(a.reps * U);
    k.tiles = (int)((periods + per - 1) / per);
    return k;
}

// A thread's share of a window of a chunk: vectors first, first + step, ... (count of them); the channel (of the unit) of slot 0.
struct Share {
    int first, step, count, ch0, rep, col;
};
template <typename T> __device__ __forceinline__ Share make_share(const GnArgs &a, const Chunk &k, int window) {
    Share s;
    s.rep = a.win_cols == 1 ? (int)threadIdx.x : (int)(threadIdx.x / (unsigned)a.win_cols);
    s.col = (int)threadIdx.x - s.rep * a.win_cols;
    const int c = window * a.win_cols + s.col;
    s.first = c + s.rep * a.cols;
    s.step = a.reps * a.cols;
    s.count = (s.rep < a.reps && c < a.cols && s.first < k.vecs) ? (int)((unsigned)(k.vecs - s.first + s.step - 1) / (unsigned)s.step) : 0;
    s.ch0 = a.cu == 1 ? 0 : (int)((unsigned)(c * kV<T> + k.head) % (unsigned)a.cu);
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
__device__ __forceinline__ void retreat(const GnArgs &a, Rows &r, int tiles_vectors) {
    for (int u = 0; u < tiles_vectors; ++u) {
        r.row -= a.step_rows;
        r.col -= a.step_cols;
        if (r.col < 0) {
            r.col += a.nlon;
            --r.row;
        }
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

// Weight, bias and group (of the unit) of the V slots from channel ch on.  The loads go out together.
template <int V> __device__ __forceinline__ void slot_params(const GnArgs &a, const Chunk &k, int ch, float (&w)[V], float (&b)[V], int (&g)[V]) {
    if (a.cu == 1) {
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
// the ring of tiles
// ------------------------------------------------------------------------------------------------
// Thread 0 starts the copies.  The tiles of a job are numbered in the order of the sums: the CTA's chunks, in them windows, tiles of a window.  Tile n of
// a job lies in stage n % stages, counted from the other end in every second job: the second pass goes backward, so that stages become free
// in that order for the next job.
//   The sums let go of tile n as long as a tile n + stages follows, which then takes its stage, and hold the last `stages` tiles; the second
// pass begins with these, and puts tile n - stages where tile n was, or the first tiles of the next job.
// A wait that runs out (a copy that does not come) makes the tile read as NaN, and so every result that depends on it, and nothing more
// is loaded.
template <typename T, int U> struct Position {  // of a tile
    int job, task, window, tile;
    Chunk k;
    __device__ __forceinline__ bool find(const GnArgs &a, int rank) {  // from `task` on, the first chunk that has tiles
        window = tile = 0;
        for (; task < a.tasks; task += a.team) {
            k = make_chunk<T, U>(a, job, task);
            if (k.tiles) return true;
        }
        return false;
    }
    __device__ __forceinline__ bool start(const GnArgs &a, int j, int rank) {
        job = j;
        task = rank;
        return job < a.jobs && find(a, rank);
    }
    __device__ __forceinline__ bool next(const GnArgs &a, int rank) {
        if (++tile < k.tiles) return true;
        tile = 0;
        if (++window < a.windows) return true;
        task += a.team;
        return find(a, rank);
    }
    __device__ __forceinline__ bool previous(const GnArgs &a) {
        if (--tile >= 0) return true;
        if (--window >= 0) {
            tile = k.tiles - 1;
            return true;
        }
        for (task -= a.team; task >= 0; task -= a.team) {
            k = make_chunk<T, U>(a, job, task);
            if (!k.tiles) continue;
            window = a.windows - 1;
            tile = k.tiles - 1;
            return true;
        }
        return false;
    }
};

constexpr long long kWaitCycles = 200000000LL;  // about a tenth of a second

template <typename T, int U, bool TWO> struct Walk {
    uint32_t data, bars;           // stage s: full barrier at bars + 16 s, empty barrier 8 bytes further
    unsigned full_parity, empty_parity, used;  // a bit a stage (the last two: thread 0's)
    int rank, stages, stage_bytes;
    volatile int *dead;
    Position<T, U> *here, *after;  // thread 0's: the next tile to load of this job and of the next one (in shared memory: registers are short)
    bool more_after;
    bool flip;
    int total;                     // tiles of the job
    int number, stage;             // of the tile at hand
    int due;                       // thread 0: stage to refill, one tile later, when the other warps are done with it too: -1 none
    int due_what;                  // 0 forward, 1 backward, 2 with the next job's

    __device__ __forceinline__ uint32_t full(int s) const { return bars + 16u * s; }
    __device__ __forceinline__ uint32_t empty(int s) const { return bars + 16u * s + 8u; }
    __device__ __forceinline__ void init(const GnArgs &a, unsigned char *mem, unsigned long long *barriers, int *flag, Position<T, U> *positions, int first_job, int rank_) {
        rank = rank_;
        stages = a.stages;
        stage_bytes = a.tile_bytes * (TWO ? 2 : 1);
        data = ptx::smem_u32(mem);
        bars = ptx::smem_u32(barriers);
        full_parity = empty_parity = used = 0;
        dead = flag;
        here = positions;
        after = positions + 1;
        due = -1;
        flip = true;
        more_after = false;
        if ((int)threadIdx.x < stages) {
            ptx::mbar_init(full(threadIdx.x), 1);
            ptx::mbar_init(empty(threadIdx.x), kWarps);
            ptx::fence_barrier_init();
        }
        if (threadIdx.x == 0) *flag = 0;
        __syncthreads();
        if (threadIdx.x == 0) {
            more_after = after->start(a, first_job, rank);
            for (int s = 0; s < stages && more_after; ++s) put(a, s, 2);
        }
    }
    // all threads: the sums of a job begin
    __device__ __forceinline__ void begin(const GnArgs &a, int job, const Chunk &first) {
        flip = !flip;
        total = first.tiles * a.windows;
        for (int t = rank + a.team; t < a.tasks; t += a.team) total += a.windows * make_chunk<T, U>(a, job, t).tiles;
        if (rank >= a.tasks) total = 0;
        number = -1;
        stage = flip ? stages : -1;
        if (threadIdx.x == 0) {
            settle(a);
            Position<T, U> *p = here;
            here = after;
            after = p;
            more_after = after->start(a, job + a.teams, rank);
        }
    }
    // all threads: the second pass of a job begins
    __device__ __forceinline__ void turn(const GnArgs &a) {
        number = total;
        stage = (total - 1) % stages + 1;  // (one beyond the last tile's)
        if (total == 0) stage = 0;
        if (flip) stage = stages - 1 - stage;
        if (threadIdx.x == 0) {
            settle(a);
            if (total > stages) {
                for (int i = 0; i <= stages; ++i) here->previous(a);
            } else {
                for (int n = stages - 1; n >= total && more_after; --n) put(a, flip ? stages - 1 - n : n, 2);  // stages that this job leaves free
            }
        }
    }
    // all threads: no second pass
    __device__ __forceinline__ void skip(const GnArgs &a) {
        if (threadIdx.x == 0) settle(a);
        __syncwarp();
        if ((threadIdx.x & 31) == 0)
            for (int n = max(0, total - stages); n < total; ++n) ptx::mbar_arrive(empty(flip ? stages - 1 - n % stages : n % stages));
        if (threadIdx.x == 0)
            for (int n = stages - 1; n >= 0 && more_after; --n) put(a, flip ? stages - 1 - n : n, 2);
    }
    __device__ __forceinline__ void step(bool back) {
        const int d = back != flip ? -1 : 1;
        number += back ? -1 : 1;
        stage += d;
        if (stage == stages) stage = 0;
        if (stage < 0) stage = stages - 1;
    }
    __device__ __forceinline__ bool wait(uint32_t bar, unsigned parity) {
        if (ptx::mbar_try_wait(bar, parity)) return true;
        const long long limit = *dead ? 100000 : kWaitCycles, t0 = clock64();
        while (!ptx::mbar_try_wait(bar, parity))
            if (clock64() - t0 > limit) {
                *dead = 1;
                return false;
            }
        return true;
    }
    __device__ void load(const GnArgs &a, const Position<T, U> &p, int s) {
        const Chunk &k = p.k;
        const int per = a.reps * U, q0 = p.tile * per;
        const T *x = reinterpret_cast<const T *>(a.x) + k.base + k.head;
        const T *dy = reinterpret_cast<const T *>(a.dy) + k.base + k.head;
        const uint32_t to = data + (uint32_t)(s * stage_bytes), bar = full(s);
        if (a.windows == 1) {
            const int v0 = q0 * a.cols;
            const uint32_t bytes = 16u * (uint32_t)min(per * a.cols, k.vecs - v0);
            ptx::mbar_arrive_expect_tx(bar, TWO ? 2 * bytes : bytes);
            ptx::bulk_load(to, x + (long long)v0 * kV<T>, bytes, bar);
            if (TWO) ptx::bulk_load(to + a.tile_bytes, dy + (long long)v0 * kV<T>, bytes, bar);
        } else {
            const int c0 = p.window * a.win_cols, width = min(a.win_cols, a.cols - c0);
            uint32_t bytes = 0;
            for (int q = 0; q < per; ++q) bytes += 16u * (uint32_t)max(0, min(width, k.vecs - (q0 + q) * a.cols - c0));
            ptx::mbar_arrive_expect_tx(bar, TWO ? 2 * bytes : bytes);
            for (int q = 0; q < per; ++q) {
                const int v0 = (q0 + q) * a.cols + c0;
                const int n = min(width, k.vecs - v0);
                if (n <= 0) break;
                ptx::bulk_load(to + 16u * q * a.win_cols, x + (long long)v0 * kV<T>, 16u * n, bar);
                if (TWO) ptx::bulk_load(to + a.tile_bytes + 16u * q * a.win_cols, dy + (long long)v0 * kV<T>, 16u * n, bar);
            }
        }
    }
    // thread 0: the next tile of that kind into stage s, once every warp has let go of what is there
    __device__ __forceinline__ void put(const GnArgs &a, int s, int what) {
        bool ok = true;
        if ((used >> s) & 1u) {
            ok = wait(empty(s), (empty_parity >> s) & 1u);
            empty_parity ^= 1u << s;
        }
        used |= 1u << s;
        Position<T, U> &p = what == 2 ? *after : *here;
        if (ok && !*dead) load(a, p, s);
        if (what == 2) more_after = p.next(a, rank);
        else if (what == 0) p.next(a, rank);
        else p.previous(a);
    }
    __device__ __forceinline__ void settle(const GnArgs &a) {
        if (threadIdx.x == 0 && due >= 0) {
            put(a, due, due_what);
            due = -1;
        }
    }
    // every thread: on to the next tile of the sums; whether it is there
    __device__ __forceinline__ bool take(const GnArgs &a) {
        step(false);
        settle(a);
        const bool ok = wait(full(stage), (full_parity >> stage) & 1u);
        full_parity ^= 1u << stage;
        return ok;
    }
    __device__ __forceinline__ bool take_back(const GnArgs &a) {
        step(true);
        settle(a);
        if (number + stages >= total) return *dead == 0;  // held
        const bool ok = wait(full(stage), (full_parity >> stage) & 1u);
        full_parity ^= 1u << stage;
        return ok;
    }
    __device__ __forceinline__ void release(int what) {
        __syncwarp();
        if ((threadIdx.x & 31) == 0) ptx::mbar_arrive(empty(stage));
        if (what < 2 || more_after) {  // (only thread 0 looks)
            due = stage;
            due_what = what;
        }
    }
    __device__ __forceinline__ void done() {
        if (number + stages < total) release(0);
    }
    __device__ __forceinline__ void done_back() { release(number >= stages ? 1 : 2); }
};

// Waits for the CTAs of a team (all are resident: the launch is cooperative).  The first one waits for the whole grid instead, after the team's
// counter was cleared.  A wait that runs out marks the results as any other does.
struct Team {
    int id, rank, count;
    __device__ __forceinline__ void sync(const GnArgs &a, volatile int *dead) {
        if (a.team == 1) {
            __syncthreads();
            return;
        }
        if (count++ == 0) {
            if (rank == 0 && threadIdx.x == 0) a.arrived[id * kCounterPitch] = 0;
            cg::this_grid().sync();
            return;
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            __threadfence();
            atomicAdd(a.arrived + id * kCounterPitch, 1u);
            const unsigned want = (unsigned)(count - 1) * (unsigned)a.team;
            const long long limit = *dead ? 100000 : kWaitCycles, t0 = clock64();
            unsigned have;
            do {
                asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(have) : "l"(a.arrived + id * kCounterPitch) : "memory");
                if (have >= want) break;
                if (clock64() - t0 > limit) {
                    *dead = 1;
                    break;
                }
            } while (true);
            __threadfence();
        }
        __syncthreads();
    }
};

// ------------------------------------------------------------------------------------------------
// joining of moments
// ------------------------------------------------------------------------------------------------
struct Moments {  // (sum of weights, K, mean - K, M2)
    float W, K, m, M2;
};
__device__ __forceinline__ Moments moments(float W, float c, float S1, float S2) {
    const float m = W > 0.f ? __fdividef(S1, W) : 0.f;
    return {W, c, m, fmaxf(fmaf(-S1, m, S2), S2 * 0.f)};  // (rounding may leave less than nothing; a NaN or infinity has to stay)
}
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

__device__ __forceinline__ double warp_sum(double v) {
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ double2 warp_sum(double2 v) { return make_double2(warp_sum(v.x), warp_sum(v.y)); }

// Partial results joined in float64, about the mean of the first (fields whose level is far above their spread lose nothing, and no division is
// needed on the way): thread `i` of `of` takes every of-th, four loads at a time.
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
        const float4 v0 = __ldcg(p);
        c = (double)v0.y + v0.z;
        W = s = q = 0.;
        for (; i < n; i += 4 * of) {
            float4 v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = i + u * of < n ? __ldcg(p + (i + u * of) * stride) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int u = 0; u < 4; ++u) add(v[u]);
        }
        W = warp_sum(W);
        s = warp_sum(s);
        q = warp_sum(q);
    }
    __device__ __forceinline__ float4 stats(const GnArgs &a) const {
        const float inv = 1.f / (float)W;
        const double m = s * inv, mean = c + m;
        const float hi = (float)mean, var = (float)(q - s * m) * inv;
        return make_float4(hi, (float)(mean - hi), 1.f / sqrtf(fmaxf(var, var * 0.f) + a.eps), inv);
    }
};

// Sums over the threads of a column, N pairs each: pair i of column c at tot[i * kMaxCols + c].
template <int N> __device__ __forceinline__ void column_sums(const GnArgs &a, const Share &s, F2 (&v)[N], F2 *red, F2 *tot) {
    int rep = s.rep, c = s.col, n = a.reps;
    if (a.windows == 1 && a.cols <= 32 && (32 & (a.cols - 1)) == 0 && (a.cols & (a.cols - 1)) == 0) {  // whole columns in a warp: lanes first
        for (int o = 16; o >= a.cols; o >>= 1)
#pragma unroll
            for (int i = 0; i < N; ++i) {
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
        for (int i = 0; i < N; ++i) red[i * kThreads + rep * a.win_cols + c] = v[i];
    __syncthreads();
    for (int o = threadIdx.x; o < N * a.win_cols; o += kThreads) {
        const int i = (int)((unsigned)o / (unsigned)a.win_cols), col = o - i * a.win_cols;
        const F2 *p = red + i * kThreads + col;
        F2 t = p[0];
        for (int r = 1; r < n; ++r) t = add2(t, p[r * a.win_cols]);
        tot[i * kMaxCols + col] = t;
    }
    __syncthreads();
}
__device__ __forceinline__ float half_of(const F2 *tot, int pair, int col, int h) { return reinterpret_cast<const float *>(tot + pair * kMaxCols + col)[h]; }

// ------------------------------------------------------------------------------------------------
// forward
// ------------------------------------------------------------------------------------------------
// q: (weights beyond those of every slot, S1, S2) of the slots' pairs
template <typename T> __device__ __forceinline__ void accumulate(const F2 (&v)[kP<T>], const F2 (&c)[kP<T>], F2 (&q)[3 * kP<T>], const F2 (&w)[kP<T>]) {
#pragma unroll
    for (int p = 0; p < kP<T>; ++p) {
        const F2 d = sub2(v[p], c[p]), wd = mul2(d, w[p]);
        q[kP<T> + p] = add2(q[kP<T> + p], wd);
        q[2 * kP<T> + p] = fma2(wd, d, q[2 * kP<T> + p]);
    }
}
// sums about c + delta from those about c
__device__ __forceinline__ void recentre(F2 W, F2 delta, F2 &S1, F2 &S2) {
    const F2 t = mul2(W, delta);
    S2 = sub2(S2, mul2(delta, sub2(add2(S1, S1), t)));
    S1 = sub2(S1, t);
}

__device__ __forceinline__ uint4 vector_at(uint32_t at, bool ok) {
    uint4 u;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "r"(at) : "memory");
    if (!ok) u = make_uint4(~0u, ~0u, ~0u, ~0u);  // a NaN in every type
    return u;
}

template <typename T, typename WALK>
__device__ void chunk_moments(const GnArgs &a, const Chunk &k, WALK &walk, F2 *red, F2 *tot, float *centre, Moments *acc) {
    constexpr int V = kV<T>, P = kP<T>, U = kTileVectors;
    const T *x = reinterpret_cast<const T *>(a.x) + k.base;
    float4 *out = a.part + ((long long)k.unit * a.chunks + k.chunk) * a.gu;
    __syncthreads();
    if (a.cu > 1)
        for (int g = threadIdx.x; g < a.gu; g += kThreads) acc[g] = {0.f, 0.f, 0.f, 0.f};
    for (int win = 0; win < a.windows; ++win) {
        const Share s = make_share<T>(a, k, win);
        F2 c[P], q[3 * P];
        float W = 0.f;
#pragma unroll
        for (int p = 0; p < P; ++p) c[p] = q[p] = q[P + p] = q[2 * P + p] = f2(0.f);
        Rows r{0, 0, 0};
        if (a.lat && s.count) r = make_rows<T>(a, k, s, 0);
        for (int j = 0; j < k.tiles; ++j) {
            const bool ok = walk.take(a);
            const uint32_t at = walk.data + (uint32_t)(walk.stage * walk.stage_bytes) + 16u * (uint32_t)(s.rep * a.win_cols + s.col);
            const uint32_t step = 16u * (uint32_t)(a.reps * a.win_cols);
            const int have = min(U, s.count - j * U);
            if (have > 0) {
                // The first centre: of the first tile, the vector that counts most (a value at the pole, far out, is then no centre for
                // rows of a hundred times its weight).
                if (j == 0) unpack(vector_at(at + (a.lat && 2 * r.row < a.nlat ? have - 1 : 0) * step, ok), c, T());
                bool plain = have == U;
                float w[U];
                Rows r0 = r;
                if (plain) {
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        w[u] = 1.f;
                        if (a.lat) {
                            w[u] = __ldg(a.lat + r.row);
                            plain = plain && r.col + r.over < a.nlon;
                            advance(a, r);
                        }
                    }
                }
                if (plain) {
                    uint4 raw[U];
#pragma unroll
                    for (int u = 0; u < U; ++u) raw[u] = vector_at(at + u * step, ok);
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        F2 v[P], wp[P];
                        unpack(raw[u], v, T());
#pragma unroll
                        for (int p = 0; p < P; ++p) wp[p] = f2(w[u]);
                        accumulate<T>(v, c, q, wp);
                        W += w[u];
                    }
                } else {
                    r = r0;
#pragma unroll 1
                    for (int u = 0; u < have; ++u) {
                        F2 v[P], wp[P];
                        unpack(vector_at(at + u * step, ok), v, T());
                        float w0 = 1.f;
#pragma unroll
                        for (int p = 0; p < P; ++p) wp[p] = f2(1.f);
                        if (a.lat) {
                            float ws[V];
                            w0 = __ldg(a.lat + r.row);
                            mixed_weights<T>(a.lat, a.nlon, a.cu, s.ch0, r.row, r.col, ws);
#pragma unroll
                            for (int p = 0; p < P; ++p) {
                                wp[p] = f2(ws[2 * p], ws[2 * p + 1]);
                                q[p] = add2(q[p], sub2(wp[p], f2(w0)));
                            }
                            advance(a, r);
                        }
                        accumulate<T>(v, c, q, wp);
                        W += w0;
                    }
                }
                if ((j & (j + 1)) == 0) {
                    const F2 inv = f2(__fdividef(1.f, W));
#pragma unroll
                    for (int p = 0; p < P; ++p) {
                        const F2 to = fma2(q[P + p], inv, c[p]), delta = sub2(to, c[p]);
                        recentre(add2(f2(W), q[p]), delta, q[P + p], q[2 * P + p]);
                        c[p] = to;
                    }
                }
            }
            walk.done();
        }
        // all threads of a column: about the centre of its first thread, then added (planes: of the first slot of all)
        if (s.rep == 0)
#pragma unroll
            for (int p = 0; p < P; ++p) {
                const float2 v = split(c[p]);
                centre[(2 * p) * kMaxCols + s.col] = v.x;
                centre[(2 * p + 1) * kMaxCols + s.col] = v.y;
            }
        __syncthreads();
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const F2 c0 = a.cu == 1 ? f2(centre[0]) : f2(centre[(2 * p) * kMaxCols + s.col], centre[(2 * p + 1) * kMaxCols + s.col]);
            q[p] = add2(q[p], f2(W));
            if (s.count) recentre(q[p], sub2(c0, c[p]), q[P + p], q[2 * P + p]);
        }
        if (a.cu == 1) {
            F2 t[3] = {q[0], q[P], q[2 * P]};
#pragma unroll
            for (int p = 1; p < P; ++p)
#pragma unroll
                for (int i = 0; i < 3; ++i) t[i] = add2(t[i], q[i * P + p]);
            float v[3];
#pragma unroll
            for (int i = 0; i < 3; ++i) {
                const float2 h = split(t[i]);
                v[i] = h.x + h.y;
                for (int o = 16; o; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
            }
            float *w = reinterpret_cast<float *>(red);
            if ((threadIdx.x & 31) == 0)
#pragma unroll
                for (int i = 0; i < 3; ++i) w[i * kWarps + (threadIdx.x >> 5)] = v[i];
            __syncthreads();
            if (threadIdx.x == 0) {
#pragma unroll
                for (int i = 0; i < 3; ++i) {
                    v[i] = w[i * kWarps];
                    for (int n = 1; n < kWarps; ++n) v[i] += w[i * kWarps + n];
                }
                Moments m = moments(v[0], centre[0], v[1], v[2]);
                for (int i = 0; i < 2 * V; ++i) {  // the values outside the vectors
                    const int e = ragged<T>(k, i);
                    if (e < 0) break;
                    join(m, Moments{weight_at(a, k, e), to_f(x[e]), 0.f, 0.f});
                }
                out[0] = make_float4(m.W, m.K, m.m, m.M2);
            }
            return;
        }
        column_sums<3 * P>(a, s, q, red, tot);
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
                        join(m, moments(half_of(tot, i2 / 2, col, i2 & 1), centre[i2 * kMaxCols + col], half_of(tot, P + i2 / 2, col, i2 & 1), half_of(tot, 2 * P + i2 / 2, col, i2 & 1)));
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

// Statistics of the groups of a chunk's unit, into shared memory.  Where they are joined here (the same order in every CTA), no second
// wait for the team is needed.
__device__ __forceinline__ void unit_stats(const GnArgs &a, const Chunk &k, float4 *st) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    __syncthreads();
    if (!a.cl) {
        if (warp == 0) {
            const int g = (int)((unsigned)k.c / (unsigned)a.cg), first = k.b * a.C + g * a.cg;
            Sums64 m;
            m.gather(a.part + (long long)first * a.chunks, a.cg * a.chunks, 1, lane, 32);
            if (lane == 0) {
                st[0] = m.stats(a);
                if (k.unit == first && k.chunk == 0) a.stats[k.b * a.G + g] = st[0];
            }
        }
    } else if (a.direct) {
        for (int g = warp; g < a.G; g += kWarps) {
            Sums64 m;
            m.gather(a.part + (long long)k.b * a.chunks * a.G + g, a.chunks, a.G, lane, 32);
            if (lane == 0) {
                st[g] = m.stats(a);
                if (k.chunk == 0) a.stats[k.b * a.G + g] = st[g];
            }
        }
    } else {
        for (int g = threadIdx.x; g < a.G; g += kThreads) st[g] = __ldcg(a.stats + (long long)k.b * a.G + g);
    }
    __syncthreads();
}
// ... joined once: a CTA of the team for every group of the sample
__device__ __forceinline__ void finish_stats(const GnArgs &a, int job, int rank, double *red) {
    const int warp = threadIdx.x >> 5;
    for (int g = rank; g < a.G; g += a.team) {
        Sums64 m;
        m.gather(a.part + (long long)job * a.chunks * a.G + g, a.chunks, a.G, threadIdx.x, kThreads);
        __syncthreads();
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
            a.stats[(long long)job * a.G + g] = m.stats(a);
        }
    }
}

template <typename T, int ACT, typename WALK>
__device__ void chunk_apply(const GnArgs &a, const Chunk &k, WALK &walk, float4 *st) {
    constexpr int V = kV<T>, P = kP<T>, U = kTileVectors;
    const T *x = reinterpret_cast<const T *>(a.x) + k.base;
    T *y = reinterpret_cast<T *>(a.out) + k.base;
    unit_stats(a, k, st);
    uint4 *yv = reinterpret_cast<uint4 *>(y + k.head);
    for (int win = a.windows - 1; win >= 0; --win) {
        const Share s = make_share<T>(a, k, win);
        F2 m[P], sc[P], sh[P];
        {
            float w[V], b[V];
            int g[V];
            slot_params<V>(a, k, s.ch0, w, b, g);
#pragma unroll
            for (int p = 0; p < P; ++p) {
                const float4 u = st[g[2 * p]], v = st[g[2 * p + 1]];
                m[p] = f2(u.x, v.x);
                sc[p] = mul2(f2(u.z, v.z), f2(w[2 * p], w[2 * p + 1]));
                sh[p] = fma2(f2(-u.y, -v.y), sc[p], f2(b[2 * p], b[2 * p + 1]));
            }
        }
        for (int j = k.tiles - 1; j >= 0; --j) {
            const bool ok = walk.take_back(a);
            const uint32_t at = walk.data + (uint32_t)(walk.stage * walk.stage_bytes) + 16u * (uint32_t)(s.rep * a.win_cols + s.col);
            const uint32_t step = 16u * (uint32_t)(a.reps * a.win_cols);
            const int have = min(U, s.count - j * U);
            uint4 *to = yv + s.first + (long long)j * U * s.step;
            if (have == U) {
                uint4 raw[U];
#pragma unroll
                for (int u = 0; u < U; ++u) raw[u] = vector_at(at + u * step, ok);
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    F2 v[P];
                    unpack(raw[u], v, T());
#pragma unroll
                    for (int p = 0; p < P; ++p) v[p] = act_value<ACT>(fma2(sub2(v[p], m[p]), sc[p], sh[p]));
                    to[(long long)u * s.step] = pack(v, T());
                }
            } else {
#pragma unroll 1
                for (int u = 0; u < have; ++u) {
                    F2 v[P];
                    unpack(vector_at(at + u * step, ok), v, T());
#pragma unroll
                    for (int p = 0; p < P; ++p) v[p] = act_value<ACT>(fma2(sub2(v[p], m[p]), sc[p], sh[p]));
                    to[(long long)u * s.step] = pack(v, T());
                }
            }
            walk.done_back();
        }
    }
    if ((int)threadIdx.x < 2 * V) {
        const int e = ragged<T>(k, threadIdx.x);
        if (e >= 0) {
            const int ch = e % a.cu, c = a.cl ? ch : k.c;
            const float4 v = st[ch / a.cgu];
            const float sc = v.z * load_param(a.weight, a.pdtype, c, 1.f), sh = fmaf(-v.y, sc, load_param(a.bias, a.pdtype, c, 0.f));
            store_f(y + e, split(act_value<ACT>(f2(fmaf(to_f(x[e]) - v.x, sc, sh)))).x);
        }
    }
}

extern __shared__ __align__(16) unsigned char gn_smem[];

template <typename T, int ACT>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) gn_forward_kernel(const __grid_constant__ GnArgs a) {
    // partial sums and totals are never alive together with a tile's readers; in the ring there is no room for them
    __shared__ __align__(16) F2 red[3 * kP<T> * kThreads];
    __shared__ __align__(16) F2 tot[3 * kP<T> * kMaxCols];
    __shared__ float centre[kV<T> * kMaxCols];
    __shared__ unsigned long long bars[2 * kMaxStages];
    __shared__ int dead;
    __shared__ Position<T, kTileVectors> positions[2];
    Moments *acc = reinterpret_cast<Moments *>(gn_smem + a.stages * a.tile_bytes);
    float4 *st = reinterpret_cast<float4 *>(acc);  // (one or the other)
    Team team{(int)blockIdx.x % a.teams, (int)blockIdx.x / a.teams, 0};
    Walk<T, kTileVectors, false> walk;
    walk.init(a, gn_smem, bars, &dead, positions, team.id, team.rank);
    for (int job = team.id; job < a.jobs; job += a.teams) {
        Chunk k = make_chunk<T, kTileVectors>(a, job, min(team.rank, a.tasks - 1));
        walk.begin(a, job, k);
        int last = team.rank;
        for (int t = team.rank; t < a.tasks; t += a.team) {
            if (t != team.rank) k = make_chunk<T, kTileVectors>(a, job, t);
            chunk_moments<T>(a, k, walk, red, tot, centre, acc);
            last = t;
        }
        team.sync(a, &dead);
        if (!a.direct) {
            finish_stats(a, job, team.rank, reinterpret_cast<double *>(red));
            team.sync(a, &dead);
        }
        walk.turn(a);
        if (team.rank < a.tasks)
            for (int t = last; t >= 0; t -= a.team) {
                if (t != last) k = make_chunk<T, kTileVectors>(a, job, t);
                chunk_apply<T, ACT>(a, k, walk, st);
            }
    }
}

// ------------------------------------------------------------------------------------------------
// backward
// ------------------------------------------------------------------------------------------------
constexpr int kTileVectorsB = kTileVectors / 2;

__device__ __forceinline__ void load_stats(const GnArgs &a, const Chunk &k, float4 *st) {
    __syncthreads();
    if (a.cl)
        for (int g = threadIdx.x; g < a.G; g += kThreads) st[g] = __ldg(a.stats + (long long)k.b * a.G + g);
    else if (threadIdx.x == 0) st[0] = __ldg(a.stats + k.b * a.G + (int)((unsigned)k.c / (unsigned)a.cg));
}
// one value outside the vectors: (g, x - m)
template <typename T, int ACT> __device__ __forceinline__ float2 ragged_slope(const GnArgs &a, const Chunk &k, const float4 *st, float x, float dy, int ch) {
    const int c = a.cl ? ch : k.c;
    const float4 v = st[ch / a.cgu];
    const float sc = v.z * load_param(a.weight, a.pdtype, c, 1.f), sh = fmaf(-v.y, sc, load_param(a.bias, a.pdtype, c, 0.f)), d = x - v.x;
    return make_float2(dy * split(act_slope<ACT>(f2(fmaf(d, sc, sh)))).x, d);
}

template <typename T, int ACT, typename WALK>
__device__ void chunk_sums(const GnArgs &a, const Chunk &k, WALK &walk, F2 *red, F2 *tot, float2 *acc, float4 *st) {
    constexpr int V = kV<T>, P = kP<T>, U = kTileVectorsB;
    const T *x = reinterpret_cast<const T *>(a.x) + k.base, *dy = reinterpret_cast<const T *>(a.dy) + k.base;
    float2 *out = a.bpart + ((long long)k.unit * a.chunks + k.chunk) * a.cu;
    load_stats(a, k, st);
    if (a.cu > 1)
        for (int c = threadIdx.x; c < a.cu; c += kThreads) acc[c] = make_float2(0.f, 0.f);
    __syncthreads();
    for (int win = 0; win < a.windows; ++win) {
        const Share s = make_share<T>(a, k, win);
        F2 q[2 * P], m[P], sc[P], sh[P];  // q: sum g, sum g (x - m)
        {
            float w[V], b[V];
            int g[V];
            slot_params<V>(a, k, s.ch0, w, b, g);
#pragma unroll
            for (int p = 0; p < P; ++p) {
                const float4 u = st[g[2 * p]], v = st[g[2 * p + 1]];
                m[p] = f2(u.x, v.x);
                sc[p] = mul2(f2(u.z, v.z), f2(w[2 * p], w[2 * p + 1]));
                sh[p] = fma2(f2(-u.y, -v.y), sc[p], f2(b[2 * p], b[2 * p + 1]));
                q[p] = q[P + p] = f2(0.f);
            }
        }
        for (int j = 0; j < k.tiles; ++j) {
            const bool ok = walk.take(a);
            const uint32_t at = walk.data + (uint32_t)(walk.stage * walk.stage_bytes) + 16u * (uint32_t)(s.rep * a.win_cols + s.col);
            const uint32_t step = 16u * (uint32_t)(a.reps * a.win_cols);
            const int have = min(U, s.count - j * U);
            auto one = [&](uint4 rx, uint4 rd) {
                F2 v[P], d[P];
                unpack(rx, v, T());
                unpack(rd, d, T());
#pragma unroll
                for (int p = 0; p < P; ++p) {
                    const F2 e = sub2(v[p], m[p]), g = mul2(d[p], act_slope<ACT>(fma2(e, sc[p], sh[p])));
                    q[p] = add2(q[p], g);
                    q[P + p] = fma2(g, e, q[P + p]);
                }
            };
            if (have == U) {
                uint4 rx[U], rd[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    rx[u] = vector_at(at + u * step, ok);
                    rd[u] = vector_at(at + a.tile_bytes + u * step, ok);
                }
#pragma unroll
                for (int u = 0; u < U; ++u) one(rx[u], rd[u]);
            } else {
#pragma unroll 1
                for (int u = 0; u < have; ++u) one(vector_at(at + u * step, ok), vector_at(at + a.tile_bytes + u * step, ok));
            }
            walk.done();
        }
        if (a.cu == 1) {
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
            return;
        }
        column_sums<2 * P>(a, s, q, red, tot);
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

// (sum h, sum h xh) of the groups of a chunk's unit
__device__ void group_sums(const GnArgs &a, const Chunk &k, float2 *gsum) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (a.cl) {
        for (int g = warp; g < a.G; g += kWarps) {
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
            if (lane == 0) gsum[g] = make_float2((float)t.x, (float)t.y);
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
// ... the sums of the channels joined once: 32 channels of a sample for a CTA of the team, a lane each, the chunks dealt to the warps
__device__ __forceinline__ void finish_sums(const GnArgs &a, int job, int rank, double2 *red) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int t = rank; t < (a.C + 31) / 32; t += a.team) {
        const int c = t * 32 + lane;
        double2 v = make_double2(0., 0.);
        if (c < a.C)
            for (int n = warp; n < a.chunks; n += 4 * kWarps) {
                float2 p[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) p[u] = n + u * kWarps < a.chunks ? __ldcg(a.bpart + ((long long)job * a.chunks + n + u * kWarps) * a.C + c) : make_float2(0.f, 0.f);
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    v.x += p[u].x;
                    v.y += p[u].y;
                }
            }
        __syncthreads();
        red[threadIdx.x] = v;
        __syncthreads();
        if (warp == 0 && c < a.C) {
            for (int w = 1; w < kWarps; ++w) {
                v.x += red[w * 32 + lane].x;
                v.y += red[w * 32 + lane].y;
            }
            a.csum[(long long)job * a.C + c] = v;
        }
    }
}

// dx = sc g - a (alpha + (x - m) beta),  alpha = r (sum h - lo r sum h xh) / sum a,  beta = r^2 sum h xh / sum a
__device__ __forceinline__ float2 group_terms(const float4 &v, const float2 &t) { return make_float2(-v.z * fmaf(-v.y * v.z, t.y, t.x) * v.w, -v.z * v.z * t.y * v.w); }

template <typename T, int ACT, typename WALK>
__device__ void chunk_dx(const GnArgs &a, const Chunk &k, WALK &walk, float2 *gsum, float4 *st) {
    constexpr int V = kV<T>, P = kP<T>, U = kTileVectorsB;
    const T *x = reinterpret_cast<const T *>(a.x) + k.base, *dy = reinterpret_cast<const T *>(a.dy) + k.base;
    T *dx = reinterpret_cast<T *>(a.out) + k.base;
    load_stats(a, k, st);
    group_sums(a, k, gsum);
    __syncthreads();
    uint4 *ov = reinterpret_cast<uint4 *>(dx + k.head);
    for (int win = a.windows - 1; win >= 0; --win) {
        const Share s = make_share<T>(a, k, win);
        F2 m[P], sc[P], sh[P], al[P], be[P];
        {
            float w[V], b[V];
            int g[V];
            slot_params<V>(a, k, s.ch0, w, b, g);
#pragma unroll
            for (int p = 0; p < P; ++p) {
                const float4 u = st[g[2 * p]], v = st[g[2 * p + 1]];
                const float2 tu = group_terms(u, gsum[g[2 * p]]), tv = group_terms(v, gsum[g[2 * p + 1]]);
                m[p] = f2(u.x, v.x);
                sc[p] = mul2(f2(u.z, v.z), f2(w[2 * p], w[2 * p + 1]));
                sh[p] = fma2(f2(-u.y, -v.y), sc[p], f2(b[2 * p], b[2 * p + 1]));
                al[p] = f2(tu.x, tv.x);
                be[p] = f2(tu.y, tv.y);
            }
        }
        Rows r{0, 0, 0};  // of the vector behind the tile at hand
        if (a.lat && s.count) r = make_rows<T>(a, k, s, k.tiles * U);
        for (int j = k.tiles - 1; j >= 0; --j) {
            const bool ok = walk.take_back(a);
            const uint32_t at = walk.data + (uint32_t)(walk.stage * walk.stage_bytes) + 16u * (uint32_t)(s.rep * a.win_cols + s.col);
            const uint32_t step = 16u * (uint32_t)(a.reps * a.win_cols);
            const int have = min(U, s.count - j * U);
            uint4 *to = ov + s.first + (long long)j * U * s.step;
            auto one = [&](uint4 rx, uint4 rd, const F2 (&wt)[P], int u) {
                F2 v[P], d[P];
                unpack(rx, v, T());
                unpack(rd, d, T());
#pragma unroll
                for (int p = 0; p < P; ++p) {
                    const F2 e = sub2(v[p], m[p]), g = mul2(d[p], act_slope<ACT>(fma2(e, sc[p], sh[p])));
                    v[p] = fma2(wt[p], fma2(e, be[p], al[p]), mul2(sc[p], g));
                }
                to[(long long)u * s.step] = pack(v, T());
            };
            bool plain = have == U;
            float w[U];
#pragma unroll
            for (int u = 0; u < U; ++u) w[u] = 1.f;
            if (a.lat && s.count) {
                retreat(a, r, U);
                Rows n = r;
                if (plain)
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        w[u] = __ldg(a.lat + n.row);
                        plain = plain && n.col + n.over < a.nlon;
                        advance(a, n);
                    }
            }
            if (plain) {
                uint4 rx[U], rd[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    rx[u] = vector_at(at + u * step, ok);
                    rd[u] = vector_at(at + a.tile_bytes + u * step, ok);
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    F2 wt[P];
#pragma unroll
                    for (int p = 0; p < P; ++p) wt[p] = f2(w[u]);
                    one(rx[u], rd[u], wt, u);
                }
            } else {
                Rows n = r;
#pragma unroll 1
                for (int u = 0; u < have; ++u) {
                    F2 wt[P];
#pragma unroll
                    for (int p = 0; p < P; ++p) wt[p] = f2(1.f);
                    if (a.lat) {
                        float ws[V];
                        mixed_weights<T>(a.lat, a.nlon, a.cu, s.ch0, n.row, n.col, ws);
#pragma unroll
                        for (int p = 0; p < P; ++p) wt[p] = f2(ws[2 * p], ws[2 * p + 1]);
                        advance(a, n);
                    }
                    one(vector_at(at + u * step, ok), vector_at(at + a.tile_bytes + u * step, ok), wt, u);
                }
            }
            walk.done_back();
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

template <typename T, int ACT>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) gn_backward_kernel(const __grid_constant__ GnArgs a) {
    __shared__ __align__(16) F2 red[2 * kP<T> * kThreads];
    __shared__ __align__(16) F2 tot[2 * kP<T> * kMaxCols];
    __shared__ unsigned long long bars[2 * kMaxStages];
    __shared__ int dead;
    __shared__ Position<T, kTileVectorsB> positions[2];
    float4 *st = reinterpret_cast<float4 *>(gn_smem + 2 * a.stages * a.tile_bytes);
    float2 *acc = reinterpret_cast<float2 *>(st + a.gu);  // the sums of a chunk's channels, or those of its groups
    Team team{(int)blockIdx.x % a.teams, (int)blockIdx.x / a.teams, 0};
    Walk<T, kTileVectorsB, true> walk;
    walk.init(a, gn_smem, bars, &dead, positions, team.id, team.rank);
    for (int job = team.id; job < a.jobs; job += a.teams) {
        Chunk k = make_chunk<T, kTileVectorsB>(a, job, min(team.rank, a.tasks - 1));
        walk.begin(a, job, k);
        int last = team.rank;
        for (int t = team.rank; t < a.tasks; t += a.team) {
            if (t != team.rank) k = make_chunk<T, kTileVectorsB>(a, job, t);
            chunk_sums<T, ACT>(a, k, walk, red, tot, acc, st);
            last = t;
        }
        team.sync(a, &dead);
        if (!a.direct) {
            finish_sums(a, job, team.rank, reinterpret_cast<double2 *>(red));
            team.sync(a, &dead);
        }
        if (!a.out) {
            walk.skip(a);
            continue;
        }
        walk.turn(a);
        if (team.rank < a.tasks)
            for (int t = last; t >= 0; t -= a.team) {
                if (t != last) k = make_chunk<T, kTileVectorsB>(a, job, t);
                chunk_dx<T, ACT>(a, k, walk, acc, st);
            }
    }
    if (!a.dweight && !a.dbias) return;
    // the parameters' gradients: one warp a channel, over all samples
    cg::this_grid().sync();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int c = blockIdx.x * kWarps + warp; c < a.C; c += gridDim.x * kWarps) {
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
}

// ------------------------------------------------------------------------------------------------
// host
// ------------------------------------------------------------------------------------------------
constexpr int kMaxWaves = 4;            // chunks a CTA takes one after the other, at most, where a unit is cut
constexpr int kMaxChannels = 4096;      // what a CTA keeps per channel or group has to fit into its shared memory
constexpr int kDirect = 2048;           // partial results of a unit up to which every CTA joins them itself
constexpr size_t kSmPerCta = (228 << 10) / kCtasPerSm - 1024, kSmWhole = 227 << 10;  // shared memory of a CTA, two or one on an SM
constexpr size_t kResident = 64 << 20;  // bytes that the teams may have between two passes for L2 (126 MB) to serve the second

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
    size_t smem = 0;
};

// Chunks of a unit for a team of n CTAs.
void cut(GnArgs &a, int n, int V, bool backward) {
    const long long values = a.hw * a.cu, most = std::max<long long>(1, std::min<long long>(a.hw, values / (kThreads * V)));
    long long chunks = 1;
    double best = 0.;
    for (int w = 1; w <= kMaxWaves; ++w) {
        const long long c = std::min<long long>(most, std::max(1, w * n / a.job_units)), tasks = c * a.job_units;
        const double filled = (double)tasks / (double)((tasks + n - 1) / n * n);  // of the CTAs' time
        if (filled > best + 0.03) {
            best = filled;
            chunks = c;
        }
    }
    a.chunk_px = (int)((a.hw + chunks - 1) / chunks);
    if (a.chunk_px >= 256) a.chunk_px = (a.chunk_px + 31) / 32 * 32;  // (chunks of an aligned field begin aligned)
    a.chunks = (int)((a.hw + a.chunk_px - 1) / a.chunk_px);
    a.tasks = a.job_units * a.chunks;
    a.team = std::min(n, a.tasks);
    a.direct = !a.cl || (long long)a.chunks * (backward ? a.C : a.G) <= kDirect;
}

Launch geometry(const GroupNormDesc &d, bool backward, int sms) {
    Launch l;
    GnArgs &a = l.a;
    const int es = value_bytes(d.dtype), V = 16 / es, U = backward ? kTileVectorsB : kTileVectors;
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
    a.jobs = a.cl ? a.B : a.B * a.G;
    a.job_units = a.cl ? 1 : a.cg;
    // columns
    a.cols = a.cu / std::gcd(a.cu, V);
    a.dup = a.cols * V / a.cu;
    a.windows = ceil_div(a.cols, kMaxCols);
    a.win_cols = ceil_div(a.cols, a.windows);
    a.reps = kThreads / a.win_cols;
    for (a.lanes = 1; a.lanes < 32 && a.lanes < a.cgu * a.dup;) a.lanes *= 2;
    const long long step_px = (long long)a.reps * a.cols * V / a.cu;
    a.step_rows = (int)(step_px / a.nlon);
    a.step_cols = (int)(step_px % a.nlon);
    // the ring
    const size_t fixed = backward ? sizeof(F2) * V * (kThreads + kMaxCols) + 1024 : sizeof(F2) * V * 3 / 2 * (kThreads + kMaxCols) + sizeof(float) * V * kMaxCols + 1024;
    a.tile_bytes = 16 * a.reps * U * a.win_cols;
    const size_t stage = (size_t)a.tile_bytes * (backward ? 2 : 1);
    const size_t kept = backward ? (sizeof(float4) * a.gu + sizeof(float2) * std::max(a.cu, a.gu)) : sizeof(Moments) * a.gu;
    int per_sm = kCtasPerSm;
    size_t room = kSmPerCta - fixed;
    if (room < kept + 3 * stage) {
        per_sm = 1;
        room = kSmWhole - fixed;
    }
    a.stages = (int)std::min<size_t>(kMaxStages, (room - kept) / stage);
    l.smem = a.stages * stage + kept;
    const int grid = std::max(1, sms * per_sm);
    // Teams.  Fewer and larger ones hold more of their job on chip; more of them cover each other's waits.  Estimated time of a choice: the
    // rounds of jobs, each some microseconds of sums, waits and statistics, and the job's bytes at the team's part of the memory's rate.
    const double job_bytes = (double)a.hw * a.cu * a.job_units * es * (backward ? 2 : 1), share = 6.5e3 / grid;  // KB per us and CTA
    double best = 0.;
    int teams = 1;
    const int most_teams = std::min(a.jobs, grid);
    for (int t = 1; t <= most_teams; ++t) {
        const int n = grid / t;
        t = std::min(most_teams, grid / n);  // (the most teams of that size)
        const double again = std::max(0., job_bytes - (double)n * a.stages * (double)stage) * (job_bytes * t <= (double)kResident ? 0.3 : 0.9);
        const double traffic = job_bytes * (backward ? 1.5 : 2.) + again;
        const double us = (double)((a.jobs + t - 1) / t) * ((n > 1 ? 4. : 2.) + traffic / 1e3 / (share * n));
        if (best == 0. || us < best) {
            best = us;
            teams = t;
        }
    }
    a.teams = teams;
    cut(a, grid / teams, V, backward);
    l.grid = a.teams * a.team;
    return l;
}


struct GnWs {
    size_t part = 0, csum = 0, arrived = 0;
    size_t total() const { return part + csum + arrived; }
};
GnWs ws_sizes(const GnArgs &a, bool backward) {
    GnWs w;
    const size_t parts = (size_t)a.jobs * (size_t)a.tasks;
    w.part = up256(backward ? parts * a.cu * sizeof(float2) : parts * a.gu * sizeof(float4));
    if (backward && a.cl) w.csum = up256((size_t)a.B * a.C * sizeof(double2));
    w.arrived = up256((size_t)a.teams * kCounterPitch * sizeof(unsigned));
    return w;
}

int launch(const void *kernel, const Launch &l, cudaStream_t st) {
    SHT_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)l.smem));
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

int plan(const GroupNormDesc *d, bool backward, const void *ws, size_t ws_bytes, const void *stats, Launch *l) {
    const int sms = sm_count();
    *l = geometry(*d, backward, effective_sms(sms));
    size_t need = ws_sizes(l->a, backward).total();
    if (ws_bytes < need && effective_sms(sms) != sms) {
        // The limit on the SMs was changed after the workspace was asked for: one team on fewer CTAs never needs more chunks.
        cut(l->a, l->grid, 16 / value_bytes(d->dtype), backward);
        need = ws_sizes(l->a, backward).total();
    }
    if (!ws || ws_bytes < need) return fail(SHTB200_EWORKSPACE, "workspace too small: need " + std::to_string(need) + " bytes");
    if (((uintptr_t)ws & 255) != 0) return fail(SHTB200_EINVAL, "workspace must be 256-byte aligned");
    if (((uintptr_t)stats & 15) != 0) return fail(SHTB200_EINVAL, "the statistics must be 16-byte aligned");
    if ((long long)l->a.chunk_px * l->a.cu > (1 << 30)) return fail(SHTB200_EINVAL, "group norm shape too large");
    return SHTB200_OK;
}
// vectors are aligned in all tensors or in none
bool aligned_alike(const void *p, const void *q) { return !p || !q || (((uintptr_t)p ^ (uintptr_t)q) & 15) == 0; }

}  // namespace

size_t group_norm_workspace(const GroupNormDesc *d, bool backward) {
    if (check_desc(d)) return 0;
    if (d->batch == 0) return 256;
    return std::max<size_t>(ws_sizes(geometry(*d, backward, sm_count()).a, backward).total(), 256);
}

int group_norm_forward(const GroupNormDesc *d, const void *x, const float *lat, const void *weight, const void *bias, void *y, void *stats, void *ws, size_t ws_bytes,
                       cudaStream_t st) {
    int rc = check_desc(d);
    if (rc) return rc;
    if (d->batch == 0) return SHTB200_OK;
    if (!x || !y || !stats) return fail(SHTB200_EINVAL, "null pointer");
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
    a.arrived = reinterpret_cast<unsigned *>(reinterpret_cast<char *>(ws) + ws_sizes(a, false).part);
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
    a.csum = reinterpret_cast<double2 *>(reinterpret_cast<char *>(ws) + ws_sizes(a, true).part);
    a.arrived = reinterpret_cast<unsigned *>(reinterpret_cast<char *>(a.csum) + ws_sizes(a, true).csum);
    return launch(d->dtype == SHTB200_F32    ? backward_kernel<float>(d->activation)
                  : d->dtype == SHTB200_BF16 ? backward_kernel<__nv_bfloat16>(d->activation)
                                             : backward_kernel<__half>(d->activation),
                  l, st);
}

}  // namespace shtb200
