// Group normalisation with an activation on fields over the sphere, forward and backward.
//
// x (B, C, nlat, nlon), planes or channels last, G groups of C / G channels, a_k = weight of latitude row k:
//     mu = sum a x / sum a,  v = sum a (x - mu)^2 / sum a      (over the C / G channels and all grid points of a group)
//     xh = (x - mu) r,  r = (v + eps)^(-1/2),  z = w_c xh + b_c,  y = act(z)
// With g = dy act'(z), h = w_c g and q = a / sum a:
//     db_c = sum g,  dw_c = sum g xh,  dx = r (h - q (sum h + xh sum h xh)).
// All of it is bound by memory: a few operations per element, x (and dy) read, y (dx) written.
//
// Statistics are kept as (W, K, mean - K, M2) = (sum a, a value of the field, weighted mean less K, sum a (x - mean)^2), so that fields
// whose level is far above their spread (pressures, temperatures) lose nothing; partial results are merged in float64.

#include "common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace shtb200 {

namespace {

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

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

__device__ __forceinline__ float act_value(float z, int act) {
    if (act == SHTB200_ACT_RELU) return z <= 0.f ? 0.f : z;  // (a NaN stays one)
    if (act == SHTB200_ACT_SILU) return z / (1.f + expf(-z));
    if (act == SHTB200_ACT_GELU) return 0.5f * z * erfcf(-0.70710678f * z);
    return z;
}
__device__ __forceinline__ float act_slope(float z, int act) {
    if (act == SHTB200_ACT_RELU) return z <= 0.f ? 0.f : 1.f;
    if (act == SHTB200_ACT_SILU) {
        const float s = 1.f / (1.f + expf(-z));
        return s * (1.f + z * (1.f - s));
    }
    if (act == SHTB200_ACT_GELU) return 0.5f * erfcf(-0.70710678f * z) + z * 0.39894228f * expf(-0.5f * z * z);
    return 1.f;
}

struct GnArgs {
    const void *x, *dy;
    void *out;
    const float *lat;          // nullptr: 1 everywhere
    const void *weight, *bias;
    void *dweight, *dbias;
    float4 *stats;             // (B, G): mean, its low part, r, 1 / sum a
    float4 *part;              // forward: (B, C, chunks) (W, K, mean - K, M2)
    float2 *bpart;             // backward: (B, C, chunks) (sum g, sum g xh)
    double2 *csum;             // backward: (B, C)
    float2 *gsum;              // backward: (B, G) (sum h, sum h xh)
    long long hw;
    int B, C, G, nlon, cl, act, pdtype, chunks;
    long long chunk_px;
    float eps;
};

constexpr int kThreads = 256;

struct Moments {
    float W = 0.f, mean = 0.f, M2 = 0.f;
    __device__ __forceinline__ void add(float x, float a) {
        if (a == 0.f) return;
        const float d = x - mean;
        W += a;
        const float inc = d * (a / W);
        mean += inc;
        M2 = fmaf(a * d, x - mean, M2);
    }
    __device__ __forceinline__ void merge(float W2, float mean2, float M22) {
        if (W2 == 0.f) return;
        const float d = mean2 - mean, Wn = W + W2, f = W2 / Wn;
        mean = fmaf(d, f, mean);
        M2 += M22 + d * d * W * f;
        W = Wn;
    }
};

// Work of one CTA: channel window [c0, c0 + cw) of sample b, pixels [p0, p1); thread -> (channel c, first pixel, step).
struct Job {
    int b, c, chunk;
    long long p0, p1, step;
    long long base, pitch;  // element (p) of the thread's channel lies at base + p * pitch
    int cw, reps;
};
__device__ __forceinline__ bool make_job(const GnArgs &a, Job &j) {
    j.chunk = (int)(blockIdx.x % (unsigned)a.chunks);
    const int unit = (int)(blockIdx.x / (unsigned)a.chunks);
    const long long lo = j.chunk * a.chunk_px, hi = min(lo + a.chunk_px, a.hw);
    if (!a.cl) {
        j.b = unit / a.C;
        j.c = unit % a.C;
        j.cw = 1;
        j.reps = kThreads;
        j.base = (long long)unit * a.hw;
        j.pitch = 1;
        j.p0 = lo + threadIdx.x;
    } else {
        const int nwin = (a.C + kThreads - 1) / kThreads;
        j.b = unit / nwin;
        const int c0 = (unit % nwin) * kThreads;
        j.cw = min(kThreads, a.C - c0);
        j.reps = kThreads / j.cw;
        j.c = c0 + (int)threadIdx.x % j.cw;
        j.base = (long long)j.b * a.hw * a.C + j.c;
        j.pitch = a.C;
        j.p0 = lo + (int)threadIdx.x / j.cw;
    }
    j.p1 = hi;
    j.step = j.reps;
    return (int)threadIdx.x < j.cw * j.reps;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) gn_stats_kernel(const GnArgs a) {
    Job j;
    const bool on = make_job(a, j);
    const T *x = reinterpret_cast<const T *>(a.x) + j.base;
    Moments m;
    float K = 0.f;
    if (on) {
        K = to_f(x[j.chunk * a.chunk_px * j.pitch]);
        for (long long p = j.p0; p < j.p1; p += j.step) m.add(to_f(x[p * j.pitch]) - K, a.lat ? a.lat[p / a.nlon] : 1.f);
    }
    __shared__ float s[3][kThreads];
    s[0][threadIdx.x] = m.W;
    s[1][threadIdx.x] = m.mean;
    s[2][threadIdx.x] = m.M2;
    __syncthreads();
    if ((int)threadIdx.x < j.cw) {
        for (int r = 1; r < j.reps; ++r) m.merge(s[0][threadIdx.x + r * j.cw], s[1][threadIdx.x + r * j.cw], s[2][threadIdx.x + r * j.cw]);
        a.part[((long long)j.b * a.C + j.c) * a.chunks + j.chunk] = make_float4(m.W, K, m.mean, m.M2);
    }
}

__device__ double block_sum(double v) {
    __shared__ double s[kThreads / 32];
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    double t = 0.;
    for (int i = 0; i < kThreads / 32; ++i) t += s[i];
    return t;
}

// one CTA per (b, group)
__global__ void __launch_bounds__(kThreads) gn_finish_stats_kernel(const GnArgs a) {
    const long long n = (long long)(a.C / a.G) * a.chunks;
    const float4 *p = a.part + (long long)blockIdx.x * n;
    double W = 0., s = 0.;
    for (long long i = threadIdx.x; i < n; i += kThreads) {
        const float4 v = p[i];
        W += v.x;
        s += v.x * ((double)v.y + v.z);
    }
    W = block_sum(W);
    const double mean = block_sum(s) / W;
    double M2 = 0.;
    for (long long i = threadIdx.x; i < n; i += kThreads) {
        const float4 v = p[i];
        const double d = ((double)v.y - mean) + v.z;
        M2 += v.w + v.x * d * d;
    }
    M2 = block_sum(M2);
    if (threadIdx.x == 0) {
        const float hi = (float)mean;
        a.stats[blockIdx.x] = make_float4(hi, (float)(mean - hi), (float)(1. / sqrt(M2 / W + (double)a.eps)), (float)(1. / W));
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) gn_apply_kernel(const GnArgs a) {
    Job j;
    if (!make_job(a, j)) return;
    const T *x = reinterpret_cast<const T *>(a.x) + j.base;
    T *y = reinterpret_cast<T *>(a.out) + j.base;
    const float4 st = a.stats[j.b * a.G + j.c / (a.C / a.G)];
    const float w = load_param(a.weight, a.pdtype, j.c, 1.f), b = load_param(a.bias, a.pdtype, j.c, 0.f);
    const float scale = st.z * w, shift = fmaf(-st.y, scale, b);
    for (long long p = j.p0; p < j.p1; p += j.step) y[p * j.pitch] = from_f<T>(act_value(fmaf(to_f(x[p * j.pitch]) - st.x, scale, shift), a.act));
}

template <typename T>
__global__ void __launch_bounds__(kThreads) gn_backward_sums_kernel(const GnArgs a) {
    Job j;
    const bool on = make_job(a, j);
    const T *x = reinterpret_cast<const T *>(a.x) + j.base;
    const T *dy = reinterpret_cast<const T *>(a.dy) + j.base;
    const float4 st = a.stats[j.b * a.G + j.c / (a.C / a.G)];
    const float w = load_param(a.weight, a.pdtype, j.c, 1.f), b = load_param(a.bias, a.pdtype, j.c, 0.f);
    float s1 = 0.f, s2 = 0.f;
    if (on)
        for (long long p = j.p0; p < j.p1; p += j.step) {
            const float xh = fmaf(to_f(x[p * j.pitch]) - st.x, st.z, -st.y * st.z);
            const float g = to_f(dy[p * j.pitch]) * act_slope(fmaf(xh, w, b), a.act);
            s1 += g;
            s2 = fmaf(g, xh, s2);
        }
    __shared__ float s[2][kThreads];
    s[0][threadIdx.x] = s1;
    s[1][threadIdx.x] = s2;
    __syncthreads();
    if ((int)threadIdx.x < j.cw) {
        for (int r = 1; r < j.reps; ++r) {
            s1 += s[0][threadIdx.x + r * j.cw];
            s2 += s[1][threadIdx.x + r * j.cw];
        }
        a.bpart[((long long)j.b * a.C + j.c) * a.chunks + j.chunk] = make_float2(s1, s2);
    }
}

// one CTA per (b, group)
__global__ void __launch_bounds__(kThreads) gn_finish_backward_kernel(const GnArgs a) {
    const int cg = a.C / a.G, b = blockIdx.x / a.G, g = blockIdx.x % a.G;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    double A = 0., Q = 0.;
    for (int i = warp; i < cg; i += kThreads / 32) {
        const int c = g * cg + i;
        const float2 *p = a.bpart + ((long long)b * a.C + c) * a.chunks;
        double s1 = 0., s2 = 0.;
        for (int k = lane; k < a.chunks; k += 32) {
            const float2 v = p[k];
            s1 += v.x;
            s2 += v.y;
        }
        for (int o = 16; o; o >>= 1) {
            s1 += __shfl_xor_sync(0xffffffffu, s1, o);
            s2 += __shfl_xor_sync(0xffffffffu, s2, o);
        }
        if (lane == 0) {
            a.csum[(long long)b * a.C + c] = make_double2(s1, s2);
            const double w = load_param(a.weight, a.pdtype, c, 1.f);
            A += w * s1;
            Q += w * s2;
        }
    }
    A = block_sum(A);
    Q = block_sum(Q);
    if (threadIdx.x == 0) a.gsum[blockIdx.x] = make_float2((float)A, (float)Q);
}

__global__ void __launch_bounds__(kThreads) gn_param_grads_kernel(const GnArgs a) {
    const int c = blockIdx.x * kThreads + threadIdx.x;
    if (c >= a.C) return;
    double s1 = 0., s2 = 0.;
    for (int b = 0; b < a.B; ++b) {
        const double2 v = a.csum[(long long)b * a.C + c];
        s1 += v.x;
        s2 += v.y;
    }
    store_param(a.dbias, a.pdtype, c, (float)s1);
    store_param(a.dweight, a.pdtype, c, (float)s2);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) gn_dx_kernel(const GnArgs a) {
    Job j;
    if (!make_job(a, j)) return;
    const T *x = reinterpret_cast<const T *>(a.x) + j.base;
    const T *dy = reinterpret_cast<const T *>(a.dy) + j.base;
    T *dx = reinterpret_cast<T *>(a.out) + j.base;
    const int bg = j.b * a.G + j.c / (a.C / a.G);
    const float4 st = a.stats[bg];
    const float2 gs = a.gsum[bg];
    const float w = load_param(a.weight, a.pdtype, j.c, 1.f), b = load_param(a.bias, a.pdtype, j.c, 0.f);
    for (long long p = j.p0; p < j.p1; p += j.step) {
        const float xh = fmaf(to_f(x[p * j.pitch]) - st.x, st.z, -st.y * st.z);
        const float h = w * to_f(dy[p * j.pitch]) * act_slope(fmaf(xh, w, b), a.act);
        const float q = st.w * (a.lat ? a.lat[p / a.nlon] : 1.f);
        dx[p * j.pitch] = from_f<T>(st.z * fmaf(-q, fmaf(xh, gs.y, gs.x), h));
    }
}

struct GnWs {
    size_t part = 0, csum = 0, gsum = 0;
    size_t total() const { return part + csum + gsum; }
};
size_t up256(size_t b) { return (b + 255) / 256 * 256; }

// chunks of pixels: enough CTAs to fill the GPU a few times over, at least 1024 elements a CTA
void geometry(const GroupNormDesc &d, GnArgs &a, long long *units) {
    a.hw = (long long)d.nlat * d.nlon;
    a.B = d.batch;
    a.C = d.channels;
    a.G = d.groups;
    a.nlon = d.nlon;
    a.cl = d.channels_last;
    a.act = d.activation;
    a.pdtype = d.param_dtype;
    a.eps = d.eps;
    *units = a.cl ? (long long)a.B * ceil_div(a.C, kThreads) : (long long)a.B * a.C;
    const int cw = a.cl ? std::min(a.C, kThreads) : 1;
    const long long least = std::max(1, 1024 / cw);
    long long chunks = std::max<long long>(1, 148 * 8 / std::max<long long>(1, *units));
    chunks = std::min(chunks, (a.hw + least - 1) / least);
    a.chunk_px = (a.hw + chunks - 1) / chunks;
    a.chunks = (int)((a.hw + a.chunk_px - 1) / a.chunk_px);
}

GnWs ws_sizes(const GroupNormDesc &d, bool backward) {
    GnArgs a{};
    long long units;
    geometry(d, a, &units);
    GnWs w;
    const size_t bc = (size_t)d.batch * d.channels;
    w.part = up256(bc * a.chunks * (backward ? sizeof(float2) : sizeof(float4)));
    if (backward) {
        w.csum = up256(bc * sizeof(double2));
        w.gsum = up256((size_t)d.batch * d.groups * sizeof(float2));
    }
    return w;
}

template <typename T>
int forward_t(GnArgs &a, long long units, cudaStream_t st) {
    const unsigned grid = (unsigned)(units * a.chunks);
    gn_stats_kernel<T><<<grid, kThreads, 0, st>>>(a);
    gn_finish_stats_kernel<<<a.B * a.G, kThreads, 0, st>>>(a);
    gn_apply_kernel<T><<<grid, kThreads, 0, st>>>(a);
    SHT_CUDA_CHECK(cudaGetLastError());
    return SHTB200_OK;
}
template <typename T>
int backward_t(GnArgs &a, long long units, cudaStream_t st) {
    const unsigned grid = (unsigned)(units * a.chunks);
    gn_backward_sums_kernel<T><<<grid, kThreads, 0, st>>>(a);
    gn_finish_backward_kernel<<<a.B * a.G, kThreads, 0, st>>>(a);
    if (a.dweight || a.dbias) gn_param_grads_kernel<<<ceil_div(a.C, kThreads), kThreads, 0, st>>>(a);
    if (a.out) gn_dx_kernel<T><<<grid, kThreads, 0, st>>>(a);
    SHT_CUDA_CHECK(cudaGetLastError());
    return SHTB200_OK;
}

int check_desc(const GroupNormDesc *d) {
    if (!d) return fail(SHTB200_EINVAL, "group norm descriptor is null");
    if (d->batch < 0 || d->channels < 1 || d->groups < 1 || d->nlat < 1 || d->nlon < 1) return fail(SHTB200_EINVAL, "bad group norm shape");
    if (d->channels % d->groups) return fail(SHTB200_EINVAL, "channels must be divisible by groups");
    if (d->dtype < SHTB200_F32 || d->dtype > SHTB200_F16 || d->param_dtype < SHTB200_F32 || d->param_dtype > SHTB200_F16) return fail(SHTB200_EINVAL, "unknown element type");
    if (d->activation < SHTB200_ACT_NONE || d->activation > SHTB200_ACT_GELU) return fail(SHTB200_EINVAL, "unknown activation");
    if (!(d->eps >= 0.f)) return fail(SHTB200_EINVAL, "eps must be >= 0");
    if ((long long)d->batch * d->channels > (1LL << 24) || (long long)d->nlat * d->nlon > (1LL << 31) - 1) return fail(SHTB200_EINVAL, "group norm shape too large");
    return SHTB200_OK;
}

}  // namespace

size_t group_norm_workspace(const GroupNormDesc *d, bool backward) {
    if (check_desc(d)) return 0;
    return std::max<size_t>(ws_sizes(*d, backward).total(), 256);
}

int group_norm_forward(const GroupNormDesc *d, const void *x, const float *lat, const void *weight, const void *bias, void *y, void *stats, void *ws, size_t ws_bytes,
                       cudaStream_t st) {
    int rc = check_desc(d);
    if (rc) return rc;
    if (d->batch == 0) return SHTB200_OK;
    if (!x || !y || !stats) return fail(SHTB200_EINVAL, "null pointer");
    const GnWs w = ws_sizes(*d, false);
    if (!ws || ws_bytes < w.total()) return fail(SHTB200_EWORKSPACE, "workspace too small: need " + std::to_string(w.total()) + " bytes");
    GnArgs a{};
    long long units;
    geometry(*d, a, &units);
    a.x = x;
    a.out = y;
    a.lat = lat;
    a.weight = weight;
    a.bias = bias;
    a.stats = reinterpret_cast<float4 *>(stats);
    a.part = reinterpret_cast<float4 *>(ws);
    return d->dtype == SHTB200_F32 ? forward_t<float>(a, units, st) : d->dtype == SHTB200_BF16 ? forward_t<__nv_bfloat16>(a, units, st) : forward_t<__half>(a, units, st);
}

int group_norm_backward(const GroupNormDesc *d, const void *dy, const void *x, const float *lat, const void *weight, const void *bias, const void *stats, void *dx, void *dweight,
                        void *dbias, void *ws, size_t ws_bytes, cudaStream_t st) {
    int rc = check_desc(d);
    if (rc) return rc;
    if (d->batch == 0) return fail(SHTB200_EINVAL, "an empty batch has no gradient to compute");
    if (!x || !dy || !stats) return fail(SHTB200_EINVAL, "null pointer");
    const GnWs w = ws_sizes(*d, true);
    if (!ws || ws_bytes < w.total()) return fail(SHTB200_EWORKSPACE, "workspace too small: need " + std::to_string(w.total()) + " bytes");
    GnArgs a{};
    long long units;
    geometry(*d, a, &units);
    a.x = x;
    a.dy = dy;
    a.out = dx;
    a.lat = lat;
    a.weight = weight;
    a.bias = bias;
    a.dweight = dweight;
    a.dbias = dbias;
    a.stats = reinterpret_cast<float4 *>(const_cast<void *>(stats));
    char *base = reinterpret_cast<char *>(ws);
    a.bpart = reinterpret_cast<float2 *>(base);
    a.csum = reinterpret_cast<double2 *>(base + w.part);
    a.gsum = reinterpret_cast<float2 *>(base + w.part + w.csum);
    return d->dtype == SHTB200_F32 ? backward_t<float>(a, units, st) : d->dtype == SHTB200_BF16 ? backward_t<__nv_bfloat16>(a, units, st) : backward_t<__half>(a, units, st);
}

}  // namespace shtb200
