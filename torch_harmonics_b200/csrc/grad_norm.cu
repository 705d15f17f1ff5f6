// Global norm of a set of gradients, and clipping to a largest norm.
//
//     N = (sum over all tensors and entries |g|^2)^(1/2)   or   N = max |g|,      f = min(1, max_norm / (N + 1e-6)),      g <- f g
//
// Bound by memory: the gradients are read once for the norm; where f < 1 they are read again and written.  Where f = 1
// the second kernel ends after it has read the partial sums, so a step below the limit costs one read.
//
// The tensors travel as kernel arguments (a table of pointers and lengths): no copy to the device precedes the launch,
// nothing is kept between calls, and a captured call replays with the addresses it was captured with.

#include "common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

namespace shtb200 {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxTensors = 896;         // tensors of one launch: the table has to fit into 32,764 bytes of kernel arguments
constexpr int kChunk = 8192;             // values of one unit of work
constexpr int kMaxBlocks = 148 * 4;

struct Table {
    const void *src[kMaxTensors];
    void *dst[kMaxTensors];
    long long n[kMaxTensors];            // values (a complex entry is two)
    int first[kMaxTensors + 1];          // first unit of work of every tensor
    unsigned char dtype[kMaxTensors];
    int count = 0;
};
static_assert(sizeof(Table) + 64 <= 32764, "kernel arguments");

__device__ __forceinline__ float load_value(const void *p, int dtype, long long i) {
    if (dtype == SHTB200_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(p)[i]);
    if (dtype == SHTB200_F16) return __half2float(reinterpret_cast<const __half *>(p)[i]);
    return reinterpret_cast<const float *>(p)[i];
}
__device__ __forceinline__ void store_value(void *p, int dtype, long long i, float v) {
    if (dtype == SHTB200_BF16) reinterpret_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
    else if (dtype == SHTB200_F16) reinterpret_cast<__half *>(p)[i] = __float2half_rn(v);
    else reinterpret_cast<float *>(p)[i] = v;
}

__device__ __forceinline__ int tensor_of(const Table &t, int unit) {
    int lo = 0, hi = t.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (t.first[mid] <= unit) lo = mid;
        else hi = mid;
    }
    return lo;
}

// (fmax drops a NaN; the largest magnitude has to keep it)
__device__ __forceinline__ double larger(double a, double b) { return (b > a || b != b) ? b : a; }

__device__ double block_join(double v, int kind) {
    __shared__ double s[kThreads / 32];
    for (int o = 16; o; o >>= 1) {
        const double u = __shfl_xor_sync(0xffffffffu, v, o);
        v = kind == SHTB200_NORM_INF ? larger(v, u) : v + u;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    double t = s[0];
    for (int i = 1; i < kThreads / 32; ++i) t = kind == SHTB200_NORM_INF ? larger(t, s[i]) : t + s[i];
    return t;
}

// partial sums of squares (or largest squared magnitudes): one float64 value a block
__global__ void __launch_bounds__(kThreads) norm_partial_kernel(const __grid_constant__ Table t, int kind, double *part) {
    double acc = 0.;
    const int units = t.first[t.count];
    for (int u = blockIdx.x; u < units; u += gridDim.x) {
        const int k = tensor_of(t, u);
        const long long lo = (long long)(u - t.first[k]) * kChunk, hi = min(lo + kChunk, t.n[k]);
        const int dt = t.dtype[k];
        if (kind == SHTB200_NORM_INF && dt == SHTB200_C64) {
            for (long long i = lo + 2 * threadIdx.x; i < hi; i += 2 * kThreads) {
                const double re = load_value(t.src[k], dt, i), im = load_value(t.src[k], dt, i + 1);
                acc = larger(acc, re * re + im * im);
            }
        } else {
            for (long long i = lo + threadIdx.x; i < hi; i += kThreads) {
                const double v = load_value(t.src[k], dt, i);
                acc = kind == SHTB200_NORM_INF ? larger(acc, v * v) : fma(v, v, acc);
            }
        }
    }
    acc = block_join(acc, kind);
    if (threadIdx.x == 0) part[blockIdx.x] = acc;
}

__device__ float total_norm(const double *part, int nparts, int kind) {
    double acc = 0.;
    for (int i = threadIdx.x; i < nparts; i += kThreads) acc = kind == SHTB200_NORM_INF ? larger(acc, part[i]) : acc + part[i];
    return (float)sqrt(block_join(acc, kind));
}

__global__ void __launch_bounds__(kThreads) norm_total_kernel(const double *part, int nparts, int kind, float *norm) {
    const float v = total_norm(part, nparts, kind);
    if (threadIdx.x == 0) *norm = v;
}

__global__ void __launch_bounds__(kThreads) scale_kernel(const __grid_constant__ Table t, const double *part, int nparts, int kind, float max_norm, float *norm) {
    float total;
    if (part) {
        total = total_norm(part, nparts, kind);
        if (blockIdx.x == 0 && threadIdx.x == 0) *norm = total;
    } else {
        total = *norm;
    }
    float f = max_norm / (total + 1e-6f);
    if (f > 1.f) f = 1.f;  // (a NaN stays one)
    const int units = t.first[t.count];
    for (int u = blockIdx.x; u < units; u += gridDim.x) {
        const int k = tensor_of(t, u);
        if (f == 1.f && t.dst[k] == t.src[k]) continue;
        const long long lo = (long long)(u - t.first[k]) * kChunk, hi = min(lo + kChunk, t.n[k]);
        const int dt = t.dtype[k];
        for (long long i = lo + threadIdx.x; i < hi; i += kThreads) store_value(t.dst[k], dt, i, load_value(t.src[k], dt, i) * f);
    }
}

size_t bytes_of(int dtype) { return dtype == SHTB200_C64 ? 8 : dtype == SHTB200_F32 ? 4 : 2; }

int check_tensors(int count, const void *const *src, void *const *dst, const long long *numel, const int *dtype) {
    if (count < 0 || (count > 0 && (!src || !numel || !dtype))) return fail(SHTB200_EINVAL, "bad tensor list");
    struct Range {
        uintptr_t lo, hi;
        bool written;
    };
    std::vector<Range> r;
    for (int i = 0; i < count; ++i) {
        if (dtype[i] < SHTB200_F32 || dtype[i] > SHTB200_C64) return fail(SHTB200_EINVAL, "unknown element type");
        if (numel[i] < 0 || numel[i] > (1LL << 40) / std::max(count, 1)) return fail(SHTB200_EINVAL, "bad tensor length");
        if (numel[i] == 0) continue;
        if (!src[i] || (dst && !dst[i])) return fail(SHTB200_EINVAL, "null pointer");
        const size_t es = std::min<size_t>(bytes_of(dtype[i]), 4), bytes = bytes_of(dtype[i]) * (size_t)numel[i];
        if ((uintptr_t)src[i] % es || (dst && (uintptr_t)dst[i] % es)) return fail(SHTB200_EINVAL, "a tensor is not aligned to its element type");
        if (dst) {
            r.push_back({(uintptr_t)dst[i], (uintptr_t)dst[i] + bytes, true});
            if (src[i] != dst[i]) r.push_back({(uintptr_t)src[i], (uintptr_t)src[i] + bytes, false});
        }
    }
    // Two tensors that share memory would be scaled twice, in no fixed order.
    std::sort(r.begin(), r.end(), [](const Range &a, const Range &b) { return a.lo < b.lo; });
    uintptr_t end_any = 0, end_written = 0;
    for (const Range &x : r) {
        if (x.lo < (x.written ? end_any : end_written)) return fail(SHTB200_EINVAL, "two of the tensors to be scaled share memory");
        end_any = std::max(end_any, x.hi);
        if (x.written) end_written = std::max(end_written, x.hi);
    }
    return SHTB200_OK;
}

}  // namespace

size_t grad_norm_workspace(int count) { return sizeof(double) * (size_t)kMaxBlocks * std::max(1, ceil_div(std::max(count, 0), kMaxTensors)); }

namespace {

// The tables of a list of tensors, kMaxTensors a launch; empty tensors are left out.
std::vector<Table> make_tables(int count, const void *const *src, void *const *dst, const long long *numel, const int *dtype) {
    std::vector<Table> tables;
    long long units = 0;
    for (int i = 0; i < count; ++i) {
        if (numel[i] == 0) continue;
        const long long n = numel[i] * (dtype[i] == SHTB200_C64 ? 2 : 1), u = (n + kChunk - 1) / kChunk;
        if (tables.empty() || tables.back().count == kMaxTensors) {
            tables.emplace_back();
            units = 0;
        }
        Table &t = tables.back();
        const int k = t.count++;
        t.src[k] = src[i];
        t.dst[k] = dst ? dst[i] : nullptr;
        t.n[k] = n;
        t.dtype[k] = (unsigned char)dtype[i];
        t.first[k] = (int)units;
        units += u;
        t.first[k + 1] = (int)units;
    }
    return tables;
}

int blocks_of(const Table &t) { return std::min(kMaxBlocks, t.first[t.count]); }

int launch_partials(const std::vector<Table> &tables, int kind, double *part, cudaStream_t st) {
    int nparts = 0;
    for (const Table &t : tables) {
        norm_partial_kernel<<<blocks_of(t), kThreads, 0, st>>>(t, kind, part + nparts);
        nparts += blocks_of(t);
    }
    return nparts;
}

int check_norm(int count, int kind, const float *norm, const void *ws, size_t ws_bytes) {
    if (kind != SHTB200_NORM_L2 && kind != SHTB200_NORM_INF) return fail(SHTB200_EINVAL, "unknown norm");
    if (!norm) return fail(SHTB200_EINVAL, "null pointer");
    if (!ws || ws_bytes < grad_norm_workspace(count)) return fail(SHTB200_EWORKSPACE, "workspace too small: need " + std::to_string(grad_norm_workspace(count)) + " bytes");
    if ((uintptr_t)ws & 7) return fail(SHTB200_EINVAL, "workspace must be 8-byte aligned");
    return SHTB200_OK;
}

}  // namespace

int grad_norm(int count, const void *const *src, const long long *numel, const int *dtype, int kind, float *norm, void *ws, size_t ws_bytes, cudaStream_t st) {
    int rc = check_norm(count, kind, norm, ws, ws_bytes);
    if (rc || (rc = check_tensors(count, src, nullptr, numel, dtype))) return rc;
    const std::vector<Table> tables = make_tables(count, src, nullptr, numel, dtype);
    double *part = reinterpret_cast<double *>(ws);
    const int nparts = launch_partials(tables, kind, part, st);
    norm_total_kernel<<<1, kThreads, 0, st>>>(part, nparts, kind, norm);
    SHT_CUDA_CHECK(cudaGetLastError());
    return SHTB200_OK;
}

int clip_grads(int count, const void *const *src, void *const *dst, const long long *numel, const int *dtype, int kind, float max_norm, float *norm, void *ws, size_t ws_bytes,
               cudaStream_t st) {
    if (!(max_norm >= 0.f)) return fail(SHTB200_EINVAL, "max_norm must be >= 0");
    int rc = check_norm(count, kind, norm, ws, ws_bytes);
    if (rc || (rc = check_tensors(count, src, dst, numel, dtype))) return rc;
    const std::vector<Table> tables = make_tables(count, src, dst, numel, dtype);
    double *part = reinterpret_cast<double *>(ws);
    const int nparts = launch_partials(tables, kind, part, st);
    if (tables.empty()) norm_total_kernel<<<1, kThreads, 0, st>>>(part, nparts, kind, norm);
    for (const Table &t : tables) scale_kernel<<<blocks_of(t), kThreads, 0, st>>>(t, part, nparts, kind, max_norm, norm);
    SHT_CUDA_CHECK(cudaGetLastError());
    return SHTB200_OK;
}

int scale_grads(int count, const void *const *src, void *const *dst, const long long *numel, const int *dtype, float max_norm, const float *norm, cudaStream_t st) {
    if (!(max_norm >= 0.f)) return fail(SHTB200_EINVAL, "max_norm must be >= 0");
    if (!norm) return fail(SHTB200_EINVAL, "null pointer");
    int rc = check_tensors(count, src, dst, numel, dtype);
    if (rc) return rc;
    for (const Table &t : make_tables(count, src, dst, numel, dtype)) scale_kernel<<<blocks_of(t), kThreads, 0, st>>>(t, nullptr, 0, 0, max_norm, const_cast<float *>(norm));
    SHT_CUDA_CHECK(cudaGetLastError());
    return SHTB200_OK;
}

}  // namespace shtb200
