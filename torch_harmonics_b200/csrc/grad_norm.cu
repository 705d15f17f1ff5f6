// Global norm of a set of gradients, and clipping to a largest norm.
//
//     N = (sum over all tensors and entries |g|^2)^(1/2)   or   N = max |g|,      f = min(1, max_norm / (N + 1e-6)),      g <- f g
//
// Bound by memory: the gradients are read once for the norm; where f < 1 they are read again and written.  Where f = 1
// the second kernel ends after it has read the partial sums, so a step below the limit costs one read.  1.5 GB below the limit: 242 us on a
// B200, 6.25 TB/s (95 % of its copy rate); above it, scaled in place: 733 us, 6.2 TB/s over two reads and a write.  246 MB: 124 us in place, 126 into new
// tensors.  The largest magnitude of 1.5 GB of complex entries takes as long as their sum of squares (245 and 247 us).
//
// The tensors travel as kernel arguments (a table of pointers and lengths): no copy to the device precedes the launch,
// nothing is kept between calls, and a captured call replays with the addresses it was captured with.

#include "common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <climits>
#include <type_traits>

namespace shtb200 {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxTensors = 896;         // tensors of one launch: the table has to fit into 32,764 bytes of kernel arguments
constexpr int kFewTensors = 64;          // a small table for few: copying 30 KB of arguments twice a call costs more than scaling a small network (8.4 us on the device, with it 4.8)
constexpr int kUnitBytes = 32768;        // one unit of work: 8 vectors of 16 bytes a thread, all of them in flight before the first is used
constexpr int kVectors = kUnitBytes / 16 / kThreads;
constexpr int kScaleVectors = 4;         // (eight in flight spill: the scaling kernel also holds the addresses it writes to)
constexpr int kBlocksPerSm = 4;
constexpr int kMaxBlocks = 148 * kBlocksPerSm;

template <int N> struct Table {
    const void *src[N];
    void *dst[N];
    long long n[N];                      // values (a complex entry is two)
    int first[N + 1];                    // first unit of work of every tensor
    unsigned char dtype[N];
    int count;
};
static_assert(sizeof(Table<kMaxTensors>) + 64 <= 32764, "kernel arguments");

__host__ __device__ constexpr int unit_values(int dtype) { return dtype == SHTB200_BF16 || dtype == SHTB200_F16 ? kUnitBytes / 2 : kUnitBytes / 4; }

constexpr long long values_of(long long numel, int dtype) { return numel * (dtype == SHTB200_C64 ? 2 : 1); }
constexpr long long units_of(long long numel, int dtype) { return (values_of(numel, dtype) + unit_values(dtype) - 1) / unit_values(dtype); }

template <typename T> struct Pack {  // 16 bytes of values
    static constexpr int n = 16 / sizeof(T);
    uint4 v;
    __device__ __forceinline__ float get(int i) const;
    __device__ __forceinline__ void scale(float f);
};
template <> __device__ __forceinline__ float Pack<float>::get(int i) const { return __uint_as_float(i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w); }
template <> __device__ __forceinline__ float Pack<__nv_bfloat16>::get(int i) const {
    const unsigned u = i < 2 ? v.x : i < 4 ? v.y : i < 6 ? v.z : v.w;
    return __uint_as_float(i & 1 ? u & 0xffff0000u : u << 16);
}
template <> __device__ __forceinline__ float Pack<__half>::get(int i) const {
    const unsigned u = i < 2 ? v.x : i < 4 ? v.y : i < 6 ? v.z : v.w;
    return __half2float(__ushort_as_half((unsigned short)(i & 1 ? u >> 16 : u & 0xffffu)));
}
__device__ __forceinline__ float load_one(const float *p) { return *p; }
__device__ __forceinline__ float load_one(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
__device__ __forceinline__ float load_one(const __half *p) { return __half2float(*p); }
__device__ __forceinline__ void store_one(float *p, float v) { *p = v; }
__device__ __forceinline__ void store_one(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void store_one(__half *p, float v) { *p = __float2half_rn(v); }
template <> __device__ __forceinline__ void Pack<float>::scale(float f) {
    v = make_uint4(__float_as_uint(get(0) * f), __float_as_uint(get(1) * f), __float_as_uint(get(2) * f), __float_as_uint(get(3) * f));
}
template <> __device__ __forceinline__ void Pack<__nv_bfloat16>::scale(float f) {
    __nv_bfloat162 r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __floats2bfloat162_rn(get(2 * i) * f, get(2 * i + 1) * f);
    v = *reinterpret_cast<uint4 *>(r);
}
template <> __device__ __forceinline__ void Pack<__half>::scale(float f) {
    __half2 r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __floats2half2_rn(get(2 * i) * f, get(2 * i + 1) * f);
    v = *reinterpret_cast<uint4 *>(r);
}

// Last tensor that starts at or before `unit`, searched from `lo` on (the units of a block ascend or descend).
template <int N> __device__ __forceinline__ int tensor_of(const Table<N> &t, int unit, int lo, int hi) {
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (t.first[mid] <= unit) lo = mid;
        else hi = mid;
    }
    return lo;
}

// The launches of a call may begin while the one before ends; each waits for its results (and so for all before) before it reads anything.
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_begin() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// (fmax drops a NaN; the largest magnitude has to keep it)
__device__ __forceinline__ double larger(double a, double b) { return (b > a || b != b) ? b : a; }

template <int kind> __device__ double block_join(double v) {
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

// The squares are added in float64: their range (1e-45^2 to 3e38^2) is float64's, and no sum of any length loses anything.
// pairs: entries are complex, their magnitude joins two values (for the largest magnitude; a sum of squares need not know).
template <int kind, typename T>
__device__ __forceinline__ void gather_unit(const T *p, int n, bool pairs, double acc[2]) {
    const int head = min(n, (int)((16 - ((uintptr_t)p & 15)) & 15) / (int)sizeof(T));
    if (kind == SHTB200_NORM_INF && pairs) {  // float pairs, 8-byte aligned: vector or not, a pair is never split
        for (int i = 2 * threadIdx.x; i < n; i += 2 * kThreads) {
            const double re = load_one(p + i), im = load_one(p + i + 1);
            acc[0] = larger(acc[0], fma(re, re, im * im));
        }
        return;
    }
    const uint4 *q = reinterpret_cast<const uint4 *>(p + head);
    const int vecs = (n - head) / Pack<T>::n;
    Pack<T> v[kVectors];
#pragma unroll
    for (int k = 0; k < kVectors; ++k) {
        const int i = threadIdx.x + k * kThreads;
        v[k].v = i < vecs ? __ldg(q + i) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int k = 0; k < kVectors; ++k)
#pragma unroll
        for (int i = 0; i < Pack<T>::n; ++i) {
            const double x = v[k].get(i);
            acc[i & 1] = kind == SHTB200_NORM_INF ? larger(acc[i & 1], fabs(x)) : fma(x, x, acc[i & 1]);
        }
    const int rest = n - vecs * Pack<T>::n;  // values before and behind the vectors: fewer than 2 Pack::n
    if ((int)threadIdx.x < rest) {
        const double x = load_one(p + ((int)threadIdx.x < head ? threadIdx.x : vecs * Pack<T>::n + threadIdx.x));
        acc[0] = kind == SHTB200_NORM_INF ? larger(acc[0], fabs(x)) : fma(x, x, acc[0]);
    }
}

// Partial sums of squares (or largest magnitudes, squared): one float64 value a block.
template <int kind, int N>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm) norm_partial_kernel(const __grid_constant__ Table<N> t, double *part) {
    wait_for_previous();
    let_next_begin();
    double acc[2] = {0., 0.}, pair[2] = {0., 0.};
    const int units = t.first[t.count];
    int k = 0;
    for (int u = blockIdx.x; u < units; u += gridDim.x) {
        k = tensor_of(t, u, k, t.count);
        const int dt = t.dtype[k], uv = unit_values(dt);
        const long long lo = (long long)(u - t.first[k]) * uv;
        const int n = (int)min((long long)uv, t.n[k] - lo);
        if (dt == SHTB200_BF16) gather_unit<kind>(reinterpret_cast<const __nv_bfloat16 *>(t.src[k]) + lo, n, false, acc);
        else if (dt == SHTB200_F16) gather_unit<kind>(reinterpret_cast<const __half *>(t.src[k]) + lo, n, false, acc);
        else if (kind == SHTB200_NORM_INF && dt == SHTB200_C64) gather_unit<kind>(reinterpret_cast<const float *>(t.src[k]) + lo, n, true, pair);
        else gather_unit<kind>(reinterpret_cast<const float *>(t.src[k]) + lo, n, false, acc);
    }
    double v = kind == SHTB200_NORM_INF ? larger(acc[0], acc[1]) : acc[0] + acc[1];
    if (kind == SHTB200_NORM_INF) v = larger(v * v, pair[0]);
    v = block_join<kind>(v);
    if (threadIdx.x == 0) part[blockIdx.x] = v;
}

template <int kind> __device__ float total_norm(const double *part, int nparts) {
    double acc = 0.;
    for (int i = threadIdx.x; i < nparts; i += kThreads) acc = kind == SHTB200_NORM_INF ? larger(acc, part[i]) : acc + part[i];
    return (float)sqrt(block_join<kind>(acc));
}

template <int kind>
__global__ void __launch_bounds__(kThreads) norm_total_kernel(const double *part, int nparts, float *norm) {
    wait_for_previous();
    const float v = total_norm<kind>(part, nparts);
    if (threadIdx.x == 0) *norm = v;
}

template <typename T>
__device__ __forceinline__ void scale_unit(const T *p, T *d, int n, float f) {
    if ((((uintptr_t)p ^ (uintptr_t)d) & 15) != 0) {  // no vector is aligned on both sides
        for (int i = threadIdx.x; i < n; i += kThreads) store_one(d + i, load_one(p + i) * f);
        return;
    }
    const int head = min(n, (int)((16 - ((uintptr_t)p & 15)) & 15) / (int)sizeof(T));
    const uint4 *q = reinterpret_cast<const uint4 *>(p + head);
    uint4 *o = reinterpret_cast<uint4 *>(d + head);
    const int vecs = (n - head) / Pack<T>::n;
#pragma unroll 1
    for (int r = 0; r < kVectors; r += kScaleVectors) {
        Pack<T> v[kScaleVectors];
#pragma unroll
        for (int k = 0; k < kScaleVectors; ++k) {
            const int i = threadIdx.x + (r + k) * kThreads;
            v[k].v = i < vecs ? q[i] : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int k = 0; k < kScaleVectors; ++k) {
            const int i = threadIdx.x + (r + k) * kThreads;
            v[k].scale(f);
            if (i < vecs) o[i] = v[k].v;
        }
    }
    const int rest = n - vecs * Pack<T>::n;
    if ((int)threadIdx.x < rest) {
        const int i = (int)threadIdx.x < head ? threadIdx.x : vecs * Pack<T>::n + threadIdx.x;
        store_one(d + i, load_one(p + i) * f);
    }
}

// The units are taken from the end: what the norm has read last is still in L2.
template <int kind, int N>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm) scale_kernel(const __grid_constant__ Table<N> t, const double *part, int nparts, float max_norm, float *norm) {
    wait_for_previous();
    float total;
    if (part) {
        total = total_norm<kind>(part, nparts);
        if (blockIdx.x == 0 && threadIdx.x == 0) *norm = total;
    } else {
        total = *norm;
    }
    float f = max_norm / (total + 1e-6f);
    if (f > 1.f) f = 1.f;  // (a NaN stays one)
    const int units = t.first[t.count];
    int k = t.count - 1;
    for (int u = units - 1 - (int)blockIdx.x; u >= 0; u -= gridDim.x) {
        k = tensor_of(t, u, 0, k + 1);
        if (f == 1.f && t.dst[k] == t.src[k]) continue;
        const int dt = t.dtype[k], uv = unit_values(dt);
        const long long lo = (long long)(u - t.first[k]) * uv;
        const int n = (int)min((long long)uv, t.n[k] - lo);
        if (dt == SHTB200_BF16) scale_unit(reinterpret_cast<const __nv_bfloat16 *>(t.src[k]) + lo, reinterpret_cast<__nv_bfloat16 *>(t.dst[k]) + lo, n, f);
        else if (dt == SHTB200_F16) scale_unit(reinterpret_cast<const __half *>(t.src[k]) + lo, reinterpret_cast<__half *>(t.dst[k]) + lo, n, f);
        else scale_unit(reinterpret_cast<const float *>(t.src[k]) + lo, reinterpret_cast<float *>(t.dst[k]) + lo, n, f);
    }
}

size_t bytes_of(int dtype) { return dtype == SHTB200_C64 ? 8 : dtype == SHTB200_F32 ? 4 : 2; }

// norm: read by every block, and in a clipping written by one
int check_tensors(int count, const void *const *src, void *const *dst, const long long *numel, const int *dtype, const float *norm, bool norm_written) {
    if (count < 0 || (count > 0 && (!src || !numel || !dtype))) return fail(SHTB200_EINVAL, "bad tensor list");
    struct Range {
        uintptr_t lo, hi;
        bool written;
    };
    std::vector<Range> r;
    long long units = 0;  // of a launch: they are counted in 32 bits, with room for a step beyond the last
    int in_launch = 0;
    for (int i = 0; i < count; ++i) {
        if (dtype[i] < SHTB200_F32 || dtype[i] > SHTB200_C64) return fail(SHTB200_EINVAL, "unknown element type");
        if (numel[i] < 0 || numel[i] > (1LL << 44)) return fail(SHTB200_EINVAL, "bad tensor length");
        if (numel[i] == 0) continue;
        if (in_launch++ == kMaxTensors) {
            units = 0;
            in_launch = 1;
        }
        units += units_of(numel[i], dtype[i]);
        if (units > INT_MAX - kMaxBlocks) return fail(SHTB200_EINVAL, "too many entries: at most 2^31 pieces of 32 KB in " + std::to_string(kMaxTensors) + " tensors");
        if (!src[i] || (dst && !dst[i])) return fail(SHTB200_EINVAL, "null pointer");
        const size_t es = std::min<size_t>(bytes_of(dtype[i]), 4), bytes = bytes_of(dtype[i]) * (size_t)numel[i];
        if ((uintptr_t)src[i] % es || (dst && (uintptr_t)dst[i] % es)) return fail(SHTB200_EINVAL, "a tensor is not aligned to its element type");
        if (dst) {
            r.push_back({(uintptr_t)dst[i], (uintptr_t)dst[i] + bytes, true});
            if (src[i] != dst[i]) r.push_back({(uintptr_t)src[i], (uintptr_t)src[i] + bytes, false});
        }
    }
    // Two tensors that share memory would be scaled twice, in no fixed order, and a norm among them read before or after it is scaled.
    if (dst) r.push_back({(uintptr_t)norm, (uintptr_t)norm + sizeof(float), norm_written});
    std::sort(r.begin(), r.end(), [](const Range &a, const Range &b) { return a.lo < b.lo; });
    uintptr_t end_any = 0, end_written = 0;
    for (const Range &x : r) {
        if (x.lo < (x.written ? end_any : end_written)) return fail(SHTB200_EINVAL, "two of the tensors to be scaled, or one and the norm, share memory");
        end_any = std::max(end_any, x.hi);
        if (x.written) end_written = std::max(end_written, x.hi);
    }
    return SHTB200_OK;
}

}  // namespace

size_t grad_norm_workspace(int count) { return sizeof(double) * (size_t)kMaxBlocks * std::max(1, ceil_div(std::max(count, 0), kMaxTensors)); }

namespace {

template <typename... P> int launch(void (*kernel)(P...), int grid, cudaStream_t st, std::remove_const_t<P> &...args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    void *pointers[] = {&args...};  // (the table is not copied on the way)
    SHT_CUDA_CHECK(cudaLaunchKernelExC(&cfg, (const void *)kernel, pointers));
    return SHTB200_OK;
}

// A list of tensors, kMaxTensors a launch; empty tensors are left out.
struct List {
    const void *const *src;
    void *const *dst;
    const long long *numel;
    const int *dtype;
    std::vector<int> index;  // of the tensors that are not empty
    int launches() const { return ceil_div((int)index.size(), kMaxTensors); }
    int count(int launch) const { return std::min(kMaxTensors, (int)index.size() - launch * kMaxTensors); }
    template <int N> void fill(int launch, Table<N> *t) const {
        t->count = count(launch);
        t->first[0] = 0;
        for (int k = 0; k < t->count; ++k) {
            const int i = index[(size_t)launch * kMaxTensors + k];
            t->src[k] = src[i];
            t->dst[k] = dst ? dst[i] : nullptr;
            t->n[k] = values_of(numel[i], dtype[i]);
            t->dtype[k] = (unsigned char)dtype[i];
            t->first[k + 1] = t->first[k] + (int)units_of(numel[i], dtype[i]);
        }
    }
};
List make_list(int count, const void *const *src, void *const *dst, const long long *numel, const int *dtype) {
    List l{src, dst, numel, dtype, {}};
    l.index.reserve((size_t)std::max(count, 0));
    for (int i = 0; i < count; ++i)
        if (numel[i]) l.index.push_back(i);
    return l;
}

template <int N> int launch_partials(const List &l, int i, int kind, double *part, int *nparts, cudaStream_t st) {
    Table<N> t;
    l.fill(i, &t);
    const int blocks = std::min(kMaxBlocks, t.first[t.count]);
    double *to = part + *nparts;
    const int rc = launch(kind == SHTB200_NORM_INF ? norm_partial_kernel<SHTB200_NORM_INF, N> : norm_partial_kernel<SHTB200_NORM_L2, N>, blocks, st, t, to);
    *nparts += blocks;
    return rc;
}
int launch_partials(const List &l, int kind, double *part, int *nparts, cudaStream_t st) {
    *nparts = 0;
    int rc = SHTB200_OK;
    for (int i = 0; i < l.launches() && !rc; ++i)
        rc = l.count(i) <= kFewTensors ? launch_partials<kFewTensors>(l, i, kind, part, nparts, st) : launch_partials<kMaxTensors>(l, i, kind, part, nparts, st);
    return rc;
}
template <int N> int launch_scale(const List &l, int i, int kind, const double *part, int nparts, float max_norm, float *norm, cudaStream_t st) {
    Table<N> t;
    l.fill(i, &t);
    const int blocks = std::min(kMaxBlocks, t.first[t.count]);
    return launch(kind == SHTB200_NORM_INF ? scale_kernel<SHTB200_NORM_INF, N> : scale_kernel<SHTB200_NORM_L2, N>, blocks, st, t, part, nparts, max_norm, norm);
}
int launch_scale(const List &l, int kind, const double *part, int nparts, float max_norm, float *norm, cudaStream_t st) {
    int rc = SHTB200_OK;
    for (int i = 0; i < l.launches() && !rc; ++i)
        rc = l.count(i) <= kFewTensors ? launch_scale<kFewTensors>(l, i, kind, part, nparts, max_norm, norm, st)
                                       : launch_scale<kMaxTensors>(l, i, kind, part, nparts, max_norm, norm, st);
    return rc;
}
int launch_total(const double *part, int nparts, int kind, float *norm, cudaStream_t st) {
    return launch(kind == SHTB200_NORM_INF ? norm_total_kernel<SHTB200_NORM_INF> : norm_total_kernel<SHTB200_NORM_L2>, 1, st, part, nparts, norm);
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
    if (rc || (rc = check_tensors(count, src, nullptr, numel, dtype, norm, true))) return rc;
    double *part = reinterpret_cast<double *>(ws);
    int nparts = 0;
    if ((rc = launch_partials(make_list(count, src, nullptr, numel, dtype), kind, part, &nparts, st))) return rc;
    return launch_total(part, nparts, kind, norm, st);
}

int clip_grads(int count, const void *const *src, void *const *dst, const long long *numel, const int *dtype, int kind, float max_norm, float *norm, void *ws, size_t ws_bytes,
               cudaStream_t st) {
    if (!(max_norm >= 0.f)) return fail(SHTB200_EINVAL, "max_norm must be >= 0");
    int rc = check_norm(count, kind, norm, ws, ws_bytes);
    if (rc || (rc = check_tensors(count, src, dst, numel, dtype, norm, true))) return rc;
    const List l = make_list(count, src, dst, numel, dtype);
    double *part = reinterpret_cast<double *>(ws);
    int nparts = 0;
    if ((rc = launch_partials(l, kind, part, &nparts, st))) return rc;
    return l.index.empty() ? launch_total(part, nparts, kind, norm, st) : launch_scale(l, kind, part, nparts, max_norm, norm, st);
}

int scale_grads(int count, const void *const *src, void *const *dst, const long long *numel, const int *dtype, float max_norm, const float *norm, cudaStream_t st) {
    if (!(max_norm >= 0.f)) return fail(SHTB200_EINVAL, "max_norm must be >= 0");
    if (!norm) return fail(SHTB200_EINVAL, "null pointer");
    int rc = check_tensors(count, src, dst, numel, dtype, norm, false);
    if (rc) return rc;
    return launch_scale(make_list(count, src, dst, numel, dtype), SHTB200_NORM_L2, nullptr, 0, max_norm, const_cast<float *>(norm), st);
}

}  // namespace shtb200
