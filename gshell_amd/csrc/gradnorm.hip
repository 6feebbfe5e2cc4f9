// GS_CXXFLAGS: -Xclang -target-feature -Xclang -packed-fp32-ops
// Global norm of a list of gradients and clipping by it (gfx950).
//
//     n = (sum_i |g_i|^p)^(1/p),  p = 1, 2, inf          out_i = g_i min(1, max_norm / (n + 1e-6))
//
// Two launches for a list of up to TABLE tensors (their addresses travel as kernel arguments): the first adds up one partial sum a workgroup, in 64 bits (a square of an
// fp32 value neither overflows nor vanishes there, and the order of the sum no longer shows); in the second every workgroup adds the partial sums for itself, in
// the same order, and scales its share of the elements.  Bound by memory: each gradient is read once, then read again and written.  The second launch walks the
// elements from the end: what the first has read last is still in the 256 MB cache.  In place and with a factor of one it writes nothing.
//
// Measured, GPU time of both launches, new tensors for the result: 30 fp32 tensors of 22 million elements 58 us (264 MB read and written, 4.5 TB/s; a copy of
// 1 GB reaches 5.2 TB/s), 300 bf16 tensors of 600 million 785 us (3.6 GB, 4.6 TB/s), 16 fp32 tensors of half a million 10 us (two launches, each as long as its
// slowest chain of loads).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <new>
#include <vector>

#include "../../include/gshell_hip.h"
#include "common.hpp"

namespace {

typedef __bf16 bf16;
typedef _Float16 f16;

constexpr int TABLE = 120;          // tensors a launch: the table stays below the 4 KB of kernel arguments
constexpr int THREADS = 256, CHUNK_BYTES = THREADS * 16 * 2;          // two loads of 16 bytes a thread: 785 us for the 600 million, four 815, eight more; 10.1 us for the half million, four 11.0
constexpr int MAX_BLOCKS = 2048;          // eight workgroups a CU; 1024 789 us, 4096 810

struct Table {
    const void* src[TABLE];
    void* dst[TABLE];
    int64_t numel[TABLE];
    uint32_t first[TABLE + 1];          // first chunk of each tensor
    uint8_t type[TABLE];
    int n;
};

template <typename T> struct __attribute__((packed)) Pack { T v[16 / sizeof(T)]; };

__device__ __forceinline__ int find(const uint32_t* first, int n, uint32_t chunk) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (first[mid] <= chunk) lo = mid;
        else hi = mid;
    }
    return lo;
}

enum { NORM_2 = 0, NORM_1 = 1, NORM_INF = 2 };
__device__ __forceinline__ double larger(double a, double b) { return a != a ? a : b != b ? b : a > b ? a : b; }          // a NaN stays
template <int P> __device__ __forceinline__ double add(double s, float g) {
    const double v = (double)g;
    return P == NORM_2 ? __builtin_fma(v, v, s) : P == NORM_1 ? s + fabs(v) : larger(s, fabs(v));
}
template <int P> __device__ __forceinline__ double join(double a, double b) { return P == NORM_INF ? larger(a, b) : a + b; }

template <int P> __device__ __forceinline__ double block_join(double s, double* tmp) {
#pragma unroll
    for (int d = 32; d; d >>= 1) s = join<P>(s, __shfl_xor(s, d));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) tmp[threadIdx.x >> 6] = s;
    __syncthreads();
    return join<P>(join<P>(tmp[0], tmp[1]), join<P>(tmp[2], tmp[3]));
}

template <typename T, int P> __device__ __forceinline__ double chunk_sum(const T* p, int64_t n, double s) {
    constexpr int VEC = 16 / sizeof(T), ROUNDS = CHUNK_BYTES / (THREADS * 16);
    if (n >= (int64_t)THREADS * VEC * ROUNDS) {
        Pack<T> q[ROUNDS];
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) q[r] = *(const Pack<T>*)(p + (r * THREADS + threadIdx.x) * VEC);
        double part[ROUNDS];
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) {
            part[r] = 0.0;
#pragma unroll
            for (int k = 0; k < VEC; ++k) part[r] = add<P>(part[r], (float)q[r].v[k]);
        }
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) s = join<P>(s, part[r]);
    } else {
        for (int i = threadIdx.x; i < n; i += THREADS) s = add<P>(s, (float)p[i]);
    }
    return s;
}

template <int P> __global__ void __launch_bounds__(THREADS) k_norm_partials(Table T, double* part) {
    __shared__ double tmp[4];
    const uint32_t chunks = T.first[T.n];
    double s = 0.0;
    for (uint32_t c = blockIdx.x; c < chunks; c += gridDim.x) {
        const int t = find(T.first, T.n, c);
        const int64_t per = T.type[t] == 0 ? CHUNK_BYTES / 4 : CHUNK_BYTES / 2, at = (int64_t)(c - T.first[t]) * per, left = T.numel[t] - at, n = left < per ? left : per;
        if (T.type[t] == 0) s = chunk_sum<float, P>((const float*)T.src[t] + at, n, s);
        else if (T.type[t] == 1) s = chunk_sum<bf16, P>((const bf16*)T.src[t] + at, n, s);
        else s = chunk_sum<f16, P>((const f16*)T.src[t] + at, n, s);
    }
    s = block_join<P>(s, tmp);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}

template <int P> __device__ __forceinline__ float total_norm(const double* part, int n, double* tmp) {
    double s = 0.0;
    for (int i = threadIdx.x; i < n; i += THREADS) s = join<P>(s, part[i]);
    s = block_join<P>(s, tmp);
    return (float)(P == NORM_2 ? sqrt(s) : s);
}

template <typename T> __device__ __forceinline__ void chunk_scale(const T* p, T* q, int64_t n, float coef) {
    constexpr int VEC = 16 / sizeof(T), ROUNDS = CHUNK_BYTES / (THREADS * 16);
    if (n >= (int64_t)THREADS * VEC * ROUNDS) {
        Pack<T> v[ROUNDS];
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) v[r] = *(const Pack<T>*)(p + (r * THREADS + threadIdx.x) * VEC);
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) {
#pragma unroll
            for (int k = 0; k < VEC; ++k) v[r].v[k] = (T)((float)v[r].v[k] * coef);
            *(Pack<T>*)(q + (r * THREADS + threadIdx.x) * VEC) = v[r];
        }
    } else {
        for (int i = threadIdx.x; i < n; i += THREADS) q[i] = (T)((float)p[i] * coef);
    }
}

template <int P> __global__ void __launch_bounds__(THREADS) k_norm_scale(Table T, const double* part, int parts, float max_norm, float* norm_out) {
    __shared__ double tmp[4];
    const float norm = total_norm<P>(part, parts, tmp);
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = norm;
    float coef = max_norm / (norm + 1e-6f);
    coef = coef > 1.f ? 1.f : coef;          // a NaN stays
    const uint32_t chunks = T.n ? T.first[T.n] : 0;
    for (uint32_t k = blockIdx.x; k < chunks; k += gridDim.x) {
        const uint32_t c = chunks - 1 - k;
        const int t = find(T.first, T.n, c);
        if (coef == 1.f && T.src[t] == T.dst[t]) continue;
        const int64_t per = T.type[t] == 0 ? CHUNK_BYTES / 4 : CHUNK_BYTES / 2, at = (int64_t)(c - T.first[t]) * per, left = T.numel[t] - at, n = left < per ? left : per;
        if (T.type[t] == 0) chunk_scale((const float*)T.src[t] + at, (float*)T.dst[t] + at, n, coef);
        else if (T.type[t] == 1) chunk_scale((const bf16*)T.src[t] + at, (bf16*)T.dst[t] + at, n, coef);
        else chunk_scale((const f16*)T.src[t] + at, (f16*)T.dst[t] + at, n, coef);
    }
}

// `from` .. : as many tensors as one table holds (empty ones left out)
static int fill(Table& T, int& from, int n, const void* const* src, void* const* dst, const int64_t* numel, const int32_t* type) {
    uint64_t chunks = 0;
    T.n = 0;
    while (from < n && T.n < TABLE) {
        const int k = from++;
        if (numel[k] == 0) continue;
        GS_REQUIRE(src[k] && numel[k] > 0 && type[k] >= 0 && type[k] <= 2 && (!dst || dst[k]), "gs_grad_norm: null tensor or unknown type");
        T.src[T.n] = src[k];
        T.dst[T.n] = dst ? dst[k] : nullptr;
        T.numel[T.n] = numel[k];
        T.type[T.n] = (uint8_t)type[k];
        T.first[T.n] = (uint32_t)chunks;
        chunks += (uint64_t)gs::cdiv(numel[k] * (type[k] == 0 ? 4 : 2), CHUNK_BYTES);
        GS_REQUIRE(chunks < (1ull << 31), "gs_grad_norm: too many elements for one launch");
        ++T.n;
    }
    T.first[T.n] = (uint32_t)chunks;
    return 0;
}
static unsigned grid_of(const Table& T) { return T.first[T.n] < (uint32_t)MAX_BLOCKS ? T.first[T.n] : (unsigned)MAX_BLOCKS; }

template <int P>
int run(int n, const void* const* src, void* const* dst, const int64_t* numel, const int32_t* type, float max_norm, float* norm_out, double* part, hipStream_t stream) {
    int parts = 0, tables = 0;
    std::vector<int> starts(n / TABLE + 1);
    Table T;
    for (int from = 0; from < n;) {
        const int start = from;
        if (const int rc = fill(T, from, n, src, dst, numel, type)) return rc;
        if (T.n == 0) continue;
        starts[tables++] = start;
        hipLaunchKernelGGL(k_norm_partials<P>, dim3(grid_of(T)), dim3(THREADS), 0, stream, T, part + parts);
        parts += (int)grid_of(T);
    }
    bool told = false;
    if (dst)
        for (int t = tables - 1; t >= 0; --t) {          // the last table first: it is what the cache holds
            int from = starts[t];
            if (const int rc = fill(T, from, n, src, dst, numel, type)) return rc;
            hipLaunchKernelGGL(k_norm_scale<P>, dim3(grid_of(T)), dim3(THREADS), 0, stream, T, (const double*)part, parts, max_norm, told ? nullptr : norm_out);
            told = true;
        }
    if (!told) {
        T.n = 0, T.first[0] = 0;
        hipLaunchKernelGGL(k_norm_scale<P>, dim3(1), dim3(THREADS), 0, stream, T, (const double*)part, parts, max_norm, norm_out);
    }
    GS_LAUNCH_CHECK();
    return 0;
}

// Whether a stretch of memory that is written overlaps another that is written, or one that is read from somewhere else.
static bool overlap(int n, const void* const* src, void* const* dst, const int64_t* numel, const int32_t* type) {
    struct Stretch { uintptr_t at, end; bool written; };
    std::vector<Stretch> all;
    all.reserve(2 * (size_t)n);
    for (int k = 0; k < n; ++k) {
        if (numel[k] == 0) continue;
        const uintptr_t bytes = (uintptr_t)numel[k] * (type[k] == 0 ? 4 : 2);
        all.push_back({(uintptr_t)dst[k], (uintptr_t)dst[k] + bytes, true});
        if (src[k] != dst[k]) all.push_back({(uintptr_t)src[k], (uintptr_t)src[k] + bytes, false});
    }
    std::sort(all.begin(), all.end(), [](const Stretch& a, const Stretch& b) { return a.at < b.at; });
    uintptr_t end = 0, written = 0;          // ends of what came before: of all, of what is written
    for (const Stretch& s : all) {
        if (s.at < (s.written ? end : written)) return true;
        end = s.end > end ? s.end : end;
        if (s.written && s.end > written) written = s.end;
    }
    return false;
}

}  // namespace

extern "C" int64_t gs_grad_norm_workspace_bytes(int n_tensors) { return n_tensors < 0 ? -1 : (gs::cdiv(n_tensors, TABLE) + 1) * MAX_BLOCKS * 8; }

extern "C" int gs_grad_norm(int n_tensors, const void* const* grads, void* const* out, const int64_t* numel, const int32_t* dtypes, int norm_type, float max_norm,
                            float* norm, void* workspace, int64_t workspace_bytes, gs_stream_t stream) {
    GS_REQUIRE(n_tensors >= 0 && norm && (n_tensors == 0 || (grads && numel && dtypes)), "gs_grad_norm: null argument");
    GS_REQUIRE(norm_type == 0 || norm_type == 1 || norm_type == 2, "gs_grad_norm: norm_type is 0 (2-norm), 1 (1-norm) or 2 (largest magnitude)");
    GS_REQUIRE(!out || max_norm >= 0.f, "gs_grad_norm: max_norm must not be negative or NaN");
    for (int k = 0; k < n_tensors; ++k) GS_REQUIRE(numel[k] == 0 || (numel[k] > 0 && grads[k] && (!out || out[k]) && dtypes[k] >= 0 && dtypes[k] <= 2), "gs_grad_norm: null tensor or unknown type");
    try {          // the lists on the host may not fit
        GS_REQUIRE(!out || !overlap(n_tensors, grads, out, numel, dtypes), "gs_grad_norm: an output shares memory with another output or another gradient");
        GS_REQUIRE(workspace && workspace_bytes >= gs_grad_norm_workspace_bytes(n_tensors), "gs_grad_norm: workspace too small");
        GS_REQUIRE(((uintptr_t)workspace & 7) == 0, "gs_grad_norm: the workspace must start on 8 bytes");
        const auto go = norm_type == 0 ? run<NORM_2> : norm_type == 1 ? run<NORM_1> : run<NORM_INF>;
        return go(n_tensors, grads, out, numel, dtypes, max_norm, norm, (double*)workspace, (hipStream_t)stream);
    } catch (const std::bad_alloc&) {
        gs::set_error("gs_grad_norm: out of host memory");
        return 3;
    }
}
