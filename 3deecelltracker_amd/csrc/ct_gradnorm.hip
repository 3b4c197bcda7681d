// ct_gradnorm.hip -- the l2 norm over a list of gradients, and the list scaled to at most a given norm.
//
//   norm = sqrt( sum_i sum_j g_i[j]^2 )        out_i = g_i * clip / max(norm, clip)        norm not finite: out_i = NaN
//
// Two launches whatever the number of tensors: the list is cut into chunks of kChunk values, every workgroup takes a contiguous run of chunks and
// finds its first tensor by bisection in a table on the device.  Sums are held in 64 bits: a square of a 32-bit value neither overflows nor
// vanishes there, and the partial sums are added in one order that depends on the sizes alone, so a norm repeats bit for bit.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/ctamd.h"

namespace {

constexpr int kChunk = 4096, kBlocks = 2048, kThreads = 256;

struct Entry { const void* in; void* out; int64_t n; int64_t first; int64_t type; };     // first: chunks of the tensors before it
constexpr int kPerLaunch = 64;
struct Batch { Entry e[kPerLaunch]; };                                                   // 2.5 KB of kernel arguments: the host's arrays are free on return

__global__ __launch_bounds__(kPerLaunch) void table_kernel(const Batch b, int n, Entry* __restrict__ table) {
    if ((int)threadIdx.x < n) table[threadIdx.x] = b.e[threadIdx.x];
}

// table words are read with agent-scope loads: an earlier launch wrote them, and they stand at wave-uniform addresses (ct_fresh.h)
__device__ __forceinline__ int64_t word(const Entry* t, int i, int k) {
    return __hip_atomic_load(reinterpret_cast<const int64_t*>(t + i) + k, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

template <typename S> struct Piece { static constexpr int V = 16 / sizeof(S); S v[V]; };

// f(entry, begin, end) for every run of values [begin, end) that this workgroup has
template <typename F>
__device__ __forceinline__ void each_run(const Entry* __restrict__ table, int n, F f) {
    const int64_t total = word(table, n, 3);
    const int64_t c0 = total * blockIdx.x / gridDim.x, c1 = total * (blockIdx.x + 1) / gridDim.x;
    if (c0 >= c1) return;
    int lo = 0, hi = n;                                     // the last entry that begins at or before c0: entries without values are passed over
    while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (word(table, mid, 3) <= c0) lo = mid; else hi = mid; }
    for (int i = lo; i < n; ++i) {
        const int64_t first = word(table, i, 3);
        if (first >= c1) break;
        const int64_t size = word(table, i, 2), b = (c0 > first ? c0 - first : 0) * kChunk, e = (c1 - first) * kChunk;
        f(i, b, e < size ? e : size);
    }
}

__device__ __forceinline__ double block_sum(double v) {
    __shared__ double part[kThreads / 64];
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0;
#pragma unroll
    for (int i = 0; i < kThreads / 64; ++i) v += part[i];
    return v;
}

template <typename S>
__device__ __forceinline__ double squares(const S* __restrict__ p, int64_t n) {
    typedef Piece<S> P;
    constexpr int V = P::V, U = 4;
    double acc = 0.0;
    const int64_t whole = n / V;
    int64_t i = threadIdx.x;
    for (; i + (U - 1) * kThreads < whole; i += U * kThreads) {
        P r[U];
#pragma unroll
        for (int u = 0; u < U; ++u) __builtin_memcpy(&r[u], p + (i + u * kThreads) * V, 16);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int k = 0; k < V; ++k) { const double x = (float)r[u].v[k]; acc = fma(x, x, acc); }
    }
    for (; i < whole; i += kThreads) {
        P r;
        __builtin_memcpy(&r, p + i * V, 16);
#pragma unroll
        for (int k = 0; k < V; ++k) { const double x = (float)r.v[k]; acc = fma(x, x, acc); }
    }
    const int64_t last = whole * V + threadIdx.x;
    if (last < n) { const double x = (float)p[last]; acc = fma(x, x, acc); }
    return acc;
}

__global__ __launch_bounds__(kThreads) void norm_kernel(const Entry* __restrict__ table, int n, double* __restrict__ part) {
    double acc = 0.0;
    each_run(table, n, [&](int i, int64_t b, int64_t e) {
        const void* in = (const void*)word(table, i, 0);
        const int type = (int)word(table, i, 4);
        if (type == CT_F32) acc += squares((const float*)in + b, e - b);
        else if (type == CT_BF16) acc += squares((const __bf16*)in + b, e - b);
        else acc += squares((const _Float16*)in + b, e - b);
    });
    acc = block_sum(acc);
    if (threadIdx.x == 0) part[blockIdx.x] = acc;
}

__device__ __forceinline__ double norm_of(const double* __restrict__ part, int parts) {
    double v = 0.0;
    for (int i = threadIdx.x; i < parts; i += kThreads) v += __hip_atomic_load(part + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return sqrt(block_sum(v));
}

__global__ __launch_bounds__(kThreads) void norm_only_kernel(const double* __restrict__ part, int parts, float* __restrict__ norm) {
    const double v = norm_of(part, parts);
    if (threadIdx.x == 0) *norm = (float)v;
}

template <typename S>
__device__ __forceinline__ void scaled(const S* p, S* o, int64_t n, float f, float f2) {
    typedef Piece<S> P;
    constexpr int V = P::V, U = 4;
    const int64_t whole = n / V;
    int64_t i = threadIdx.x;
    for (; i + (U - 1) * kThreads < whole; i += U * kThreads) {
        P r[U];
#pragma unroll
        for (int u = 0; u < U; ++u) __builtin_memcpy(&r[u], p + (i + u * kThreads) * V, 16);
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int k = 0; k < V; ++k) r[u].v[k] = (S)((float)r[u].v[k] * f * f2);
            __builtin_memcpy(o + (i + u * kThreads) * V, &r[u], 16);
        }
    }
    for (; i < whole; i += kThreads) {
        P r;
        __builtin_memcpy(&r, p + i * V, 16);
#pragma unroll
        for (int k = 0; k < V; ++k) r.v[k] = (S)((float)r.v[k] * f * f2);
        __builtin_memcpy(o + i * V, &r, 16);
    }
    const int64_t last = whole * V + threadIdx.x;
    if (last < n) o[last] = (S)((float)p[last] * f * f2);
}

__global__ __launch_bounds__(kThreads) void clip_kernel(const Entry* __restrict__ table, int n, const double* __restrict__ part, int parts,
                                                        double clip, float* __restrict__ norm_out) {
    const double norm = norm_of(part, parts);
    if (blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
    const double factor = isfinite(norm) ? (norm > clip ? clip / norm : 1.0) : (double)NAN;
    // a factor below the 32-bit normal numbers is applied in two steps, the second a power of two
    const bool tiny = factor < 0x1p-100;
    const float f = (float)(tiny ? factor * 0x1p100 : factor), f2 = tiny ? 0x1p-100f : 1.f;
    each_run(table, n, [&](int i, int64_t b, int64_t e) {
        const void* in = (const void*)word(table, i, 0);
        void* out = (void*)word(table, i, 1);
        const int type = (int)word(table, i, 4);
        if (factor == 1.0 && in == out) return;
        if (type == CT_F32) scaled((const float*)in + b, (float*)out + b, e - b, f, f2);
        else if (type == CT_BF16) scaled((const __bf16*)in + b, (__bf16*)out + b, e - b, f, f2);
        else scaled((const _Float16*)in + b, (_Float16*)out + b, e - b, f, f2);
    });
}

int64_t chunks_of(int64_t n) { return (n + kChunk - 1) / kChunk; }
int blocks_of(int64_t chunks) { return chunks < 1 ? 1 : chunks < kBlocks ? (int)chunks : kBlocks; }

}  // namespace

extern "C" {

size_t ct_gradset_table_bytes(int n) { return n < 0 ? 0 : ((size_t)n + 1) * sizeof(Entry); }
size_t ct_gradset_workspace_bytes(void) { return kBlocks * sizeof(double); }

int64_t ct_gradset_chunks(int n, const int64_t* sizes) {
    if (n < 0 || (n > 0 && !sizes)) return -1;
    int64_t c = 0;
    for (int i = 0; i < n; ++i) { if (sizes[i] < 0) return -1; c += chunks_of(sizes[i]); }
    return c;
}

int ct_gradset_write(int n, const void* const* in, void* const* out, const int64_t* sizes, const int* types, void* table, size_t table_bytes,
                     ct_stream_t stream) {
    if (n < 0 || (n > 0 && (!in || !sizes || !types)) || !table || ((uintptr_t)table & 7)) return CT_EINVAL;
    if (table_bytes < ct_gradset_table_bytes(n)) return CT_EWORKSPACE;
    for (int i = 0; i < n; ++i) {
        if (sizes[i] < 0 || (types[i] != CT_F32 && types[i] != CT_BF16 && types[i] != CT_F16)) return CT_EINVAL;
        const uintptr_t mask = types[i] == CT_F32 ? 3 : 1;
        if (sizes[i] > 0 && (!in[i] || ((uintptr_t)in[i] & mask) || (out && (!out[i] || ((uintptr_t)out[i] & mask))))) return CT_EINVAL;
    }
    hipStream_t st = (hipStream_t)stream;
    int64_t first = 0;
    for (int i0 = 0; i0 <= n; i0 += kPerLaunch) {
        Batch b;
        const int m = n + 1 - i0 < kPerLaunch ? n + 1 - i0 : kPerLaunch;
        for (int k = 0; k < m; ++k) {
            const int i = i0 + k;
            b.e[k] = i < n ? Entry{in[i], out ? out[i] : const_cast<void*>(in[i]), sizes[i], first, types[i]} : Entry{nullptr, nullptr, 0, first, CT_F32};
            if (i < n) first += chunks_of(sizes[i]);
        }
        hipLaunchKernelGGL(table_kernel, dim3(1), dim3(kPerLaunch), 0, st, b, m, (Entry*)table + i0);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return (int)e;
    }
    return CT_OK;
}

int ct_gradset_norm(const void* table, int n, int64_t chunks, float* norm, void* workspace, size_t workspace_bytes, ct_stream_t stream) {
    if (!table || n < 0 || chunks < 0 || !norm || !workspace || ((uintptr_t)workspace & 7)) return CT_EINVAL;
    if (workspace_bytes < ct_gradset_workspace_bytes()) return CT_EWORKSPACE;
    hipStream_t st = (hipStream_t)stream;
    const int parts = blocks_of(chunks);
    hipLaunchKernelGGL(norm_kernel, dim3(parts), dim3(kThreads), 0, st, (const Entry*)table, n, (double*)workspace);
    hipLaunchKernelGGL(norm_only_kernel, dim3(1), dim3(kThreads), 0, st, (const double*)workspace, parts, norm);
    return (int)hipGetLastError();
}

int ct_gradset_clip(const void* table, int n, int64_t chunks, double clip_norm, float* norm, void* workspace, size_t workspace_bytes, ct_stream_t stream) {
    if (!table || n < 0 || chunks < 0 || !norm || !workspace || ((uintptr_t)workspace & 7) || !(clip_norm > 0.0) || clip_norm > 1.7e308) return CT_EINVAL;
    if (workspace_bytes < ct_gradset_workspace_bytes()) return CT_EWORKSPACE;
    hipStream_t st = (hipStream_t)stream;
    const int parts = blocks_of(chunks);
    hipLaunchKernelGGL(norm_kernel, dim3(parts), dim3(kThreads), 0, st, (const Entry*)table, n, (double*)workspace);
    hipLaunchKernelGGL(clip_kernel, dim3(parts), dim3(kThreads), 0, st, (const Entry*)table, n, (const double*)workspace, parts, clip_norm, norm);
    return (int)hipGetLastError();
}

}  // extern "C"
