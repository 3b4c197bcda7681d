// ct_gradnorm.hip -- the l2 norm over a list of gradients, and the list scaled to at most a given norm.
//
//   norm = sqrt( sum_i sum_j g_i[j]^2 )        out_i = g_i * clip / max(norm, clip)        norm not finite: out_i = NaN
//
// Two launches whatever the number of tensors: the list is cut into chunks of kChunk values, every workgroup takes a contiguous run of chunks and
// finds its first tensor by bisection in a table on the device.  Sums are held in 64 bits: a square of a 32-bit value neither overflows nor
// vanishes there, and the partial sums are added in one order that depends on the sizes alone, so a norm repeats bit for bit.
//
// Bound by memory, and for small lists by the launches and by loads that wait for each other (measured on MI355X):
//   * 300 M bf16 values into other tensors: 385 to 397 us, 1.8 GB in three passes = 4.6 TB/s where a copy runs at 5.1 (146 + 238 us; the norm alone, with
//     nothing being written back beside it, goes at 5.5 TB/s, 64-bit sums and all).  The second pass goes backwards, which saves 1 %.
//   * 1200 tensors, 9 M values: 19.4 us (8.4 + 11.8); with halving instead of the 64-wide search, tails piece by piece and 2048 workgroups 28.5.
//   * 9 tensors, 0.56 M values: 10.7 us (3.7 + 4.6 and the call); as a list that is used once 61 us, most of it the host's checks.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/ctamd.h"

namespace {

constexpr int kChunk = 4096, kBlocks = 2048, kThreads = 256;

struct Entry { const void* in; void* out; int64_t n; int64_t first; int64_t type; };     // first: chunks of the tensors before it
constexpr int kWords = sizeof(Entry) / 8, kPerLaunch = 64;
struct Batch { Entry e[kPerLaunch]; };                                                   // 2.5 KB of kernel arguments: the host's arrays are free on return

__global__ __launch_bounds__(kPerLaunch) void table_kernel(const Batch b, int n, Entry* __restrict__ table) {
    if ((int)threadIdx.x < n) table[threadIdx.x] = b.e[threadIdx.x];
}

// table words are read with agent-scope loads by lanes: an earlier launch wrote them, and plain loads of wave-uniform words would be scalar (ct_fresh.h)
__device__ __forceinline__ int64_t word(const Entry* t, int i, int k) {
    return __hip_atomic_load(reinterpret_cast<const int64_t*>(t + i) + k, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ int64_t lane_of(int64_t v, int lane) {
    return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)v, lane));
}

template <typename S> struct Piece { static constexpr int V = 16 / sizeof(S); S v[V]; };

// The last entry that begins at or before chunk c (entries without values are passed over): the 64 lanes look at 64 entries at a time, so a list of
// 1200 takes two loads after one another where halving would take eleven
__device__ __forceinline__ int entry_of(const Entry* __restrict__ table, int n, int64_t c) {
    const int lane = threadIdx.x & 63;
    int lo = 0, span = n;
    while (span > 1) {
        const int step = (span + 63) / 64;
        const bool in = lane * step < span;
        const int k = __popcll(__ballot(in && word(table, in ? lo + lane * step : lo, 3) <= c)) - 1;
        lo += k * step;
        span = span - k * step < step ? span - k * step : step;
    }
    return lo;
}

// f(in, out, type, begin, end) for every run of values [begin, end) of one tensor that this workgroup has, in order or from the last to the first
template <bool BACK, typename F>
__device__ __forceinline__ void each_run(const Entry* __restrict__ table, int n, int64_t total, F f) {
    const int64_t c0 = total * blockIdx.x / gridDim.x, c1 = total * (blockIdx.x + 1) / gridDim.x;
    if (c0 >= c1) return;
    const int lane = threadIdx.x & 63;
    int i = entry_of(table, n, BACK ? c1 - 1 : c0);
    int64_t next = word(table, i, lane < kWords ? lane : 0);
    for (; BACK ? i >= 0 : i < n; i += BACK ? -1 : 1) {
        const int64_t e = next;
        if (BACK ? i > 0 : i + 1 < n) next = word(table, i + (BACK ? -1 : 1), lane < kWords ? lane : 0);       // on its way while this tensor is read
        const int64_t size = lane_of(e, 2), first = lane_of(e, 3);
        if (!BACK && first >= c1) break;
        const int64_t b = (c0 > first ? c0 - first : 0) * kChunk, end = (c1 - first) * kChunk;
        if (b < (end < size ? end : size)) f((const void*)lane_of(e, 0), (void*)lane_of(e, 1), (int)lane_of(e, 4), b, end < size ? end : size);
        if (BACK && first <= c0) break;
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
    // the rest, its loads together: pieces that do not exist are the last one, and not counted
    const int64_t last = whole * V + threadIdx.x;
    const double x = last < n ? (double)(float)p[last] : 0.0;
    if (whole > 0) {
        P r[U];
#pragma unroll
        for (int u = 0; u < U; ++u) __builtin_memcpy(&r[u], p + (i + u * kThreads < whole ? i + u * kThreads : whole - 1) * V, 16);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i + u * kThreads < whole) {
#pragma unroll
                for (int k = 0; k < V; ++k) { const double y = (float)r[u].v[k]; acc = fma(y, y, acc); }
            }
    }
    return fma(x, x, acc);
}

__global__ __launch_bounds__(kThreads) void norm_kernel(const Entry* __restrict__ table, int n, int64_t chunks, double* __restrict__ part) {
    double acc = 0.0;
    each_run<false>(table, n, chunks, [&](const void* in, void*, int type, int64_t b, int64_t e) {
        if (type == CT_F32) acc += squares((const float*)in + b, e - b);
        else if (type == CT_BF16) acc += squares((const __bf16*)in + b, e - b);
        else acc += squares((const _Float16*)in + b, e - b);
    });
    acc = block_sum(acc);
    if (threadIdx.x == 0) part[blockIdx.x] = acc;
}

__device__ __forceinline__ double norm_of(const double* __restrict__ part, int parts) {
    double r[kBlocks / kThreads], v = 0.0;
#pragma unroll
    for (int u = 0; u < kBlocks / kThreads; ++u) {
        const int i = threadIdx.x + u * kThreads;
        r[u] = i < parts ? __hip_atomic_load(part + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0.0;
    }
#pragma unroll
    for (int u = 0; u < kBlocks / kThreads; ++u) v += r[u];
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
    const int64_t whole = n / V, last = whole * V + threadIdx.x;
    const float x = last < n ? (float)p[last] : 0.f;
    int64_t i = whole - 1 - threadIdx.x;
    for (; i - (U - 1) * kThreads >= 0; i -= U * kThreads) {
        P r[U];
#pragma unroll
        for (int u = 0; u < U; ++u) __builtin_memcpy(&r[u], p + (i - u * kThreads) * V, 16);
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int k = 0; k < V; ++k) r[u].v[k] = (S)((float)r[u].v[k] * f * f2);
            __builtin_memcpy(o + (i - u * kThreads) * V, &r[u], 16);
        }
    }
    if (whole > 0) {                                        // the rest, its loads together
        P r[U];
#pragma unroll
        for (int u = 0; u < U; ++u) __builtin_memcpy(&r[u], p + (i - u * kThreads >= 0 ? i - u * kThreads : 0) * V, 16);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i - u * kThreads >= 0) {
#pragma unroll
                for (int k = 0; k < V; ++k) r[u].v[k] = (S)((float)r[u].v[k] * f * f2);
                __builtin_memcpy(o + (i - u * kThreads) * V, &r[u], 16);
            }
    }
    if (last < n) o[last] = (S)(x * f * f2);
}

__global__ __launch_bounds__(kThreads) void clip_kernel(const Entry* __restrict__ table, int n, int64_t chunks, const double* __restrict__ part, int parts,
                                                        double clip, float* __restrict__ norm_out) {
    const double norm = norm_of(part, parts);
    if (blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
    const double factor = isfinite(norm) ? (norm > clip ? clip / norm : 1.0) : (double)NAN;
    // a factor below the 32-bit normal numbers is applied in two steps, the second a power of two
    const bool tiny = factor < 0x1p-100;
    const float f = (float)(tiny ? factor * 0x1p100 : factor), f2 = tiny ? 0x1p-100f : 1.f;
    // from the last values to the first: what the norm read last is still in the memory-side cache
    each_run<true>(table, n, chunks, [&](const void* in, void* out, int type, int64_t b, int64_t e) {
        if (factor == 1.0 && in == out) return;
        if (type == CT_F32) scaled((const float*)in + b, (float*)out + b, e - b, f, f2);
        else if (type == CT_BF16) scaled((const __bf16*)in + b, (__bf16*)out + b, e - b, f, f2);
        else scaled((const _Float16*)in + b, (_Float16*)out + b, e - b, f, f2);
    });
}

int64_t chunks_of(int64_t n) { return (n + kChunk - 1) / kChunk; }
// a workgroup a chunk up to 1024, then 4 chunks each: every workgroup of the second launch adds up the partial sums of all
int blocks_of(int64_t chunks) {
    const int64_t b = chunks <= 1024 ? chunks : chunks / 4 > 1024 ? chunks / 4 : 1024;
    return b < 1 ? 1 : b < kBlocks ? (int)b : kBlocks;
}

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
    hipLaunchKernelGGL(norm_kernel, dim3(parts), dim3(kThreads), 0, st, (const Entry*)table, n, chunks, (double*)workspace);
    hipLaunchKernelGGL(norm_only_kernel, dim3(1), dim3(kThreads), 0, st, (const double*)workspace, parts, norm);
    return (int)hipGetLastError();
}

int ct_gradset_clip(const void* table, int n, int64_t chunks, double clip_norm, float* norm, void* workspace, size_t workspace_bytes, ct_stream_t stream) {
    if (!table || n < 0 || chunks < 0 || !norm || !workspace || ((uintptr_t)workspace & 7) || !(clip_norm > 0.0) || clip_norm > 1.7e308) return CT_EINVAL;
    if (workspace_bytes < ct_gradset_workspace_bytes()) return CT_EWORKSPACE;
    hipStream_t st = (hipStream_t)stream;
    const int parts = blocks_of(chunks);
    hipLaunchKernelGGL(norm_kernel, dim3(parts), dim3(kThreads), 0, st, (const Entry*)table, n, chunks, (double*)workspace);
    hipLaunchKernelGGL(clip_kernel, dim3(parts), dim3(kThreads), 0, st, (const Entry*)table, n, chunks, (const double*)workspace, parts, clip_norm, norm);
    return (int)hipGetLastError();
}

}  // extern "C"
