// ct_grouped.hip -- products of ragged row groups with one weight block each, and their gradients.
//
//   y[r][n]     = act( scale[g][n] * sum_k x[r][k] w[g][k][n] + shift[g][n] )     o_g <= r < o_{g+1}
//   dx[r][k]    = sum_n dy[r][n] w[g][k][n]                                        (the same product, w read transposed)
//   dw[g][k][n] = sum_{o_g <= r < o_{g+1}} x[r][k] dy[r][n]
//
// All three are C[M][N] = sum_c A(m, c) B(c, n) on tiles of a group; they differ in which index of an operand is contiguous in memory:
//   product           A = x   (c contiguous)   B = w   (n contiguous)
//   product, w^T      A = dy  (c contiguous)   B = w   (c contiguous)
//   dw                A = x   (m contiguous)   B = dy  (n contiguous), c = the group's rows
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/ctamd.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

struct BF { typedef __bf16 S; };
struct HF { typedef _Float16 S; };
struct FF { typedef float S; };

// ------------------------------------------------------------------------------------------------
// the group of a tile
// ------------------------------------------------------------------------------------------------
struct Slot { int group, begin, end, row; };        // row: first row of the tile (< end); group == G: rows behind the last group; group < 0: nothing

__device__ __forceinline__ int clampi(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }

// Which `step` rows of which group tile `idx` stands for: groups are cut into ceil(rows / step) tiles each, numbered in order.  Every wave counts
// for itself, 64 groups at a time (a running sum over the lanes).  Offsets are clamped to [0, rows] and to rise, so whatever they hold no tile
// leaves the tensors.
__device__ __forceinline__ Slot find_slot(const int32_t* __restrict__ off, int G, int rows, int step, int idx, bool tail) {
    const int lane = threadIdx.x & 63;
    int base = 0;
    for (int g0 = 0; g0 <= G; g0 += 64) {
        const int g = g0 + lane;
        int b = 0, e = 0;
        if (g <= G) {
            b = clampi(off[g], 0, rows);
            e = g < G ? clampi(off[g + 1], b, rows) : tail ? rows : b;
        }
        const int tiles = (e - b + step - 1) / step;
        int sum = tiles;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) { const int v = __shfl_up(sum, d); if (lane >= d) sum += v; }
        const unsigned long long hit = __ballot(base + sum > idx);
        if (hit) {
            const int src = __ffsll(hit) - 1;
            Slot s;
            s.group = g0 + src;
            s.begin = __builtin_amdgcn_readfirstlane(__shfl(b, src));
            s.end = __builtin_amdgcn_readfirstlane(__shfl(e, src));
            s.row = s.begin + step * (idx - base - __builtin_amdgcn_readfirstlane(__shfl(sum - tiles, src)));
            return s;
        }
        base += __builtin_amdgcn_readfirstlane(__shfl(sum, 63));
    }
    return Slot{-1, 0, 0, 0};
}

// ------------------------------------------------------------------------------------------------
// staging: 16-byte pieces, whole ones as one load of any alignment, those at an edge value by value
// ------------------------------------------------------------------------------------------------
template <typename S> struct Piece { static constexpr int V = 16 / sizeof(S); S v[V]; };

template <typename S>
__device__ __forceinline__ Piece<S> load_piece(const S* p, int have) {
    Piece<S> r;
    if (have >= Piece<S>::V) { __builtin_memcpy(&r, p, 16); return r; }
#pragma unroll
    for (int i = 0; i < Piece<S>::V; ++i) r.v[i] = (S)0.f;
    if (have > 0) {
#pragma unroll
        for (int i = 0; i < Piece<S>::V; ++i) if (i < have) r.v[i] = p[i];
    }
    return r;
}

// One operand's tile of E rows-or-columns x BK contraction steps in LDS.
//   CC (contraction contiguous): [e][BK], 16-byte pieces; 16-bit: piece p of row e stands at p ^ (e & 7); fp32: rows padded by 4 words
//   !CC: [c][E]; 16-bit: 32-byte blocks, block b of row c stands at b ^ swizzle(c): the 8 rows c .. c + 3, c + 8 .. c + 11 that half a wave's
//        transposed read touches fall on different banks; fp32: rows padded by 4 words
template <typename S, bool CC, int E, int BK>
struct Tile {
    static constexpr bool H = sizeof(S) == 2;
    static constexpr int V = 16 / sizeof(S);
    static constexpr int LD = H ? (CC ? BK : E) : (CC ? BK + 4 : E + 4);
    static constexpr int WORDS = LD * (CC ? E : BK);
    static constexpr int PIECES = E * BK / V;

    __device__ static constexpr int swizzle(int c) {
        return E >= 128 ? (c & 3) | (c >> 3 & 1) << 2 : E == 64 ? (c >> 1 & 1) | (c >> 3 & 1) << 1 : E == 32 ? c >> 3 & 1 : 0;
    }
    __device__ static __forceinline__ int at(int e, int c) {        // offset of the piece that holds (e, c); e or c a multiple of V
        if constexpr (!H) return CC ? e * LD + c : c * LD + e;
        if constexpr (CC) return e * LD + (((c >> 3) ^ (e & 7)) << 3);
        const int f = swizzle(c);
        return c * LD + ((((e >> 4) ^ f) << 4) | (e & 8));
    }
};

template <typename S, bool CC, int E, int BK, int NT>
struct Stage {
    typedef Tile<S, CC, E, BK> T;
    static constexpr int N = (T::PIECES + NT - 1) / NT;
    Piece<S> r[N];
    // base: element (e = 0, c = 0); `e_have` rows-or-columns and `c_have` contraction steps exist from there on
    __device__ __forceinline__ void load(const S* base, int64_t ld, int e_have, int c_have) {
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const int q = threadIdx.x + NT * u;
            if (T::PIECES % NT != 0 && q >= T::PIECES) break;
            constexpr int W = (CC ? BK : E) / T::V;                 // pieces along the contiguous index
            const int i = q / W, j = (q % W) * T::V;                // i: strided index, j: contiguous index
            const int have = i < (CC ? e_have : c_have) ? (CC ? c_have : e_have) - j : 0;
            r[u] = load_piece<S>(base + i * ld + j, have);
        }
    }
    __device__ __forceinline__ void store(S* lds) const {
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const int q = threadIdx.x + NT * u;
            if (T::PIECES % NT != 0 && q >= T::PIECES) break;
            constexpr int W = (CC ? BK : E) / T::V;
            const int i = q / W, j = (q % W) * T::V;
            *reinterpret_cast<Piece<S>*>(lds + (CC ? T::at(i, j) : T::at(j, i))) = r[u];
        }
    }
};

// ------------------------------------------------------------------------------------------------
// fragments: lane (l16, lk) of a 16-wide strip holds contraction steps 8 lk .. 8 lk + 7 of 32 (16 bit) or 4 lk .. 4 lk + 3 of 16 (fp32)
// ------------------------------------------------------------------------------------------------
template <typename S, bool CC, int E, int BK>
__device__ __forceinline__ s16x8 frag16(const S* lds, int e0, int c0, int l16, int lk) {
    typedef Tile<S, CC, E, BK> T;
    if constexpr (CC) {
        return *reinterpret_cast<const s16x8*>(lds + T::at(e0 + l16, c0 + 8 * lk));
    } else {
        // the transposed read: of 16 lanes, lane i gives the address of 4 neighbours of row i >> 2 and receives column i of the 4 rows
        const int c = c0 + 8 * lk + (l16 >> 2), e = e0 + 4 * (l16 & 3);
        typedef __attribute__((address_space(3))) s16x4* lp;
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(lds + T::at(e & ~7, c) + (e & 7)));
        const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(lds + T::at(e & ~7, c + 4) + (e & 7)));
        return s16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    }
}
template <bool CC, int E, int BK>
__device__ __forceinline__ f32x4 frag32(const float* lds, int e0, int c0, int l16, int lk) {
    typedef Tile<float, CC, E, BK> T;
    const int c = c0 + 4 * lk;
    if constexpr (CC) return *reinterpret_cast<const f32x4*>(lds + T::at(e0 + l16, c));
    const float* p = lds + T::at(e0 + l16, c);
    return f32x4{p[0], p[T::LD], p[2 * T::LD], p[3 * T::LD]};
}

__device__ __forceinline__ f32x4 mfma(BF, s16x8 a, s16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(HF, s16x8 a, s16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(FF, f32x4 a, f32x4 b, f32x4 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
    return c;
}

template <typename O>
__device__ __forceinline__ void store4(O* p, f32x4 v, int have) {   // 4 neighbours, rounded to nearest
    O r[4] = {(O)v[0], (O)v[1], (O)v[2], (O)v[3]};
    if (have >= 4) { __builtin_memcpy(p, r, sizeof(r)); return; }
#pragma unroll
    for (int i = 0; i < 4; ++i) if (i < have) p[i] = r[i];
}

// ------------------------------------------------------------------------------------------------
// one tile: acc[i][j] holds D = B^T A^T of strips (n strip i, m strip j): a lane has 4 neighbours along n of one m
// ------------------------------------------------------------------------------------------------
template <typename TT, bool ACC, bool BCC, int BM, int BN, int BK, int WM, int WN>
struct Core {
    typedef typename TT::S S;
    static constexpr int NT = 64 * WM * WN, SM = BM / WM / 16, SN = BN / WN / 16, KS = sizeof(S) == 2 ? 32 : 16;
    typedef Tile<S, ACC, BM, BK> TA;
    typedef Tile<S, BCC, BN, BK> TB;
    static constexpr int LDS_BYTES = 2 * (TA::WORDS + TB::WORDS) * (int)sizeof(S);
    f32x4 acc[SN][SM];

    __device__ __forceinline__ void run(S* lds, const S* A, int64_t lda, int m_have, const S* B, int64_t ldb, int n_have, int steps) {
        const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, l16 = lane & 15, lk = lane >> 4;
        const int m0 = (wv % WM) * (BM / WM), n0 = (wv / WM) * (BN / WN);
#pragma unroll
        for (int i = 0; i < SN; ++i)
#pragma unroll
            for (int j = 0; j < SM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        Stage<S, ACC, BM, BK, NT> sa;
        Stage<S, BCC, BN, BK, NT> sb;
        S* la[2] = {lds, lds + TA::WORDS};
        S* lb[2] = {lds + 2 * TA::WORDS, lds + 2 * TA::WORDS + TB::WORDS};
        sa.load(A, lda, m_have, steps); sb.load(B, ldb, n_have, steps);
        sa.store(la[0]); sb.store(lb[0]);
        __syncthreads();
        int buf = 0;
        for (int c0 = 0; c0 < steps; c0 += BK) {
            const bool more = c0 + BK < steps;
            if (more) {
                A += ACC ? (int64_t)BK : BK * lda; B += BCC ? (int64_t)BK : BK * ldb;
                sa.load(A, lda, m_have, steps - c0 - BK); sb.load(B, ldb, n_have, steps - c0 - BK);
            }
            const S* pa = buf ? la[1] : la[0];
            const S* pb = buf ? lb[1] : lb[0];
#pragma unroll
            for (int s = 0; s < BK; s += KS) {
                if constexpr (sizeof(S) == 2) {
                    s16x8 fa[SM], fb[SN];
#pragma unroll
                    for (int j = 0; j < SM; ++j) fa[j] = frag16<S, ACC, BM, BK>(pa, m0 + 16 * j, s, l16, lk);
#pragma unroll
                    for (int i = 0; i < SN; ++i) fb[i] = frag16<S, BCC, BN, BK>(pb, n0 + 16 * i, s, l16, lk);
#pragma unroll
                    for (int i = 0; i < SN; ++i)
#pragma unroll
                        for (int j = 0; j < SM; ++j) acc[i][j] = mfma(TT{}, fb[i], fa[j], acc[i][j]);
                } else {
                    f32x4 fa[SM], fb[SN];
#pragma unroll
                    for (int j = 0; j < SM; ++j) fa[j] = frag32<ACC, BM, BK>(pa, m0 + 16 * j, s, l16, lk);
#pragma unroll
                    for (int i = 0; i < SN; ++i) fb[i] = frag32<BCC, BN, BK>(pb, n0 + 16 * i, s, l16, lk);
#pragma unroll
                    for (int i = 0; i < SN; ++i)
#pragma unroll
                        for (int j = 0; j < SM; ++j) acc[i][j] = mfma(TT{}, fb[i], fa[j], acc[i][j]);
                }
            }
            if (more) { sa.store(buf ? la[0] : la[1]); sb.store(buf ? lb[0] : lb[1]); }
            __syncthreads();
            buf ^= 1;
        }
    }
    // f(m, n, four neighbours along n)
    template <typename F> __device__ __forceinline__ void each(F f) const {
        const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, l16 = lane & 15, lk = lane >> 4;
        const int m0 = (wv % WM) * (BM / WM), n0 = (wv / WM) * (BN / WN);
#pragma unroll
        for (int j = 0; j < SM; ++j)
#pragma unroll
            for (int i = 0; i < SN; ++i) f(m0 + 16 * j + l16, n0 + 16 * i + 4 * lk, acc[i][j]);
    }
};

struct ProductP {
    const void* x; int64_t ldx; int rows, K;
    const void* w; int64_t wg, ldw; int N;
    const int32_t* off; int G;
    const float* scale; const float* shift; int64_t ag; float slope;
    int tail;
    void* y; int64_t ldy;
    int nt;                                  // column tiles
};

template <typename TT, typename O, bool WT, int BM, int BN, int BK, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void product_kernel(const ProductP p) {
    typedef typename TT::S S;
    typedef Core<TT, true, WT, BM, BN, BK, WM, WN> C;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int idx = blockIdx.x / p.nt, n0 = (blockIdx.x - idx * p.nt) * BN;
    const Slot s = find_slot(p.off, p.G, p.rows, BM, idx, p.tail);
    if (s.group < 0) return;
    O* const y = (O*)p.y + (int64_t)s.row * p.ldy + n0;
    const int m_have = s.end - s.row, n_have = p.N - n0;
    C core;
    if (s.group == p.G) {                    // rows behind the last group
        core.run((S*)smem, (const S*)p.x, 0, 0, (const S*)p.w, 0, 0, 0);
        core.each([&](int m, int n, f32x4 v) { if (m < m_have) store4(y + (int64_t)m * p.ldy + n, f32x4{0.f, 0.f, 0.f, 0.f}, n_have - n); });
        return;
    }
    const S* const w = (const S*)p.w + s.group * p.wg + (WT ? n0 * p.ldw : (int64_t)n0);
    core.run((S*)smem, (const S*)p.x + (int64_t)s.row * p.ldx, p.ldx, m_have, w, p.ldw, n_have, p.K);
    const float* const sc = p.scale ? p.scale + s.group * p.ag + n0 : nullptr;
    const float* const sh = p.shift ? p.shift + s.group * p.ag + n0 : nullptr;
    core.each([&](int m, int n, f32x4 v) {
        if (m >= m_have) return;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (n + i >= n_have) break;
            if (sc) v[i] *= sc[n + i];
            if (sh) v[i] += sh[n + i];
            v[i] = v[i] >= 0.f ? v[i] : v[i] * p.slope;
        }
        store4(y + (int64_t)m * p.ldy + n, v, n_have - n);
    });
}

struct DwP {
    const void* x; int64_t ldx; int rows, K;
    const void* dy; int64_t lddy; int N;
    const int32_t* off; int G;
    void* dw; int64_t wg, ldw;
    int mt, nt;
};

template <typename TT, typename O, int BM, int BN, int BK, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void dw_kernel(const DwP p) {
    typedef typename TT::S S;
    typedef Core<TT, false, false, BM, BN, BK, WM, WN> C;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int g = blockIdx.x / (p.mt * p.nt), t = blockIdx.x - g * p.mt * p.nt, m0 = (t / p.nt) * BM, n0 = (t % p.nt) * BN;
    const int b = clampi(p.off[g], 0, p.rows), e = clampi(p.off[g + 1], b, p.rows);
    C core;
    core.run((S*)smem, (const S*)p.x + b * p.ldx + m0, p.ldx, p.K - m0, (const S*)p.dy + b * p.lddy + n0, p.lddy, p.N - n0, e - b);
    O* const out = (O*)p.dw + g * p.wg + m0 * p.ldw + n0;
    core.each([&](int m, int n, f32x4 v) { if (m < p.K - m0) store4(out + m * p.ldw + n, v, p.N - n0 - n); });
}

constexpr int64_t kMaxBlocks = (1 << 24) - 1;               // a grid has fewer than 2^32 work items

bool type_ok(int t) { return t == CT_F32 || t == CT_BF16 || t == CT_F16; }

template <typename TT, typename O, bool WT>
int product_run(const ProductP& p0, hipStream_t st) {
    constexpr int B = 64, BK = sizeof(typename TT::S) == 2 ? 64 : 32;
    typedef Core<TT, true, WT, B, B, BK, 2, 2> C;
    ProductP p = p0;
    p.nt = (p.N + B - 1) / B;
    const int64_t tiles = (int64_t)p.rows / B + (p.rows < p.G + 1 ? p.rows : p.G + 1);      // sum of ceil(rows_g / B) is no more
    const int64_t blocks = tiles * p.nt;
    if (blocks > kMaxBlocks) return CT_ESHAPE;
    hipLaunchKernelGGL((product_kernel<TT, O, WT, B, B, BK, 2, 2>), dim3((unsigned)blocks), dim3(256), C::LDS_BYTES, st, p);
    return (int)hipGetLastError();
}
template <typename TT, typename O>
int dw_run(const DwP& p0, hipStream_t st) {
    constexpr int B = 64, BK = sizeof(typename TT::S) == 2 ? 64 : 32;
    typedef Core<TT, false, false, B, B, BK, 2, 2> C;
    DwP p = p0;
    p.mt = (p.K + B - 1) / B; p.nt = (p.N + B - 1) / B;
    const int64_t blocks = (int64_t)p.G * p.mt * p.nt;
    if (blocks > kMaxBlocks) return CT_ESHAPE;
    hipLaunchKernelGGL((dw_kernel<TT, O, B, B, BK, 2, 2>), dim3((unsigned)blocks), dim3(256), C::LDS_BYTES, st, p);
    return (int)hipGetLastError();
}

}  // namespace

extern "C" {

size_t ct_grouped_product_workspace_bytes(int type, int rows, int K, int N, int G) { return 0; }

int ct_grouped_product(int type, int out_type, const void* x, int64_t ldx, int rows, int K, const void* w, int64_t w_group_stride, int64_t ldw,
                       int w_transposed, int N, const int32_t* offsets, int G, const float* scale, const float* shift, int64_t affine_stride,
                       float slope, int fill_tail, void* y, int64_t ldy, void* workspace, size_t workspace_bytes, ct_stream_t stream) {
    if (!type_ok(type) || !(out_type == type || out_type == CT_F32) || rows < 0 || K < 0 || N <= 0 || G <= 0) return CT_EINVAL;
    if (rows == 0) return CT_OK;
    if (!offsets || !y || (K > 0 && (!x || !w)) || ldy < N || ldx < K || (K > 0 && ldw < (w_transposed ? K : N)) || w_group_stride < 0 || affine_stride < 0) return CT_EINVAL;
    const ProductP p{x, ldx, rows, K, w, w_group_stride, ldw, N, offsets, G, scale, shift, affine_stride, slope, fill_tail != 0, y, ldy, 0};
    hipStream_t st = (hipStream_t)stream;
    const bool wt = w_transposed != 0, f32 = out_type == CT_F32;
    if (type == CT_F32) return wt ? product_run<FF, float, true>(p, st) : product_run<FF, float, false>(p, st);
    if (type == CT_BF16) {
        if (f32) return wt ? product_run<BF, float, true>(p, st) : product_run<BF, float, false>(p, st);
        return wt ? product_run<BF, __bf16, true>(p, st) : product_run<BF, __bf16, false>(p, st);
    }
    if (f32) return wt ? product_run<HF, float, true>(p, st) : product_run<HF, float, false>(p, st);
    return wt ? product_run<HF, _Float16, true>(p, st) : product_run<HF, _Float16, false>(p, st);
}

size_t ct_grouped_product_dw_workspace_bytes(int type, int rows, int K, int N, int G) { return 0; }

int ct_grouped_product_dw(int type, int out_type, const void* x, int64_t ldx, int rows, int K, const void* dy, int64_t lddy, int N,
                          const int32_t* offsets, int G, void* dw, int64_t dw_group_stride, int64_t lddw, void* workspace, size_t workspace_bytes,
                          ct_stream_t stream) {
    if (!type_ok(type) || !(out_type == type || out_type == CT_F32) || rows < 0 || K <= 0 || N <= 0 || G <= 0) return CT_EINVAL;
    if (!offsets || !dw || (rows > 0 && (!x || !dy)) || ldx < K || lddy < N || lddw < N || dw_group_stride < (int64_t)(K - 1) * lddw + N) return CT_EINVAL;
    const DwP p{x, ldx, rows, K, dy, lddy, N, offsets, G, dw, dw_group_stride, lddw, 0, 0};
    hipStream_t st = (hipStream_t)stream;
    const bool f32 = out_type == CT_F32;
    if (type == CT_F32) return dw_run<FF, float>(p, st);
    if (type == CT_BF16) return f32 ? dw_run<BF, float>(p, st) : dw_run<BF, __bf16>(p, st);
    return f32 ? dw_run<HF, float>(p, st) : dw_run<HF, _Float16>(p, st);
}

}  // extern "C"
