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

#include <type_traits>

#include "../../include/ctamd.h"
#include "ct_fresh.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 loose __attribute__((aligned(2)));            // 16 bytes at any address of a value
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
// tiles in LDS
// ------------------------------------------------------------------------------------------------
template <typename S> struct Piece { static constexpr int V = 16 / sizeof(S); S v[V]; };

// One operand's tile of E rows-or-columns x BK contraction steps, in rows of 16-byte pieces without padding (a direct load fills LDS linearly):
//   CC (contraction contiguous)   row = e; piece p stands at p ^ (e & 7), so 8 lanes that read one piece of 8 rows meet different banks
//   !CC                           row = c; 16 bit: 32-byte blocks, block b stands at b ^ swz(c): the 8 rows c .. c + 3, c + 8 .. c + 11 that half a
//                                 wave's transposed read touches meet different banks; fp32: 64-byte blocks, b ^ (c >> 2 & 3), for rows 4 lk + j
template <typename S, bool CC, int E, int BK>
struct Tile {
    static constexpr bool H = sizeof(S) == 2;
    static constexpr int V = 16 / sizeof(S), LD = CC ? BK : E, ROWS = CC ? E : BK, W = LD / V, PIECES = W * ROWS, BYTES = PIECES * 16;
    static_assert(W >= 4 && (W & (W - 1)) == 0, "rows of a power of two of pieces");

    __device__ static constexpr int at_piece(int row, int p) {      // where logical piece p of a row stands; its own inverse
        if (CC) return p ^ (row & (W < 8 ? W - 1 : 7));
        if (H) {
            const int f = E >= 128 ? (row & 3) | (row >> 3 & 1) << 2 : E == 64 ? (row >> 1 & 1) | (row >> 3 & 1) << 1 : row >> 3 & 1;
            return p ^ (f << 1);
        }
        return p ^ ((row >> 2 & (W / 4 - 1) & 3) << 2);
    }
    __device__ static __forceinline__ int at(int e, int c) {
        const int row = CC ? e : c, col = CC ? c : e;
        return row * LD + at_piece(row, col / V) * V + col % V;
    }
};

// A tile on its way through registers: pieces of any alignment.
//   whole: every piece lies in the operand.   edge: the tile may reach past it; the load of a piece that does is moved back, and what was fetched
//   too early is shifted out when the piece is stored (zeros come in): no branch for a single piece, and all loads are in flight together.
template <typename S, bool CC, int E, int BK, int NT, bool EDGE>
struct Stage {
    typedef Tile<S, CC, E, BK> T;
    static constexpr int V = T::V, N = T::PIECES / NT;
    static_assert(T::PIECES % NT == 0, "every thread has the same number of pieces");
    u32x4 r[N];

    // base: element (e = 0, c = 0), from which rows x cols elements of the operand exist; a row of it has `len` elements in all
    __device__ __forceinline__ void load(const S* base, uint32_t ld, int rows, int cols, int len) {
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const int q = threadIdx.x + NT * u;
            int row = q / T::W, col = (q % T::W) * V;
            if constexpr (EDGE || CC) row = row < rows ? row : rows - 1;             // (whole and CC: rows past the operand take its last one, their results are not stored)
            if constexpr (!EDGE) {
                r[u] = *reinterpret_cast<const loose*>((const char*)base + (row * ld + col) * (uint32_t)sizeof(S));
            } else if (len >= V) {
                col = col < cols - V ? col : cols - V;
                r[u] = *reinterpret_cast<const loose*>(base + (int64_t)(row * ld) + col);
            } else {
                Piece<S> v;
#pragma unroll
                for (int i = 0; i < V; ++i) v.v[i] = base[(int64_t)(row * ld) + (col + i < cols ? col + i : cols - 1)];
                r[u] = __builtin_bit_cast(u32x4, v);
            }
        }
    }
    __device__ __forceinline__ void store(S* lds, int rows, int cols, int len) {
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const int q = threadIdx.x + NT * u, row = q / T::W, col = (q % T::W) * V;
            if constexpr (EDGE) {
                typedef unsigned __int128 u128;
                u128 v = __builtin_bit_cast(u128, r[u]);
                if (len >= V) {
                    const int drop = col - (cols - V);                               // values fetched before the piece
                    if (drop > 0) v = drop >= V ? (u128)0 : v >> (8 * sizeof(S) * drop);
                } else {                                                             // a row is shorter than a piece: clear what lies past it
                    const int keep = cols - col;
                    v = keep <= 0 ? (u128)0 : keep >= V ? v : v & (((u128)1 << (8 * sizeof(S) * keep)) - 1);
                }
                if (!CC && row >= rows) v = 0;                                       // a contraction step that does not exist
                r[u] = __builtin_bit_cast(u32x4, v);
            }
            *reinterpret_cast<u32x4*>(lds + row * T::LD + T::at_piece(row, col / V) * V) = r[u];
        }
    }
};

// The same straight into LDS: 16 bytes a lane, a wave fills 1 KB; the source of a lane is the piece that stands where the lane writes.
// Sources have to be whole pieces (the address a multiple of 4 bytes); rows past the operand take the last one (their results are not stored).
// The instruction is written out because the compiler's own form makes it wait for all such loads before any read of LDS; Core waits for them.
__device__ __forceinline__ void direct16(const void* base, uint32_t voff, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" :: "s"(lds), "v"(voff), "s"(base) : "memory");
}
template <typename S, bool CC, int E, int BK, int NT>
struct Direct {
    typedef Tile<S, CC, E, BK> T;
    static constexpr int N = T::PIECES / NT;
    static_assert(T::PIECES % NT == 0, "every wave loads the same number of pieces");
    uint32_t voff[N];
    __device__ __forceinline__ void init(uint32_t ld, int rows) {
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const int q = threadIdx.x + NT * u;
            int row = q / T::W;
            const int col = T::at_piece(row, q % T::W) * T::V;
            if (CC) row = row < rows ? row : rows - 1;
            voff[u] = (row * ld + col) * (uint32_t)sizeof(S);
        }
    }
    __device__ __forceinline__ void load(const S* tile, uint32_t lds) const {
        const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const uint64_t p = (uint64_t)(uintptr_t)tile;                                 // the same for all lanes: say so
        const void* const base = (const void*)(uintptr_t)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(p >> 32)) << 32 |
                                                          (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)p));
#pragma unroll
        for (int u = 0; u < N; ++u) direct16(base, voff[u], __builtin_amdgcn_readfirstlane(lds + (wave * 64 + NT * u) * 16));
    }
};

// ------------------------------------------------------------------------------------------------
// fragments: lane (l16, lk) of a 16-wide strip holds contraction steps 8 lk .. 8 lk + 7 of 32 (16 bit) or 4 lk .. 4 lk + 3 of 16 (fp32)
// ------------------------------------------------------------------------------------------------
// Byte offsets of a wave's strips in a tile: the lane's part is the same for every step but one bit, so it is worked out once and the rest are constants.
template <typename S, bool CC, int E, int BK, int STRIPS>
struct Strips {
    typedef Tile<S, CC, E, BK> T;
    static constexpr bool H = sizeof(S) == 2;
    static constexpr int ROW = T::LD * (int)sizeof(S), KS = H ? 32 : 16;       // a step of KS contraction values is 4 pieces of a CC row
    int off[CC ? 2 : STRIPS];

    // the wave's strips from e0 on, its contraction steps from c0 on (a multiple of KS, of 2 KS if there are several)
    __device__ __forceinline__ void init(int e0, int c0) {
        const int lane = threadIdx.x & 63, l16 = lane & 15, lk = lane >> 4;
        if constexpr (CC) {                                                     // e0 is a multiple of 16: the row's swizzle is the lane's
            off[0] = (e0 + l16) * ROW + T::at_piece(l16, c0 / T::V + lk) * 16;
            off[1] = T::W >= 8 ? (e0 + l16) * ROW + T::at_piece(l16, c0 / T::V + 4 + lk) * 16 : off[0];
        } else {
#pragma unroll
            for (int j = 0; j < STRIPS; ++j) {
                // 16 bit, the transposed read: of 16 lanes, lane i gives the address of 4 neighbours of row i >> 2 and receives column i of the 4 rows
                const int c = H ? 8 * lk + (l16 >> 2) : 4 * lk, e = e0 + 16 * j + (H ? 4 * (l16 & 3) : l16);
                off[j] = T::at(e, c) * (int)sizeof(S) + c0 * ROW;
            }
        }
    }
    // strip j, contraction step s (a multiple of KS)
    __device__ __forceinline__ typename std::conditional<H, s16x8, f32x4>::type read(const unsigned char* lds, int j, int s) const {
        if constexpr (CC) {
            const unsigned char* p = lds + off[T::W >= 8 ? s / KS & 1 : 0] + j * 16 * ROW + s / KS / 2 * 128;
            return *reinterpret_cast<const typename std::conditional<H, s16x8, f32x4>::type*>(p);
        } else if constexpr (H) {
            typedef __attribute__((address_space(3))) s16x4* lp;
            const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(lds + off[j] + s * ROW));
            const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(lds + off[j] + (s + 4) * ROW));
            return s16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
        } else {
            const unsigned char* p = lds + off[j] + s * ROW;
            f32x4 v;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const float*>(p + i * ROW);
            return v;
        }
    }
};

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

// The bits of a fragment's contraction steps k0, k0 + 1, .. that lie in [lo, hi): whatever stands in the others, a NaN too, becomes zero
template <bool H> __device__ __forceinline__ u32x4 steps_in(int k0, int lo, int hi) {
    u32x4 m;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (H) m[i] = (k0 + 2 * i >= lo && k0 + 2 * i < hi ? 0xffffu : 0u) | (k0 + 2 * i + 1 >= lo && k0 + 2 * i + 1 < hi ? 0xffff0000u : 0u);
        else m[i] = k0 + i >= lo && k0 + i < hi ? 0xffffffffu : 0u;
    }
    return m;
}
template <typename F> __device__ __forceinline__ F masked(F f, u32x4 m) { return __builtin_bit_cast(F, __builtin_bit_cast(u32x4, f) & m); }

// How a tile reaches LDS
//   DIRECT   straight from memory; REGS through registers (values of any alignment).  Both want operands no smaller than the tile: a last stage that
//            would reach past the contraction's end begins earlier instead and masks the steps that were done, likewise at the end of a group's rows.
//   EDGE     through registers, operands of any size
enum Way { DIRECT, REGS, EDGE };

// ------------------------------------------------------------------------------------------------
// one tile: acc[i][j] holds D = B^T A^T of strips (n strip i, m strip j): a lane has 4 neighbours along n of one m
// ------------------------------------------------------------------------------------------------
// WM x WN waves share the tile, WK of them each take a part of every stage's contraction steps (small tiles: more of a long sum in flight) and add
// up through LDS at the end, in order.  Two stages in LDS, one in flight while the other is multiplied.
template <typename TT, bool ACC, bool BCC, int BM, int BN, int BK, int WM, int WN, int WK, Way WAY>
struct Core {
    typedef typename TT::S S;
    static constexpr bool H = sizeof(S) == 2;
    static constexpr int NT = 64 * WM * WN * WK, SM = BM / WM / 16, SN = BN / WN / 16, KS = H ? 32 : 16, PK = BK / WK;
    static_assert(PK % KS == 0 && (PK == KS || PK % (2 * KS) == 0) && SM * 16 * WM == BM && SN * 16 * WN == BN, "whole strips");
    typedef Tile<S, ACC, BM, BK> TA;
    typedef Tile<S, BCC, BN, BK> TB;
    static constexpr int STAGE_BYTES = TA::BYTES + TB::BYTES, SUM_BYTES = WK > 1 ? BM * BN * WK * 4 : 0;
    static constexpr int LDS_BYTES = 2 * STAGE_BYTES > SUM_BYTES ? 2 * STAGE_BYTES : SUM_BYTES;
    // fp32 sums of one wave run over at most kChain steps and are then added to the total: a long chain loses a bit for every fourfold length
    static constexpr int kChain = 512;
    static constexpr bool FOLD = !H && WK == 1;
    typedef typename std::conditional<H, s16x8, f32x4>::type Frag;
    f32x4 acc[SN][SM];

    __device__ __forceinline__ void place(int& m0, int& n0, int& kz) const {
        const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        m0 = (wv % WM) * (BM / WM); n0 = (wv / WM % WN) * (BN / WN); kz = wv / (WM * WN);
    }
    Strips<S, ACC, BM, BK, SM> ra;
    Strips<S, BCC, BN, BK, SN> rb;
    template <bool MASK>
    __device__ __forceinline__ void multiply(const unsigned char* stage, int kz, int lo, int hi) {
        const int k0 = kz * PK + KS / 4 * ((threadIdx.x & 63) >> 4);
#pragma unroll
        for (int s0 = 0; s0 < PK; s0 += KS) {
            Frag fa[SM], fb[SN];
            u32x4 mask;
            if (MASK) mask = steps_in<H>(k0 + s0, lo, hi);
#pragma unroll
            for (int j = 0; j < SM; ++j) {
                fa[j] = ra.read(stage, j, s0);
                if (MASK) fa[j] = masked(fa[j], mask);
            }
#pragma unroll
            for (int i = 0; i < SN; ++i) {
                fb[i] = rb.read(stage + TA::BYTES, i, s0);
                if (MASK) fb[i] = masked(fb[i], mask);
            }
#pragma unroll
            for (int i = 0; i < SN; ++i)
#pragma unroll
                for (int j = 0; j < SM; ++j) acc[i][j] = mfma(TT{}, fb[i], fa[j], acc[i][j]);
        }
    }

    // A, B: element (0 of the tile, contraction step 0 of the operand); m_have rows-or-columns of A and n_have of B exist from there, rows of them (where
    // m or n is contiguous) have len_a, len_b values.  The steps [begin, end) of `extent` are summed.
    __device__ __forceinline__ void run(unsigned char* smem, const S* A, uint32_t lda, int m_have, int len_a, const S* B, uint32_t ldb, int n_have, int len_b,
                                        int begin, int end, int extent) {
        int m0, n0, kz;
        place(m0, n0, kz);
        ra.init(m0, kz * PK); rb.init(n0, kz * PK);
        f32x4 total[FOLD ? SN : 1][FOLD ? SM : 1];
#pragma unroll
        for (int i = 0; i < SN; ++i)
#pragma unroll
            for (int j = 0; j < SM; ++j) {
                acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
                if constexpr (FOLD) total[i][j] = acc[i][j];
            }
        const int stages = (end - begin + BK - 1) / BK;
        auto la = [&](int t) { return (S*)(smem + (t & 1) * STAGE_BYTES); };
        auto lb = [&](int t) { return (S*)(smem + (t & 1) * STAGE_BYTES + TA::BYTES); };
        auto from = [&](int t) { const int c = begin + t * BK; return WAY == EDGE || c + BK <= extent ? c : extent - BK; };
        auto pa = [&](int t) { return A + (ACC ? (int64_t)from(t) : (int64_t)from(t) * lda); };
        auto pb = [&](int t) { return B + (BCC ? (int64_t)from(t) : (int64_t)from(t) * ldb); };
        const int full = WAY == EDGE ? stages : (end - begin) / BK;             // stages all of whose steps count; one more may follow
        auto step = [&](int t) {
            multiply<false>(smem + (t & 1) * STAGE_BYTES, kz, 0, 0);
            if constexpr (FOLD)
                if ((t + 1) % (kChain / BK) == 0) {
#pragma unroll
                    for (int i = 0; i < SN; ++i)
#pragma unroll
                        for (int j = 0; j < SM; ++j) { total[i][j] += acc[i][j]; acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f}; }
                }
        };
        auto last = [&](int t) { multiply<true>(smem + (t & 1) * STAGE_BYTES, kz, begin + t * BK - from(t), end - from(t)); };
        if constexpr (WAY == DIRECT) {
            Direct<S, ACC, BM, BK, NT> da;
            Direct<S, BCC, BN, BK, NT> db;
            da.init(lda, m_have); db.init(ldb, n_have);
            const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)smem;
            auto issue = [&](int t) {
                da.load(pa(t), lds + (t & 1) * STAGE_BYTES);
                db.load(pb(t), lds + (t & 1) * STAGE_BYTES + TA::BYTES);
            };
            if (stages > 0) issue(0);
            auto landed = [] { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); };   // stage t is there, stage t - 1 has been read
            for (int t = 0; t < full; ++t) {
                landed();
                if (t + 1 < stages) issue(t + 1);
                step(t);
            }
            if (full < stages) { landed(); last(full); }
        } else {
            Stage<S, ACC, BM, BK, NT, WAY == EDGE> sa;
            Stage<S, BCC, BN, BK, NT, WAY == EDGE> sb;
            auto load = [&](int t) {
                const int c = end - from(t);
                sa.load(pa(t), lda, ACC ? m_have : c, ACC ? c : m_have, ACC ? extent : len_a);
                sb.load(pb(t), ldb, BCC ? n_have : c, BCC ? c : n_have, BCC ? extent : len_b);
            };
            auto store = [&](int t) {
                const int c = end - from(t);
                sa.store(la(t), ACC ? m_have : c, ACC ? c : m_have, ACC ? extent : len_a);
                sb.store(lb(t), BCC ? n_have : c, BCC ? c : n_have, BCC ? extent : len_b);
            };
            if (stages > 0) { load(0); store(0); }
            __syncthreads();
            for (int t = 0; t < full; ++t) {
                if (t + 1 < stages) load(t + 1);
                step(t);
                if (t + 1 < stages) store(t + 1);
                __syncthreads();
            }
            if (full < stages) last(full);
        }
        if constexpr (FOLD) {
#pragma unroll
            for (int i = 0; i < SN; ++i)
#pragma unroll
                for (int j = 0; j < SM; ++j) acc[i][j] += total[i][j];
        }
        if constexpr (WK > 1) {                                 // parts of the sum meet in LDS; wave kz goes on with every WK-th strip
            __syncthreads();
            f32x4* const part = (f32x4*)smem;
            const int lane = threadIdx.x & 63, mn = (threadIdx.x >> 6) % (WM * WN);
#pragma unroll
            for (int i = 0; i < SN; ++i)
#pragma unroll
                for (int j = 0; j < SM; ++j) part[((kz * WM * WN + mn) * SN * SM + i * SM + j) * 64 + lane] = acc[i][j];
            __syncthreads();
#pragma unroll
            for (int i = 0; i < SN; ++i)
#pragma unroll
                for (int j = 0; j < SM; ++j) {
                    if ((i * SM + j) % WK != kz) continue;
                    f32x4 v = part[(mn * SN * SM + i * SM + j) * 64 + lane];
#pragma unroll
                    for (int z = 1; z < WK; ++z) v += part[((z * WM * WN + mn) * SN * SM + i * SM + j) * 64 + lane];
                    acc[i][j] = v;
                }
        }
    }
    // f(m, n, four neighbours along n)
    template <typename F> __device__ __forceinline__ void each(F f) const {
        const int lane = threadIdx.x & 63, l16 = lane & 15, lk = lane >> 4;
        int m0, n0, kz;
        place(m0, n0, kz);
#pragma unroll
        for (int j = 0; j < SM; ++j)
#pragma unroll
            for (int i = 0; i < SN; ++i) {
                if (WK > 1 && (i * SM + j) % WK != kz) continue;
                f(m0 + 16 * j + l16, n0 + 16 * i + 4 * lk, acc[i][j]);
            }
    }
};

template <typename O>
__device__ __forceinline__ void store4(O* p, f32x4 v, int first, int have) {   // neighbours first .. have - 1 of 4, rounded to nearest
    O r[4] = {(O)v[0], (O)v[1], (O)v[2], (O)v[3]};
    if (first <= 0 && have >= 4) { __builtin_memcpy(p, r, sizeof(r)); return; }
#pragma unroll
    for (int i = 0; i < 4; ++i) if (i >= first && i < have) p[i] = r[i];
}
// out: CT_F32 or the operands' type
template <typename S>
__device__ __forceinline__ void store_out(void* p, int64_t at, bool f32, f32x4 v, int first, int have) {
    if (sizeof(S) == 4 || f32) store4((float*)p + at, v, first, have); else store4((S*)p + at, v, first, have);
}

// Tiles of consecutive numbers share operands, and workgroups go to the 8 XCDs (each with its own L2) in turn: a run of kRun numbers goes to one XCD.
constexpr int kXcd = 8, kRun = 32;
__device__ __forceinline__ int tile_number(int id, int count) {
    const int full = count / (kXcd * kRun) * (kXcd * kRun);
    if (id >= full) return id;
    const int block = id / (kXcd * kRun), in = id % (kXcd * kRun);
    return block * (kXcd * kRun) + (in % kXcd) * kRun + in / kXcd;
}

struct ProductP {
    const void* x; int64_t ldx; int rows, K;
    const void* w; int64_t wg, ldw; int N;
    const int32_t* off; int G;
    const float* scale; const float* shift; int64_t ag; float slope;
    int tail, out32;
    void* y; int64_t ldy;
    int slots, nt, count;                    // row tiles (at most), column tiles, workgroups
};

// The last column tile is moved back so that it ends with the matrix (its first columns are then another tile's to store): whole pieces in every tile.
__device__ __forceinline__ int moved_back(int at, int tile, int extent) { return at + tile <= extent || extent < tile ? at : extent - tile; }

template <typename TT, bool WT, int BM, int BN, int BK, int WM, int WN, int WK, Way WAY>
__global__ __launch_bounds__(64 * WM * WN * WK) void product_kernel(const ProductP p) {
    typedef typename TT::S S;
    typedef Core<TT, true, WT, BM, BN, BK, WM, WN, WK, WAY> C;
    __shared__ __attribute__((aligned(1024))) unsigned char smem[C::LDS_BYTES];
    // four row tiles side by side, then the next column tile: 32 numbers in a row touch 4 row panels and 8 column panels
    const int t = tile_number(blockIdx.x, p.count), strip = 4 * p.nt, s4 = t / strip, in = t - s4 * strip;
    const int wide = p.slots - 4 * s4 < 4 ? p.slots - 4 * s4 : 4, col = in / wide, slot = 4 * s4 + in - col * wide;
    const Slot s = find_slot(p.off, p.G, p.rows, BM, slot, p.tail);
    if (s.group < 0) return;
    const int nom = col * BN, n0 = moved_back(nom, BN, p.N), first = nom - n0;
    const int m_have = s.end - s.row, n_have = p.N - n0;
    const int64_t at = (int64_t)s.row * p.ldy + n0;
    if (s.group == p.G) {                    // rows behind the last group
        for (int i = threadIdx.x; i < BM * (BN / 4); i += C::NT) {
            const int m = i / (BN / 4), n = i % (BN / 4) * 4;
            if (m < m_have && n < n_have) store_out<S>(p.y, at + m * p.ldy + n, p.out32, f32x4{0.f, 0.f, 0.f, 0.f}, first - n, n_have - n);
        }
        return;
    }
    const S* const w = (const S*)p.w + s.group * p.wg + (WT ? n0 * p.ldw : (int64_t)n0);
    C core;
    core.run(smem, (const S*)p.x + (int64_t)s.row * p.ldx, (uint32_t)p.ldx, m_have, p.K, w, (uint32_t)p.ldw, n_have, p.N, 0, p.K, p.K);
    const float* const sc = p.scale ? p.scale + s.group * p.ag + n0 : nullptr;
    const float* const sh = p.shift ? p.shift + s.group * p.ag + n0 : nullptr;
    core.each([&](int m, int n, f32x4 v) {
        if (m >= m_have || n >= n_have) return;
        if (sc || sh) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int ni = n + i < n_have ? n + i : n_have - 1;
                if (sc) v[i] *= sc[ni];
                if (sh) v[i] += sh[ni];
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = v[i] >= 0.f ? v[i] : v[i] * p.slope;
        store_out<S>(p.y, at + m * p.ldy + n, p.out32, v, first - n, n_have - n);
    });
}

struct DwP {
    const void* x; int64_t ldx; int rows, K;
    const void* dy; int64_t lddy; int N;
    const int32_t* off; int G;
    void* dw; int64_t wg, ldw;
    int out32, mt, nt, count;
};

template <typename TT, int BM, int BN, int BK, int WM, int WN, int WK, Way WAY>
__global__ __launch_bounds__(64 * WM * WN * WK) void dw_kernel(const DwP p) {
    typedef typename TT::S S;
    typedef Core<TT, false, false, BM, BN, BK, WM, WN, WK, WAY> C;
    __shared__ __attribute__((aligned(1024))) unsigned char smem[C::LDS_BYTES];
    const int tile = tile_number(blockIdx.x, p.count), g = tile / (p.mt * p.nt), t = tile - g * p.mt * p.nt;
    const int nom_m = (t / p.nt) * BM, m0 = moved_back(nom_m, BM, p.K), nom_n = (t % p.nt) * BN, n0 = moved_back(nom_n, BN, p.N);
    const int b = clampi(fresh_i32(p.off + g), 0, p.rows), e = clampi(fresh_i32(p.off + g + 1), b, p.rows);
    C core;
    core.run(smem, (const S*)p.x + m0, (uint32_t)p.ldx, p.K - m0, p.K, (const S*)p.dy + n0, (uint32_t)p.lddy, p.N - n0, p.N, b, e, p.rows);
    const int64_t at = g * p.wg + m0 * p.ldw + n0;
    core.each([&](int m, int n, f32x4 v) {
        if (m >= nom_m - m0 && m < p.K - m0 && n < p.N - n0) store_out<S>(p.dw, at + m * p.ldw + n, p.out32, v, nom_n - n0 - n, p.N - n0 - n);
    });
}

constexpr int64_t kMaxBlocks = (1 << 22) - 1;               // a grid has fewer than 2^32 work items, a workgroup up to 512
constexpr int64_t kMaxStride = 1 << 22;                     // a tile's offsets fit 32 bits: 256 rows of 2^22 values

bool type_ok(int t) { return t == CT_F32 || t == CT_BF16 || t == CT_F16; }
bool words(const void* p, int64_t ld, int64_t more, int size) { return (((uintptr_t)p | (uintptr_t)(ld * size) | (uintptr_t)(more * size)) & 3) == 0; }

template <typename TT, bool WT, int BM, int BN, int BK, int WM, int WN, int WK, Way WAY>
int product_launch(ProductP p, hipStream_t st) {
    p.nt = (p.N + BN - 1) / BN;
    const int64_t slots = (int64_t)p.rows / BM + (p.rows < p.G + 1 ? p.rows : p.G + 1);     // sum of ceil(rows_g / BM) is no more
    if (slots * p.nt > kMaxBlocks) return CT_ESHAPE;
    p.slots = (int)slots; p.count = (int)(slots * p.nt);
    hipLaunchKernelGGL((product_kernel<TT, WT, BM, BN, BK, WM, WN, WK, WAY>), dim3((unsigned)p.count), dim3(64 * WM * WN * WK), 0, st, p);
    return (int)hipGetLastError();
}
template <typename TT, int BM, int BN, int BK, int WM, int WN, int WK, Way WAY>
int dw_launch(DwP p, hipStream_t st) {
    p.mt = (p.K + BM - 1) / BM; p.nt = (p.N + BN - 1) / BN;
    const int64_t count = (int64_t)p.G * p.mt * p.nt;
    if (count > kMaxBlocks) return CT_ESHAPE;
    p.count = (int)count;
    hipLaunchKernelGGL((dw_kernel<TT, BM, BN, BK, WM, WN, WK, WAY>), dim3((unsigned)p.count), dim3(64 * WM * WN * WK), 0, st, p);
    return (int)hipGetLastError();
}

constexpr int64_t kCus = 256;
int64_t tiles(int64_t m, int64_t n, int bm, int bn) { return ((m + bm - 1) / bm) * ((n + bn - 1) / bn); }

// Which tile.  16 x 64: a few rows a group, bound by the weights, every wave a quarter of the sum.  Large tiles where there are enough of them for all
// CUs, since each value of an operand is then fetched less often; else small ones, with the sum split over the waves.
template <typename TT, bool WT, Way WAY>
int product_pick(const ProductP& p, hipStream_t st) {
    const int64_t mean = (p.rows + p.G - 1) / p.G, r = p.rows;
    const int k = p.K, n = WT ? 1 << 30 : p.N;              // what the tile must not exceed: rows of w may be repeated, columns may not
    if constexpr (WAY != EDGE && sizeof(typename TT::S) == 2) {
        constexpr int WIDE = WAY == DIRECT ? 256 : 128;
        if (mean <= 16 && k >= WIDE && n >= 64) return product_launch<TT, WT, 16, 64, WIDE, 1, 1, 4, WAY>(p, st);
        if constexpr (WAY == DIRECT)
            if (mean >= 192 && k >= 64 && p.N >= 256 && tiles(r, p.N, 256, 256) >= kCus) return product_launch<TT, WT, 256, 256, 64, 2, 4, 1, WAY>(p, st);
        if (mean >= 96 && k >= 64 && p.N >= 128 && tiles(r, p.N, 128, 128) >= kCus) return product_launch<TT, WT, 128, 128, 64, 2, 2, 1, WAY>(p, st);
        if (k >= 128 && n >= 64) return product_launch<TT, WT, 64, 64, 128, 1, 2, 2, WAY>(p, st);
        if (k >= 32 && n >= 64) return product_launch<TT, WT, 64, 64, 32, 2, 2, 1, WAY>(p, st);
    }
    if constexpr (WAY == DIRECT && sizeof(typename TT::S) == 4) {
        if (mean <= 16 && k >= 128 && n >= 64) return product_launch<TT, WT, 16, 64, 128, 1, 1, 4, WAY>(p, st);
        if (mean >= 96 && k >= 32 && p.N >= 128 && tiles(r, p.N, 128, 128) >= 2 * kCus) return product_launch<TT, WT, 128, 128, 32, 2, 2, 1, WAY>(p, st);
        if (k >= 128 && n >= 32 && tiles(r, p.N, 64, 64) < 2 * kCus) return product_launch<TT, WT, 32, 32, 128, 1, 1, 4, WAY>(p, st);
        if (k >= 32 && n >= 64) return product_launch<TT, WT, 64, 64, 32, 2, 2, 1, WAY>(p, st);
    }
    return product_launch<TT, WT, 64, 64, 32, 2, 2, 1, EDGE>(p, st);
}
template <typename TT, Way WAY>
int dw_pick(const DwP& p, hipStream_t st) {
    const int r = p.rows, k = p.K, n = p.N;
    if constexpr (WAY != EDGE && sizeof(typename TT::S) == 2) {
        if constexpr (WAY == DIRECT)
            if (r >= 64 && k >= 256 && n >= 256 && p.G * tiles(k, n, 256, 256) >= kCus) return dw_launch<TT, 256, 256, 64, 2, 4, 1, WAY>(p, st);
        if (r >= 64 && k >= 128 && n >= 128 && p.G * tiles(k, n, 128, 128) >= kCus) return dw_launch<TT, 128, 128, 64, 2, 2, 1, WAY>(p, st);
        if (r >= 128 && k >= 64 && n >= 64) return dw_launch<TT, 64, 64, 128, 1, 2, 2, WAY>(p, st);
    }
    if constexpr (WAY == DIRECT && sizeof(typename TT::S) == 4) {
        if (r >= 32 && k >= 128 && n >= 128 && p.G * tiles(k, n, 128, 128) >= 2 * kCus) return dw_launch<TT, 128, 128, 32, 2, 2, 1, WAY>(p, st);
        if (r >= 128 && k >= 32 && n >= 32 && p.G * tiles(k, n, 64, 64) < 2 * kCus) return dw_launch<TT, 32, 32, 128, 1, 1, 4, WAY>(p, st);
        if (r >= 32 && k >= 64 && n >= 64) return dw_launch<TT, 64, 64, 32, 2, 2, 1, WAY>(p, st);
    }
    return dw_launch<TT, 64, 64, 32, 2, 2, 1, EDGE>(p, st);
}

// direct loads want addresses that are multiples of 4 bytes (16-bit values: an even stride, and an even width where the last tile is moved back)
template <typename TT>
int product_run(const ProductP& p, bool wt, hipStream_t st) {
    constexpr int size = sizeof(typename TT::S);
    if (size == 4 || (words(p.x, p.ldx, p.K, size) && words(p.w, p.ldw, p.wg, size) && (wt || p.N % 2 == 0)))
        return wt ? product_pick<TT, true, DIRECT>(p, st) : product_pick<TT, false, DIRECT>(p, st);
    return wt ? product_pick<TT, true, size == 2 ? REGS : EDGE>(p, st) : product_pick<TT, false, size == 2 ? REGS : EDGE>(p, st);
}
template <typename TT>
int dw_run(const DwP& p, hipStream_t st) {
    constexpr int size = sizeof(typename TT::S);
    if (size == 4 || (words(p.x, p.ldx, p.K, size) && words(p.dy, p.lddy, p.N, size))) return dw_pick<TT, DIRECT>(p, st);
    return dw_pick<TT, size == 2 ? REGS : EDGE>(p, st);
}

int product_any(int type, const ProductP& p, bool wt, hipStream_t st) {
    return type == CT_F32 ? product_run<FF>(p, wt, st) : type == CT_BF16 ? product_run<BF>(p, wt, st) : product_run<HF>(p, wt, st);
}
int dw_any(int type, const DwP& p, hipStream_t st) { return type == CT_F32 ? dw_run<FF>(p, st) : type == CT_BF16 ? dw_run<BF>(p, st) : dw_run<HF>(p, st); }

}  // namespace

extern "C" {

size_t ct_grouped_product_workspace_bytes(int type, int rows, int K, int N, int G) { return 0; }

int ct_grouped_product(int type, int out_type, const void* x, int64_t ldx, int rows, int K, const void* w, int64_t w_group_stride, int64_t ldw,
                       int w_transposed, int N, const int32_t* offsets, int G, const float* scale, const float* shift, int64_t affine_stride,
                       float slope, int fill_tail, void* y, int64_t ldy, void* workspace, size_t workspace_bytes, ct_stream_t stream) {
    if (!type_ok(type) || !(out_type == type || out_type == CT_F32) || rows < 0 || K <= 0 || N <= 0 || G <= 0) return CT_EINVAL;
    if (rows == 0) return CT_OK;
    if (!offsets || !y || !x || !w || ldy < N || ldx < K || ldw < (w_transposed ? K : N) || w_group_stride < 0 || affine_stride < 0) return CT_EINVAL;
    if (ldx > kMaxStride || ldw > kMaxStride) return CT_ESHAPE;
    const ProductP p{x, ldx, rows, K, w, w_group_stride, ldw, N, offsets, G, scale, shift, affine_stride, slope, fill_tail != 0, out_type == CT_F32, y, ldy, 0, 0, 0};
    return product_any(type, p, w_transposed != 0, (hipStream_t)stream);
}

size_t ct_grouped_product_grad_workspace_bytes(int type, int rows, int K, int N, int G) { return 0; }

int ct_grouped_product_grad(int type, int out_type, const void* dy, int64_t lddy, const void* x, int64_t ldx, int rows, int K, const void* w,
                            int64_t w_group_stride, int64_t ldw, int w_transposed, int N, const int32_t* offsets, int G, void* dx, int64_t lddx,
                            void* dw, int64_t dw_group_stride, int64_t lddw, void* workspace, size_t workspace_bytes, ct_stream_t stream) {
    if (!type_ok(type) || !(out_type == type || out_type == CT_F32) || rows < 0 || K <= 0 || N <= 0 || G <= 0 || !offsets) return CT_EINVAL;
    if ((rows > 0 && !dy) || lddy < N || (dw && ((rows > 0 && !x) || ldx < K || lddw < N || dw_group_stride < (int64_t)(K - 1) * lddw + N))) return CT_EINVAL;
    if (dx && ((rows > 0 && !w) || ldw < (w_transposed ? K : N) || w_group_stride < 0 || lddx < K)) return CT_EINVAL;
    if (lddy > kMaxStride || (dw && ldx > kMaxStride) || (dx && ldw > kMaxStride)) return CT_ESHAPE;
    hipStream_t st = (hipStream_t)stream;
    int rc = CT_OK;
    if (dw) rc = dw_any(type, DwP{x, ldx, rows, K, dy, lddy, N, offsets, G, dw, dw_group_stride, lddw, out_type == CT_F32, 0, 0, 0}, st);
    if (rc == CT_OK && dx && rows > 0)
        rc = product_any(type, ProductP{dy, lddy, rows, N, w, w_group_stride, ldw, K, offsets, G, nullptr, nullptr, 0, 1.f, 1, type == CT_F32, dx, lddx, 0, 0, 0},
                         !w_transposed, st);
    return rc;
}

}  // extern "C"
