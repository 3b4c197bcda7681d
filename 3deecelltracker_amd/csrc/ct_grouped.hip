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
//
// What bounds it, and what was chosen for it (measured on MI355X; a copy runs at 5.1 TB/s there, a library product of 8192^3 at 1189 TFLOP/s in bf16
// and 153 in fp32):
//   * large groups, 16 bit: the matrix pipe (55 % busy) and, next to it, LDS.  256 x 256 tiles of 8 waves, two 64 KB stages filled by direct loads:
//     32768 x 4096 x 2048 in 16 uneven groups 571 us = 963 TFLOP/s (542 to 579 over machines and group sizes; 128 x 128 tiles 620), the gradients of
//     16384 x 2048 x 1536 in 16 groups 270 us, 244 if the groups are even.
//   * a few rows a group: the weights, each read once.  16 x 64 tiles, every wave a quarter of a stage's sum: 64 rows of 2048 x 1024 blocks 27 to 34 us
//     for the 30 to 40 blocks that have rows, 40 us with all 64 (6.7 TB/s).
//   * in between: bytes from L2 to LDS (about 9.5 TB/s) and the latency of a stage; what helped was more workgroups on a CU, so two stages rather than three
//     or four wherever the tiles fill the CUs (8192 x 1024 x 1024 fp32, 64 x 64 tiles: 144 us with two, 152 with three, 161 with four), and deep or wide
//     stages where they do not (40 x 2048 x 2048 fp16: 12.3 -> 6.5 us with 8 waves sharing a 256-deep stage).
//   * fp32 goes through the exact fp32 matrix instruction: 8192 x 1024 x 1024 at 132 TFLOP/s with 128 x 128 tiles.
//   * 12013 x 61 x 512 fp32 (20 us; with all but its stores, its products or its loads taken out of a copy of the kernel 6.3, 5.6, 5.4): the three hardly
//     overlap, since the workgroups of a CU start together; runs of column tiles, other tiles and deeper stages left it at 20 to 22 us.
//   * odd strides (16 bit): a direct load wants 4-byte addresses; through registers 3001 x 777 x 1111 fp16 takes 19.5 us, 776 x 1112 14.7 directly.
//   * many groups: every workgroup looks its group up, 64 at a time, and every group may add a row tile.  65536 x 64 x 64 bf16 takes 10 us in 64 groups, 23 in
//     1024, 379 in 8192 and 18.7 ms in 65536 of one row each: the look-up is all of it from a thousand groups on.
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

// ceil(n / step); n up to 2^31 - 1 (n + step may pass it)
__device__ __forceinline__ int pieces(int n, int step) { return (int)(((uint32_t)n + (uint32_t)(step - 1)) / (uint32_t)step); }
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
        const int tiles = pieces(e - b, step);
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
// Short rows have too few places for that: fp32 of 32 values two for four rows (19 % of the LDS cycles of the 32 x 32 product tiles are conflicts, 20 % in the
// 32 x 64 gradient tiles), 16 bit of 64 values four for eight (12 % in the 16 x 64 tiles); the 128 and 256 wide ones have none.
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

// The same straight into LDS: 16 bytes a lane, a wave fills 1 KB without a register; the source of a lane is the piece that stands where the lane writes.
// Sources have to be whole pieces (the address a multiple of 4 bytes); rows past the operand take the last one (their results are not stored).
// The instruction is written out because the compiler's own form makes it wait for all such loads before any read of LDS; Core waits for them.
// A load does not wait for a base that a v_readfirstlane has just written: that takes five wait states (s_mov and s_nop 3), which the compiler counts for
// its own loads only; scripts/check_sgpr_waits.py holds the built code to it.  m0 is reserved, so a clobber of it means nothing to the compiler: it sets m0
// itself right before an instruction of its own that reads it, of which these kernels have none (a test counts them).
__device__ __forceinline__ void direct16(const void* base, uint32_t voff, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %1, %2" :: "s"(lds), "v"(voff), "s"(base) : "memory");
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
// up through LDS at the end, in order.  NB stages in LDS (2 through registers): NB - 1 are in flight while one is multiplied.
template <typename TT, bool ACC, bool BCC, int BM, int BN, int BK, int WM, int WN, int WK, int NB, Way WAY>
struct Core {
    typedef typename TT::S S;
    static constexpr bool H = sizeof(S) == 2;
    static constexpr int NT = 64 * WM * WN * WK, SM = BM / WM / 16, SN = BN / WN / 16, KS = H ? 32 : 16, PK = BK / WK;
    static_assert(PK % KS == 0 && (PK == KS || PK % (2 * KS) == 0) && SM * 16 * WM == BM && SN * 16 * WN == BN, "whole strips");
    typedef Tile<S, ACC, BM, BK> TA;
    typedef Tile<S, BCC, BN, BK> TB;
    static constexpr int STAGE_BYTES = TA::BYTES + TB::BYTES, SUM_BYTES = WK > 1 ? BM * BN * WK * 4 : 0;
    static constexpr int LDS_BYTES = NB * STAGE_BYTES > SUM_BYTES ? NB * STAGE_BYTES : SUM_BYTES;
    static_assert(WAY == DIRECT || NB == 2, "registers hold one stage");
    // fp32 sums of one wave run over at most kChain steps and are then added to the total: a long chain loses a bit for every fourfold length (7542 x 2809 x
    // 708: 3.9e-7 of the norm, 9.3e-7 as one chain; 2^20 rows in four chains 9.2e-6, 8.4e-7 folded, and a hundred times that for values of one sign).
    // Waves that share a sum fold later, theirs is a quarter or an eighth of it.  A sum that is never folded has no total to carry: a loop of its own.
    // 16-bit operands carry no more than 11 bits: their sums stay one chain of 32 bits (the totals of 256 x 256 tiles would not fit the registers).
    static constexpr int kChain = WK == 1 ? 512 : 2048, kFold = kChain / PK;
    static constexpr bool FOLD = !H;
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
            if constexpr (H) {
#pragma unroll
                for (int i = 0; i < SN; ++i)
#pragma unroll
                    for (int j = 0; j < SM; ++j) acc[i][j] = mfma(TT{}, fb[i], fa[j], acc[i][j]);
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k)                             // (the four of one strip depend on each other: the other strips' stand between them)
#pragma unroll
                    for (int i = 0; i < SN; ++i)
#pragma unroll
                        for (int j = 0; j < SM; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(fb[i][k], fa[j][k], acc[i][j], 0, 0, 0);
            }
        }
    }

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < SN; ++i)
#pragma unroll
            for (int j = 0; j < SM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    // Parts of the sum meet in LDS; wave kz goes on with every WK-th strip
    __device__ __forceinline__ void join(unsigned char* smem, int kz) {
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

    // `tiles` tiles with the same A one after the other: tile i has B(i) -- element (0 of the tile, contraction step 0), n_have(i) rows-or-columns of it
    // existing from there -- and done(i) takes its sums.  m_have rows-or-columns of A exist; rows of A and B (where m or n is contiguous) have
    // len_a, len_b values.  The steps [begin, end) of `extent` are summed.  More than one tile only if MANY, with DIRECT and WK = 1.
    template <bool MANY, typename FB, typename FN, typename FD>
    __device__ __forceinline__ void run(unsigned char* smem, const S* A, uint32_t lda, int m_have, int len_a, int tiles, FB B, uint32_t ldb, FN n_have, int len_b,
                                        int begin, int end, int extent, FD done) {
        int m0, n0, kz;
        place(m0, n0, kz);
        ra.init(m0, kz * PK); rb.init(n0, kz * PK);
        clear();
        const int stages = pieces(end - begin, BK);
        const int full = WAY == EDGE ? stages : (end - begin) / BK;             // stages all of whose steps count; one more may follow
        auto from = [&](int t) { const int c = begin + t * BK; return WAY == EDGE || c <= extent - BK ? c : extent - BK; };
        auto pa = [&](int t) { return A + (ACC ? (int64_t)from(t) : (int64_t)from(t) * lda); };
        auto pb = [&](int i, int t) { return B(i) + (BCC ? (int64_t)from(t) : (int64_t)from(t) * ldb); };
        // multiplies the stages of one tile: stretch(t, stop) those up to `stop`, rest(t) the others and the last one
        auto folded = [&](int& t, auto stretch, auto rest) {
            if constexpr (FOLD) {
                if (full > kFold) {
                    f32x4 total[SN][SM];
#pragma unroll
                    for (int i = 0; i < SN; ++i)
#pragma unroll
                        for (int j = 0; j < SM; ++j) total[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
                    do {
                        stretch(t, t + kFold);
#pragma unroll
                        for (int i = 0; i < SN; ++i)
#pragma unroll
                            for (int j = 0; j < SM; ++j) total[i][j] += acc[i][j];
                        clear();
                    } while (full - t > kFold);
                    rest(t);
#pragma unroll
                    for (int i = 0; i < SN; ++i)
#pragma unroll
                        for (int j = 0; j < SM; ++j) acc[i][j] += total[i][j];
                    return;
                }
            }
            rest(t);
        };
        auto step = [&](int u) { multiply<false>(smem + u % NB * STAGE_BYTES, kz, 0, 0); };
        auto last = [&](int t, int u) { multiply<true>(smem + u % NB * STAGE_BYTES, kz, begin + t * BK - from(t), end - from(t)); };
        auto finish = [&](int i) {
            if constexpr (WK > 1) join(smem, kz);
            done(i);
        };
        static_assert(!MANY || (WAY == DIRECT && WK == 1), "the sums of one tile are joined where the next one's stages would stand");
        if constexpr (WAY == DIRECT) {
            Direct<S, ACC, BM, BK, NT> da;
            Direct<S, BCC, BN, BK, NT> db;
            da.init(lda, m_have); db.init(ldb, n_have(0));
            const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)smem;
            const int all = MANY ? tiles * stages : stages;
            int ti = 0, tt = 0;                                                 // the next stage to ask for: of tile ti its stage tt
            auto issue = [&](int u) {
                if (!MANY) tt = u;
                da.load(pa(tt), lds + u % NB * STAGE_BYTES);
                db.load(pb(ti, tt), lds + u % NB * STAGE_BYTES + TA::BYTES);
                if (MANY && ++tt == stages) { tt = 0; ++ti; }
            };
            // stage u is there and stage u - 1 has been read by all; of the stages after u, those that have been asked for may still be on their way
            auto landed = [&](int u) {
                constexpr int AHEAD = (NB - 2) * (decltype(da)::N + decltype(db)::N);
                static_assert(AHEAD < 64, "the counter of loads in flight has 6 bits");
                if (NB > 2 && u + NB - 2 < all) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(AHEAD) : "memory");
                else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            };
#pragma unroll
            for (int u = 0; u < NB - 1; ++u) if (u < all) issue(u);
            auto sum = [&](int u) {                                             // the stages of one tile, the first of them u
                int t = 0;
                auto stretch = [&](int& t, int stop) {
                    for (; t < stop; ++t, ++u) {
                        landed(u);
                        if (u + NB - 1 < all) issue(u + NB - 1);
                        step(u);
                    }
                };
                folded(t, stretch, [&](int& t) {
                    stretch(t, full);
                    if (full < stages) {
                        landed(u);
                        if (u + NB - 1 < all) issue(u + NB - 1);
                        last(full, u);
                    }
                });
            };
            if constexpr (MANY) {
                for (int i = 0; i < tiles; ++i) {
                    if (i) clear();
                    sum(i * stages);
                    finish(i);
                    __builtin_amdgcn_s_waitcnt(0x0f70);                         // vmcnt(0), said so that the compiler does not put it among the next tile's reads
                }
            } else {
                sum(0);
                finish(0);
            }
        } else {
            auto la = [&](int t) { return (S*)(smem + t % NB * STAGE_BYTES); };
            auto lb = [&](int t) { return (S*)(smem + t % NB * STAGE_BYTES + TA::BYTES); };
            Stage<S, ACC, BM, BK, NT, WAY == EDGE> sa;
            Stage<S, BCC, BN, BK, NT, WAY == EDGE> sb;
            const int n = n_have(0);
            auto load = [&](int t) {
                const int c = end - from(t);
                sa.load(pa(t), lda, ACC ? m_have : c, ACC ? c : m_have, ACC ? extent : len_a);
                sb.load(pb(0, t), ldb, BCC ? n : c, BCC ? c : n, BCC ? extent : len_b);
            };
            auto store = [&](int t) {
                const int c = end - from(t);
                sa.store(la(t), ACC ? m_have : c, ACC ? c : m_have, ACC ? extent : len_a);
                sb.store(lb(t), BCC ? n : c, BCC ? c : n, BCC ? extent : len_b);
            };
            if (stages > 0) { load(0); store(0); }
            __syncthreads();
            int t = 0;
            auto stretch = [&](int& t, int stop) {
                for (; t < stop; ++t) {
                    if (t + 1 < stages) load(t + 1);
                    step(t);
                    if (t + 1 < stages) store(t + 1);
                    __syncthreads();
                }
            };
            folded(t, stretch, [&](int& t) {
                stretch(t, full);
                if (full < stages) last(full, full);
            });
            finish(0);
        }
    }
    // for each column strip: col(n), then row(m, n, four neighbours along n)
    template <typename C, typename R> __device__ __forceinline__ void each(C col, R row) const {
        const int lane = threadIdx.x & 63, l16 = lane & 15, lk = lane >> 4;
        int m0, n0, kz;
        place(m0, n0, kz);
#pragma unroll
        for (int i = 0; i < SN; ++i) {
            col(n0 + 16 * i + 4 * lk);
#pragma unroll
            for (int j = 0; j < SM; ++j) {
                if (WK > 1 && (i * SM + j) % WK != kz) continue;
                row(m0 + 16 * j + l16, n0 + 16 * i + 4 * lk, acc[i][j]);
            }
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
__device__ __forceinline__ f32x4 load4(const float* p, int n, int have) {       // 4 neighbours; those past `have` repeat the last one
    typedef f32x4 loose4 __attribute__((aligned(4)));
    if (n + 4 <= have) return *reinterpret_cast<const loose4*>(p + n);
    f32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = p[n + i < have ? n + i : have - 1];
    return v;
}
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
    int slots, nt, per, count;               // row tiles (at most), runs of column tiles, column tiles in a run (at most), workgroups
};

// The last column tile is moved back so that it ends with the matrix (its first columns are then another tile's to store): whole pieces in every tile.
__device__ __forceinline__ int moved_back(int at, int tile, int extent) { return at + tile <= extent || extent < tile ? at : extent - tile; }

// A tile's shape and how it is worked: what Core is made of
template <int BM_, int BN_, int BK_, int WM_, int WN_, int WK_, int NB_, Way WAY_, int RUN_ = 1>
struct Shape {
    static constexpr int BM = BM_, BN = BN_, BK = BK_, NB = NB_, RUN = RUN_, THREADS = 64 * WM_ * WN_ * WK_, WK = WK_;
    static constexpr Way WAY = WAY_;
    template <typename TT, bool ACC, bool BCC> using Of = Core<TT, ACC, BCC, BM_, BN_, BK_, WM_, WN_, WK_, NB_, WAY_>;
};

template <typename TT, bool WT, typename Sh>
__device__ __forceinline__ void product_tile(const ProductP& p, int id, unsigned char* smem) {
    typedef typename TT::S S;
    typedef typename Sh::template Of<TT, true, WT> C;
    constexpr int BM = Sh::BM, BN = Sh::BN;
    // four row tiles side by side, then the next column tile: 32 numbers in a row touch 4 row panels and 8 column panels
    const int t = tile_number(id, p.count), strip = 4 * p.nt, s4 = t / strip, in = t - s4 * strip;
    const int wide = p.slots - 4 * s4 < 4 ? p.slots - 4 * s4 : 4, col = in / wide, slot = 4 * s4 + in - col * wide;
    const Slot s = find_slot(p.off, p.G, p.rows, BM, slot, p.tail);
    if (s.group < 0) return;
    const int m_have = s.end - s.row, c0 = col * p.per, cols = (p.N + BN - 1) / BN, runs = cols - c0 < p.per ? cols - c0 : p.per;
    if (s.group == p.G) {                    // rows behind the last group
        const int n0 = c0 * BN, wide = p.N - n0 < runs * BN ? p.N - n0 : runs * BN, quads = (wide + 3) / 4;
        for (int i = threadIdx.x; i < BM * quads; i += C::NT) {
            const int m = i / quads, n = i % quads * 4;
            if (m < m_have) store_out<S>(p.y, (int64_t)(s.row + m) * p.ldy + n0 + n, p.out32, f32x4{0.f, 0.f, 0.f, 0.f}, 0, wide - n);
        }
        return;
    }
    const S* const w = (const S*)p.w + s.group * p.wg;
    const float* const sc = p.scale ? p.scale + s.group * p.ag : nullptr;
    const float* const sh = p.shift ? p.shift + s.group * p.ag : nullptr;
    auto begins = [&](int i) { return moved_back((c0 + i) * BN, BN, p.N); };
    C core;
    core.template run<(Sh::RUN > 1)>(smem, (const S*)p.x + (int64_t)s.row * p.ldx, (uint32_t)p.ldx, m_have, p.K, runs,
             [&](int i) { return w + (WT ? begins(i) * p.ldw : (int64_t)begins(i)); }, (uint32_t)p.ldw, [&](int i) { return p.N - begins(i); }, p.N, 0, p.K, p.K, [&](int i) {
        const int n0 = begins(i), first = (c0 + i) * BN - n0, n_have = p.N - n0;
        const int64_t at = (int64_t)s.row * p.ldy + n0;
        f32x4 a = {1.f, 1.f, 1.f, 1.f}, b = {0.f, 0.f, 0.f, 0.f};
        core.each([&](int n) {
            if (sc) a = load4(sc + n0, n, n_have);
            if (sh) b = load4(sh + n0, n, n_have);
        }, [&](int m, int n, f32x4 v) {
            if (m >= m_have || n >= n_have) return;
            if (sc) v *= a;
            if (sh) v += b;
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = v[k] >= 0.f ? v[k] : v[k] * p.slope;
            store_out<S>(p.y, at + m * p.ldy + n, p.out32, v, first - n, n_have - n);
        });
    });
}

struct DwP {
    const void* x; int64_t ldx; int rows, K;
    const void* dy; int64_t lddy; int N;
    const int32_t* off; int G;
    void* dw; int64_t wg, ldw;
    float* part; int step, slots;            // a long sum in parts of `step` rows, [slot][K][N] (part NULL: no parts)
    int out32, mt, nt, count;
};

template <typename TT, typename Sh, bool PARTS>
__device__ __forceinline__ void dw_tile(const DwP& p, int id, unsigned char* smem) {
    typedef typename TT::S S;
    typedef typename Sh::template Of<TT, false, false> C;
    constexpr int BM = Sh::BM, BN = Sh::BN;
    const int tile = tile_number(id, p.count), g = tile / (p.mt * p.nt), t = tile - g * p.mt * p.nt;
    const int nom_m = (t / p.nt) * BM, m0 = moved_back(nom_m, BM, p.K), nom_n = (t % p.nt) * BN, n0 = moved_back(nom_n, BN, p.N);
    int b, e;
    if constexpr (PARTS) {                   // g is a part's number
        const Slot s = find_slot(p.off, p.G, p.rows, p.step, g, false);
        if (s.group < 0) return;
        b = s.row; e = s.end - s.row < p.step ? s.end : s.row + p.step;
    } else {
        b = clampi(fresh_i32(p.off + g), 0, p.rows); e = clampi(fresh_i32(p.off + g + 1), b, p.rows);
    }
    C core;
    core.template run<false>(smem, (const S*)p.x + m0, (uint32_t)p.ldx, p.K - m0, p.K, 1, [&](int) { return (const S*)p.dy + n0; }, (uint32_t)p.lddy, [&](int) { return p.N - n0; }, p.N, b, e,
             p.rows, [](int) {});
    if constexpr (PARTS) {
        float* const part = p.part + ((int64_t)g * p.K + m0) * p.N + n0;
        core.each([](int) {}, [&](int m, int n, f32x4 v) {
            if (m >= nom_m - m0 && m < p.K - m0 && n < p.N - n0) store4(part + (int64_t)m * p.N + n, v, nom_n - n0 - n, p.N - n0 - n);
        });
    } else {
        const int64_t at = g * p.wg + m0 * p.ldw + n0;
        core.each([](int) {}, [&](int m, int n, f32x4 v) {
            if (m >= nom_m - m0 && m < p.K - m0 && n < p.N - n0) store_out<S>(p.dw, at + m * p.ldw + n, p.out32, v, nom_n - n0 - n, p.N - n0 - n);
        });
    }
}

// Parts before group g, and its own
__device__ __forceinline__ int2 parts_of(const int32_t* __restrict__ off, int rows, int step, int g) {
    const int lane = threadIdx.x & 63;
    int before = 0, own = 0;
    for (int h = lane; h <= g; h += 64) {
        const int b = clampi(off[h], 0, rows), n = pieces(clampi(off[h + 1], b, rows) - b, step);
        if (h < g) before += n; else own = n;
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) { before += __shfl_xor(before, d); own += __shfl_xor(own, d); }
    return int2{before, own};
}
// dw[g] = the sum of its parts, in order
template <typename S>
__global__ __launch_bounds__(256) void join_kernel(const DwP p) {
    const int per = (p.K * p.N + 255) / 256, g = blockIdx.x / per;
    const int2 at = parts_of(p.off, p.rows, p.step, g);
    const int i = (blockIdx.x - g * per) * 256 + threadIdx.x;
    if (i >= p.K * p.N) return;
    const float* q = p.part + (int64_t)at.x * p.K * p.N + i;
    const int own = at.x + at.y <= p.slots ? at.y : p.slots - at.x;              // (offsets that do not rise can count more parts than there are)
    float v = 0.f;
#pragma unroll 8
    for (int s = 0; s < own; ++s) v += q[(int64_t)s * p.K * p.N];
    const int k = i / p.N;
    const int64_t to = g * p.wg + k * p.ldw + (i - k * p.N);
    if (p.out32) ((float*)p.dw)[to] = v; else ((S*)p.dw)[to] = (S)v;
}

template <typename TT, bool WT, typename Sh>
__global__ __launch_bounds__(Sh::THREADS) void product_kernel(const ProductP p) {
    __shared__ __attribute__((aligned(1024))) unsigned char smem[Sh::template Of<TT, true, WT>::LDS_BYTES];
    product_tile<TT, WT, Sh>(p, blockIdx.x, smem);
}
template <typename TT, typename Sh, bool PARTS>
__global__ __launch_bounds__(Sh::THREADS) void dw_kernel(const DwP p) {
    __shared__ __attribute__((aligned(1024))) unsigned char smem[Sh::template Of<TT, false, false>::LDS_BYTES];
    dw_tile<TT, Sh, PARTS>(p, blockIdx.x, smem);
}
// Both gradients in one launch: neither alone fills the card at the sizes of a network's layers, and one launch costs as much as a small product
template <typename TT, bool WT, typename ShX, typename ShW>
__global__ __launch_bounds__(ShX::THREADS) void grad_kernel(const ProductP x, const DwP w, int w_first) {
    constexpr int LX = ShX::template Of<TT, true, WT>::LDS_BYTES, LW = ShW::template Of<TT, false, false>::LDS_BYTES;
    __shared__ __attribute__((aligned(1024))) unsigned char smem[LX > LW ? LX : LW];
    const int id = blockIdx.x, ahead = w_first ? w.count : x.count;
    if ((id < ahead) == (w_first != 0)) dw_tile<TT, ShW, false>(w, w_first ? id : id - ahead, smem);
    else product_tile<TT, WT, ShX>(x, w_first ? id - ahead : id, smem);
}

constexpr int64_t kMaxBlocks = (1 << 22) - 1;               // a grid has fewer than 2^32 work items, a workgroup up to 512
constexpr int64_t kMaxStride = 1 << 22;                     // a tile's offsets fit 32 bits: 256 rows of 2^22 values
constexpr int kMaxWidth = 1 << 30;                          // a width and a tile's fit 32 bits
constexpr int64_t kCus = 256;
constexpr int kMaxGroups = 1 << 16;                         // every workgroup looks its group up among them, 64 at a time

bool type_ok(int t) { return t == CT_F32 || t == CT_BF16 || t == CT_F16; }
bool at_value(const void* p, int type) { return ((uintptr_t)p & (type == CT_F32 ? 3 : 1)) == 0; }
bool words(const void* p, int64_t ld, int64_t more, int size) { return (((uintptr_t)p | (uintptr_t)(ld * size) | (uintptr_t)(more * size)) & 3) == 0; }
int64_t tiles(int64_t m, int64_t n, int bm, int bn) { return ((m + bm - 1) / bm) * ((n + bn - 1) / bn); }

// Workgroups of a launch; CT_ESHAPE: too many; CT_EINVAL: a tile would reach outside its operands, which the rules below never ask for
template <bool WT, typename Sh>
int plan(ProductP& p) {
    if (Sh::WAY != EDGE && (p.K < Sh::BK || (!WT && p.N < Sh::BN))) return CT_EINVAL;
    const int cols = (p.N + Sh::BN - 1) / Sh::BN;
    p.per = Sh::RUN < cols ? Sh::RUN : cols;
    p.nt = (cols + p.per - 1) / p.per;
    const int64_t slots = (int64_t)p.rows / Sh::BM + (p.rows < p.G + 1 ? p.rows : p.G + 1);     // sum of ceil(rows_g / BM) is no more
    if (slots * p.nt > kMaxBlocks) return CT_ESHAPE;
    p.slots = (int)slots; p.count = (int)(slots * p.nt);
    return CT_OK;
}
template <typename Sh>
int plan(DwP& p) {
    if (Sh::WAY != EDGE && (p.rows < Sh::BK || p.K < Sh::BM || p.N < Sh::BN)) return CT_EINVAL;
    p.mt = (p.K + Sh::BM - 1) / Sh::BM; p.nt = (p.N + Sh::BN - 1) / Sh::BN;
    const int64_t count = (int64_t)(p.part ? p.slots : p.G) * p.mt * p.nt;
    if (count > kMaxBlocks) return CT_ESHAPE;
    p.count = (int)count;
    return CT_OK;
}
template <typename TT, bool WT, typename Sh>
int launch(ProductP p, hipStream_t st) {
    const int rc = plan<WT, Sh>(p);
    if (rc != CT_OK) return rc;
    hipLaunchKernelGGL((product_kernel<TT, WT, Sh>), dim3((unsigned)p.count), dim3(Sh::THREADS), 0, st, p);
    return (int)hipGetLastError();
}
template <typename TT, typename Sh, bool PARTS = false>
int launch(DwP p, hipStream_t st) {
    const int rc = plan<Sh>(p);
    if (rc != CT_OK) return rc;
    hipLaunchKernelGGL((dw_kernel<TT, Sh, PARTS>), dim3((unsigned)p.count), dim3(Sh::THREADS), 0, st, p);
    return (int)hipGetLastError();
}
template <typename TT, bool WT, typename ShX, typename ShW>
int launch(ProductP x, DwP w, hipStream_t st) {
    static_assert(ShX::THREADS == ShW::THREADS, "one launch");
    int rc = plan<WT, ShX>(x);
    if (rc == CT_OK) rc = plan<ShW>(w);
    if (rc != CT_OK) return rc;
    if ((int64_t)x.count + w.count > kMaxBlocks) return CT_ESHAPE;
    const int w_first = (int64_t)w.rows > (int64_t)w.G * x.K;       // the longer sums begin first: mean rows of a group against the width of dy
    hipLaunchKernelGGL((grad_kernel<TT, WT, ShX, ShW>), dim3((unsigned)(x.count + w.count)), dim3(ShX::THREADS), 0, st, x, w, w_first);
    return (int)hipGetLastError();
}

// Shapes (tile, contraction steps of a stage, waves along m, n and the contraction, stages).  Two stages where tiles fill the CUs, for more workgroups on each.
template <Way W> using T256 = Shape<256, 256, 64, 2, 4, 1, 2, W>;
template <Way W> using T128 = Shape<128, 128, 64, 2, 4, 1, 2, W>;
using T128run = Shape<128, 128, 64, 2, 4, 1, 2, DIRECT, 4>;
using T128deep = Shape<128, 128, 64, 2, 4, 1, 4, DIRECT>;
template <Way W> using T64 = Shape<64, 64, 64, 2, 2, 1, 2, W>;
using T64deep = Shape<64, 64, 64, 2, 2, 1, 4, DIRECT>;
template <Way W> using T64flat = Shape<64, 64, 32, 2, 2, 1, 2, W>;
using T32 = Shape<32, 64, 128, 1, 2, 2, 2, DIRECT>;
using T32k = Shape<32, 32, 256, 1, 1, 8, 3, DIRECT>;
using T32s = Shape<32, 32, 128, 1, 1, 4, 3, DIRECT>;
using T16 = Shape<16, 64, 128, 1, 1, 4, 4, DIRECT>;
using T16r = Shape<16, 64, 128, 1, 1, 4, 2, REGS>;
using F128 = Shape<128, 128, 32, 2, 4, 1, 2, DIRECT>;
using F64 = Shape<64, 64, 32, 2, 4, 1, 2, DIRECT>;
using F32 = Shape<32, 64, 64, 1, 1, 4, 2, DIRECT>;
using F32s = Shape<32, 32, 64, 1, 1, 4, 2, DIRECT>;
using F16 = Shape<16, 64, 128, 1, 1, 4, 2, DIRECT>;
using F16k = Shape<16, 32, 128, 1, 1, 8, 3, DIRECT>;
using R64k = Shape<64, 64, 128, 2, 2, 2, 2, REGS>;
using R32k = Shape<32, 32, 256, 1, 1, 8, 2, REGS>;
using Any = Shape<64, 64, 32, 2, 2, 1, 2, EDGE>;
template <int BK> using AnyK = Shape<32, 32, BK, 1, 1, 8, 2, EDGE>;

// Which tile, by the rows a group has on average, the widths, and how many tiles that makes for 256 CUs.  Large tiles fetch each value less often, small
// ones fill the card.  us, the chosen shape and the next best:
//   16 bit   T256    32768 x 4096 x 2048, 16 groups   572 : 620 (128 x 128)        T128     8000 x 1024 x 1024, 8 groups    24.7 : 32.3 (128 x 64)
//            T128run 30000 x 64 x 1024, 10 groups    25.2 : 30.1 (T128)            T128deep 3001 x 1112 x 776, 7 groups     19.6 : 20.9 (128 x 64)
//            T64deep 500 x 2048 x 2048, 8 groups     15.5 : 20.8 (T64), 25.4 (T128) T64      8000 x 1024 x 1024, 8 groups    36.4 : 40.8 (T64deep)
//            T32     1000 x 512 x 512, 4 groups       5.5 : 6.2 (T64)              T32k     100 x 3000 x 300, 4 groups       8.4 : 11.8 (T32)
//            T32s    500 x 500 x 200, 30 groups       5.1 : 5.7 (T32)              T16      16 x 4096 x 512, 8 groups       11.3 : 13.9 (256-deep, two stages)
//   fp32     F128    8192 x 1024 x 1024, 8 groups     131 : 136 (F64)              F64      3000 x 200 x 1500, 3 groups     28.0 : 29.6 (4 waves), 33.2 (F32)
//            F32     2048 x 512 x 512, 2 groups      13.3 : 14.3 (F32s)            F32s     1213 x 512 x 512, 2 groups      11.6 : 13.2 (F32)
//            F16k    30 x 4000 x 100, 2 groups       18.7 : 28.3 (F32s)            F16      64 x 2048 x 256, 64 groups      24.1 : 26.3 (F32s)
//   odd      T128    3001 x 777 x 1111 fp16, 7 groups 18.3 : 21.0 (128 x 64)       R64k     500 x 2047 x 2047 fp16, 8 groups 22.7 : 28.7 (T64)
//   any      AnyK    2 x 3181 x 16 fp32, 3 groups      37 : 138 (Any)
template <typename TT, bool WT, Way WAY>
int product_pick(const ProductP& p, hipStream_t st) {
    const int64_t mean = ((int64_t)p.rows + p.G - 1) / p.G, r = (int64_t)p.rows + p.G * 32;       // (a group's last tile is half full on average)
    const int k = p.K, n = WT ? 1 << 30 : p.N;              // what the tile must not exceed: rows of w may be repeated, columns may not
    if constexpr (WAY == DIRECT && sizeof(typename TT::S) == 2) {
        const int64_t t128 = tiles(r, p.N, 128, 128), t64 = tiles(r, p.N, 64, 64);
        const int64_t t32 = tiles(r, p.N, 32, 32);
        if (k >= 512 && n >= 32 && t32 < 2 * kCus) return launch<TT, WT, T32k>(p, st);
        if (k >= 128 && n >= 32 && t32 < 2 * kCus) return launch<TT, WT, T32s>(p, st);
        if (mean <= 16 && k >= 128 && n >= 64) return launch<TT, WT, T16>(p, st);
        if (mean >= 192 && k >= 64 && p.N >= 256 && tiles(r, p.N, 256, 256) >= kCus) return launch<TT, WT, T256<DIRECT>>(p, st);
        if (mean >= 96 && k >= 64 && p.N >= 128 && t128 >= kCus) return k <= 128 && t128 >= 4 * kCus ? launch<TT, WT, T128run>(p, st) : launch<TT, WT, T128<DIRECT>>(p, st);
        if (mean >= 96 && k >= 256 && p.N >= 128 && t128 >= 160) return launch<TT, WT, T128deep>(p, st);
        if (k >= 128 && n >= 64 && t64 < 160) return launch<TT, WT, T32>(p, st);
        if (k >= 256 && n >= 64 && t64 <= 2 * kCus) return launch<TT, WT, T64deep>(p, st);
        if (k >= 64 && n >= 64) return launch<TT, WT, T64<DIRECT>>(p, st);
        if (k >= 32 && n >= 64) return launch<TT, WT, T64flat<DIRECT>>(p, st);
    }
    if constexpr (WAY == REGS && sizeof(typename TT::S) == 2) {
        if (k >= 512 && n >= 32 && tiles(r, p.N, 32, 32) < 2 * kCus) return launch<TT, WT, R32k>(p, st);
        if (mean <= 16 && k >= 128 && n >= 64) return launch<TT, WT, T16r>(p, st);
        if (mean >= 96 && k >= 64 && p.N >= 128 && tiles(r, p.N, 128, 128) >= 160) return launch<TT, WT, T128<REGS>>(p, st);
        if (k >= 512 && n >= 64 && tiles(r, p.N, 64, 64) <= 2 * kCus) return launch<TT, WT, R64k>(p, st);
        if (k >= 64 && n >= 64) return launch<TT, WT, T64<REGS>>(p, st);
        if (k >= 32 && n >= 64) return launch<TT, WT, T64flat<REGS>>(p, st);
    }
    if constexpr (WAY == DIRECT && sizeof(typename TT::S) == 4) {
        const int64_t t64 = tiles(r, p.N, 64, 64);
        if (k >= 128 && n >= 32 && tiles(r, p.N, 16, 32) < kCus) return launch<TT, WT, F16k>(p, st);
        if (mean <= 16 && k >= 128 && n >= 64) return launch<TT, WT, F16>(p, st);
        if (mean >= 96 && k >= 32 && p.N >= 128 && tiles(r, p.N, 128, 128) >= 2 * kCus) return launch<TT, WT, F128>(p, st);
        if (k >= 64 && n >= 64 && t64 < 2 * kCus && t64 >= kCus) return launch<TT, WT, F32>(p, st);
        if (k >= 64 && n >= 32 && t64 < kCus) return launch<TT, WT, F32s>(p, st);
        if (k >= 32 && n >= 64) return launch<TT, WT, F64>(p, st);
    }
    // narrower than any tile above: long sums in wide stages over 8 waves
    if (k >= 512 && tiles(r, p.N, 32, 32) < 2 * kCus) return launch<TT, WT, AnyK<1024 / (int)sizeof(typename TT::S)>>(p, st);
    return launch<TT, WT, Any>(p, st);
}
// Few tiles with long sums: rows a part (0: the sums stay whole).  us of the kernels in parts and whole (a call on its own pays 6 us more on the host for the
// second launch and the workspace): 61 x 512 weights from 2048 rows in one group 8.9 : 16.1, from 20000 26 : 147; 512 x 1 from 1024 10.4 : 38.9; 61 x 512 from
// 600 8.0 : 6.9.  From 64 tiles on whole sums are faster: 512 x 512 in 2 groups from 1024 rows each (128 tiles), both gradients, 27.5 whole, 35.3 in parts.
int part_rows(int rows, int K, int N, int G) {
    const int64_t blocks = G * tiles(K, N, 64, 64), mean = rows / G;
    if (blocks >= 64 || mean < 512) return 0;
    const int64_t want = (2 * kCus + blocks - 1) / blocks, step = ((mean + want - 1) / want + 63) / 64 * 64;
    return (int)(step < 128 ? 128 : step);
}
int part_slots(int rows, int step, int G) { return rows / step + (rows < G ? rows : G); }

// (128 x 128: 516 x 1022 in 9 groups, 2999 rows 12.1 us, 16.1 with 64 x 64; T64deep: 128 x 256 in 10 groups, 20000 rows 12.3 : 18.7 (T64))
template <typename TT, Way WAY>
int dw_pick(const DwP& p, hipStream_t st) {
    const int r = p.rows, k = p.K, n = p.N;
    if (p.part) {
        int rc;
        if (sizeof(typename TT::S) == 2 && k >= 64 && n >= 64) rc = launch<TT, std::conditional_t<sizeof(typename TT::S) == 2, T64<WAY>, Any>, true>(p, st);
        else if (sizeof(typename TT::S) == 4 && k >= 32 && n >= 32) rc = launch<TT, std::conditional_t<sizeof(typename TT::S) == 4, F32s, Any>, true>(p, st);
        else rc = launch<TT, Any, true>(p, st);
        if (rc != CT_OK) return rc;
        hipLaunchKernelGGL((join_kernel<typename TT::S>), dim3((unsigned)(p.G * ((p.K * p.N + 255) / 256))), dim3(256), 0, st, p);
        return (int)hipGetLastError();
    }
    if constexpr (sizeof(typename TT::S) == 2) {
        if constexpr (WAY == DIRECT)
            if (r >= 64 && k >= 256 && n >= 256 && p.G * tiles(k, n, 256, 256) >= kCus) return launch<TT, T256<WAY>>(p, st);
        if (r >= 64 && k >= 128 && n >= 128 && p.G * tiles(k, n, 128, 128) >= 160) return launch<TT, T128<WAY>>(p, st);
        if constexpr (WAY == DIRECT)
            if (r >= 256 && k >= 64 && n >= 64 && p.G * tiles(k, n, 64, 64) < kCus) return launch<TT, T64deep>(p, st);
        if (r >= 64 && k >= 64 && n >= 64) return launch<TT, T64<WAY>>(p, st);
    }
    if constexpr (WAY == DIRECT && sizeof(typename TT::S) == 4) {
        if (r >= 32 && k >= 128 && n >= 128 && p.G * tiles(k, n, 128, 128) >= 2 * kCus) return launch<TT, F128>(p, st);
        if (r >= 64 && k >= 32 && n >= 32 && p.G * tiles(k, n, 64, 64) < 2 * kCus) return launch<TT, F32s>(p, st);
        if (r >= 32 && k >= 64 && n >= 64) return launch<TT, F64>(p, st);
    }
    return launch<TT, Any>(p, st);
}
// Both gradients together where one shape suits them (2999 x 515 x 1021 fp16 in 9 groups: 17.3 + 16.3 us apart, 27.1 together; 200 x 300 x 500 fp16 in 30
// groups 12.4 apart, 8.3 together; the worst found is 300 x 128 x 1000 fp32 in 40 groups, 22.5 and 24.6, with 2.2 us less on the host); x: dx as a product (its K is the width of dy, its N the width of x)
template <typename TT, bool WT, Way WAY>
int grad_pick(const ProductP& x, const DwP& w, hipStream_t st) {
    const int64_t mean = ((int64_t)x.rows + x.G - 1) / x.G, r = (int64_t)x.rows + x.G * 32;
    auto sum = [&](int t) { return tiles(r, x.N, t, t) + w.G * tiles(w.K, w.N, t, t); };
    const int least = w.part ? 0 : w.K < w.N ? w.K : w.N;   // both widths bound a tile of dw
    auto apart = [&] {
        const int rc = dw_pick<TT, WAY>(w, st);             // (also a sum in parts)
        return rc == CT_OK ? product_pick<TT, WT, WAY>(x, st) : rc;
    };
    // One shape for both, unless it starves one of them, which apart would get tiles of its own:
    //   long sums in few tiles of dw    16384 x 512 x 512 fp32 in 1 group 1053 us together, 199 apart (16 tiles); 16384 x 1024 x 1024 in 2 groups 623 : 558 (128);
    //                                   4096 x 1024 x 1024 in 8 groups, shorter sums, 135 : 144; bf16 16384 x 512 x 512 161 : 90 (16), in 8 groups 31 : 35 (128)
    //   fp32, few tiles of dx           1024 x 1024 x 1024 in 8 groups 79 : 49 (80 tiles, 512 of dw), 1024 x 2048 x 1536 in 8 groups 164 : 132 (160);
    //                                   1024 x 512 x 512 in 8 groups, small enough for one launch to pay, 15 : 19
    auto both = [&](auto shape) {
        typedef decltype(shape) Sh;
        const int64_t tx = tiles(r, x.N, Sh::BM, Sh::BN), tw = w.G * tiles(w.K, w.N, Sh::BM, Sh::BN);
        constexpr bool H = sizeof(typename TT::S) == 2;
        if (mean >= 2048 && tw < (H ? kCus / 4 : kCus * 3 / 4)) return apart();
        if (!H && Sh::BM >= 64 && tx <= kCus * 5 / 8 && tw >= kCus * 3 / 2 && (int64_t)x.rows * w.K * w.N >= 1 << 28) return apart();
        return launch<TT, WT, Sh, Sh>(x, w, st);
    };
    if constexpr (WAY == DIRECT && sizeof(typename TT::S) == 2)
        if (mean >= 192 && least >= 256 && sum(256) >= 2 * kCus) return both(T256<WAY>{});
    if constexpr (sizeof(typename TT::S) == 2) {
        if (mean >= 96 && least >= 128 && sum(128) >= kCus) return both(T128<WAY>{});
        if (x.rows >= 64 && least >= 64) return both(T64<WAY>{});
    }
    if constexpr (WAY == DIRECT && sizeof(typename TT::S) == 4) {
        if (mean >= 96 && least >= 128 && sum(128) >= 2 * kCus) return both(F128{});
        if (x.rows >= 64 && least >= 64) {
            // 32 x 64 tiles (48 KB: 3 on a CU) where they all run at once (with the least tiles that so many rows make; the groups' ends are not known here)
            // and fill it: 2048 x 512 x 512 in 2 groups (768 tiles) 22.2 us, 26.3 with 32 x 32; 2080 rows (784) 29.3, 27.4 with 32 x 32;
            // 2048 x 256 x 256 in 16 groups (768) 11.1 and 11.6; 500 x 200 x 1000 in 4 groups 16.9, 12.8 with 32 x 32
            const int64_t n64 = tiles(r, x.N, 32, 64) + w.G * tiles(w.K, w.N, 32, 64), least64 = tiles(x.rows, x.N, 32, 64) + w.G * tiles(w.K, w.N, 32, 64);
            if (sum(64) >= 2 * kCus && n64 > 4 * kCus) return both(F64{});
            if (n64 >= 2 * kCus && least64 <= 3 * kCus) return both(F32{});
            return both(F32s{});
        }
    }
    return apart();
}

// direct loads want addresses that are multiples of 4 bytes (16-bit values: an even stride, and an even width where the last tile is moved back);
// fp32 always has them
template <typename TT> constexpr Way other() { return sizeof(typename TT::S) == 2 ? REGS : DIRECT; }
template <typename TT>
int product_run(const ProductP& p, bool wt, hipStream_t st) {
    constexpr int size = sizeof(typename TT::S);
    const bool direct = words(p.x, p.ldx, p.K, size) && words(p.w, p.ldw, p.wg, size) && (wt || p.N % 2 == 0);
    if (size == 4 || direct) return wt ? product_pick<TT, true, DIRECT>(p, st) : product_pick<TT, false, DIRECT>(p, st);
    return wt ? product_pick<TT, true, other<TT>()>(p, st) : product_pick<TT, false, other<TT>()>(p, st);
}
template <typename TT>
int dw_run(const DwP& p, hipStream_t st) {
    constexpr int size = sizeof(typename TT::S);
    if (size == 4 || (words(p.x, p.ldx, p.K, size) && words(p.dy, p.lddy, p.N, size))) return dw_pick<TT, DIRECT>(p, st);
    return dw_pick<TT, other<TT>()>(p, st);
}
template <typename TT>
int grad_run(const ProductP& x, const DwP& w, bool wt, hipStream_t st) {
    constexpr int size = sizeof(typename TT::S);
    const bool direct = words(w.x, w.ldx, w.K, size) && words(w.dy, w.lddy, w.N, size) && words(x.w, x.ldw, x.wg, size);
    if (size == 4 || direct) return wt ? grad_pick<TT, true, DIRECT>(x, w, st) : grad_pick<TT, false, DIRECT>(x, w, st);
    return wt ? grad_pick<TT, true, other<TT>()>(x, w, st) : grad_pick<TT, false, other<TT>()>(x, w, st);
}

int product_any(int type, const ProductP& p, bool wt, hipStream_t st) {
    return type == CT_F32 ? product_run<FF>(p, wt, st) : type == CT_BF16 ? product_run<BF>(p, wt, st) : product_run<HF>(p, wt, st);
}
int dw_any(int type, const DwP& p, hipStream_t st) { return type == CT_F32 ? dw_run<FF>(p, st) : type == CT_BF16 ? dw_run<BF>(p, st) : dw_run<HF>(p, st); }
int grad_any(int type, const ProductP& x, const DwP& w, bool wt, hipStream_t st) {
    return type == CT_F32 ? grad_run<FF>(x, w, wt, st) : type == CT_BF16 ? grad_run<BF>(x, w, wt, st) : grad_run<HF>(x, w, wt, st);
}

}  // namespace

extern "C" {

int ct_grouped_product(int type, int out_type, const void* x, int64_t ldx, int rows, int K, const void* w, int64_t w_group_stride, int64_t ldw,
                       int w_transposed, int N, const int32_t* offsets, int G, const float* scale, const float* shift, int64_t affine_stride,
                       float slope, int fill_tail, void* y, int64_t ldy, ct_stream_t stream) {
    if (!type_ok(type) || !(out_type == type || out_type == CT_F32) || rows < 0 || K <= 0 || N <= 0 || G <= 0) return CT_EINVAL;
    if (rows == 0) return CT_OK;
    if (!offsets || !y || !x || !w || ldy < N || ldx < K || ldw < (w_transposed ? K : N) || w_group_stride < 0 || affine_stride < 0) return CT_EINVAL;
    if (!at_value(x, type) || !at_value(w, type) || !at_value(y, out_type) || !at_value(offsets, CT_F32) || !at_value(scale, CT_F32) || !at_value(shift, CT_F32)) return CT_EINVAL;
    if (ldx > kMaxStride || ldw > kMaxStride || G > kMaxGroups || K > kMaxWidth || N > kMaxWidth) return CT_ESHAPE;
    const ProductP p{x, ldx, rows, K, w, w_group_stride, ldw, N, offsets, G, scale, shift, affine_stride, slope, fill_tail != 0, out_type == CT_F32, y, ldy, 0, 0, 0, 0};
    return product_any(type, p, w_transposed != 0, (hipStream_t)stream);
}

size_t ct_grouped_product_grad_workspace_bytes(int type, int rows, int K, int N, int G) {
    if (!type_ok(type) || rows <= 0 || K <= 0 || N <= 0 || G <= 0) return 0;
    const int step = part_rows(rows, K, N, G);
    return step ? (size_t)part_slots(rows, step, G) * K * N * sizeof(float) : 0;
}

int ct_grouped_product_grad(int type, int out_type, const void* dy, int64_t lddy, const void* x, int64_t ldx, int rows, int K, const void* w,
                            int64_t w_group_stride, int64_t ldw, int w_transposed, int N, const int32_t* offsets, int G, void* dx, int64_t lddx,
                            void* dw, int64_t dw_group_stride, int64_t lddw, void* workspace, size_t workspace_bytes, ct_stream_t stream) {
    if (!type_ok(type) || !(out_type == type || out_type == CT_F32) || rows < 0 || K <= 0 || N <= 0 || G <= 0 || !offsets) return CT_EINVAL;
    if ((rows > 0 && !dy) || lddy < N || (dw && ((rows > 0 && !x) || ldx < K || lddw < N || dw_group_stride < (int64_t)(K - 1) * lddw + N))) return CT_EINVAL;
    if (dx && ((rows > 0 && !w) || ldw < (w_transposed ? K : N) || w_group_stride < 0 || lddx < K)) return CT_EINVAL;
    if (!at_value(dy, type) || !at_value(offsets, CT_F32) || (dw && (!at_value(x, type) || !at_value(dw, out_type))) || (dx && (!at_value(w, type) || !at_value(dx, type)))) return CT_EINVAL;
    if (G > kMaxGroups || K > kMaxWidth || N > kMaxWidth || lddy > kMaxStride || (dw && ldx > kMaxStride) || (dx && ldw > kMaxStride)) return CT_ESHAPE;
    hipStream_t st = (hipStream_t)stream;
    const ProductP px{dy, lddy, rows, N, w, w_group_stride, ldw, K, offsets, G, nullptr, nullptr, 0, 1.f, 1, type == CT_F32, dx, lddx, 0, 0, 0, 0};
    const int step = dw && rows > 0 ? part_rows(rows, K, N, G) : 0;
    if (step && (!workspace || ((uintptr_t)workspace & 3))) return CT_EINVAL;
    if (step && workspace_bytes < ct_grouped_product_grad_workspace_bytes(type, rows, K, N, G)) return CT_EWORKSPACE;
    const DwP pw{x, ldx, rows, K, dy, lddy, N, offsets, G, dw, dw_group_stride, lddw, step ? (float*)workspace : nullptr, step, step ? part_slots(rows, step, G) : 0,
                 out_type == CT_F32, 0, 0, 0};
    if (dx && dw && rows > 0) return grad_any(type, px, pw, !w_transposed, st);
    if (dx && rows > 0) return product_any(type, px, !w_transposed, st);
    return dw ? dw_any(type, pw, st) : CT_OK;
}

}  // extern "C"
