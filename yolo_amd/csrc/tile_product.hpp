// Tile products on the matrix cores (gfx950): D = A * B' for two operands whose rows lie along the
// contraction, 128 bytes of a row at a time.  Three arithmetics share the data path, since a lane's
// share of a fragment is 16 bytes in all:
//
//   MathI8     a 128-byte block of a row is 128 signed bytes; two 16x16x64 products per 16x16
//              piece of D, exact in int32.
//   MathSplit  a block is 32 numbers in two halves: 64 bytes of their leading parts (fp16), then 64
//              bytes of what fp16 leaves over (fp16 again): x = hi + lo to 22 bits.  Three 16x16x32
//              products, hi*hi + hi*lo + lo*hi, in fp32; lo*lo is below 2^-22 of the product.
//   MathHalf   a block is 64 fp16 numbers; two 16x16x32 products.
//
// Lane l of a wavefront holds, of a 16-row fragment, row l % 16 and the bytes 16 * (l / 16) .. + 15 of a
// 64-byte half; D's piece has row (first operand) 4 * (l / 16) + r in register r and column (second
// operand) l % 16.
//
// A tile row is 128 bytes in LDS, its eight 16-byte chunks exchanged by chunk ^ (row % 8), so the 16
// rows a fragment read touches spread over all banks.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace yh {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));

struct MathI8 {
    using Acc = v4i;
    static constexpr int PASSES = 2;
    template <int PASS> static __device__ __forceinline__ void mma(Acc& d, const v4i (&p)[2], const v4i (&q)[2]) {
        d = __builtin_amdgcn_mfma_i32_16x16x64_i8(p[PASS], q[PASS], d, 0, 0, 0);
    }
};

struct MathSplit {
    using Acc = v4f;
    static constexpr int PASSES = 3;
    // lo * hi, hi * lo, then hi * hi
    template <int PASS> static __device__ __forceinline__ void mma(Acc& d, const v4i (&p)[2], const v4i (&q)[2]) {
        d = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, p[PASS == 0]), __builtin_bit_cast(v8h, q[PASS == 1]), d,
                                                   0, 0, 0);
    }
};

// a block is 64 fp16 numbers, for matrices that fp16 holds exactly
struct MathHalf {
    using Acc = v4f;
    static constexpr int PASSES = 2;
    template <int PASS> static __device__ __forceinline__ void mma(Acc& d, const v4i (&p)[2], const v4i (&q)[2]) {
        d = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, p[PASS]), __builtin_bit_cast(v8h, q[PASS]), d, 0, 0, 0);
    }
};

// acc[j] += fragment a * fragment b[j] (or the other way round), pass by pass: consecutive instructions write
// different registers
template <class Math, bool ROWS_B, int PASS, int TN>
__device__ __forceinline__ void mma_row(typename Math::Acc (&acc)[TN], const v4i (&fa)[2], const v4i (&fb)[TN][2]) {
#pragma unroll
    for (int j = 0; j < TN; ++j) {
        if (ROWS_B) Math::template mma<PASS>(acc[j], fb[j], fa);
        else Math::template mma<PASS>(acc[j], fa, fb[j]);
    }
    if constexpr (PASS + 1 < Math::PASSES) mma_row<Math, ROWS_B, PASS + 1, TN>(acc, fa, fb);
}

typedef __attribute__((address_space(3))) char* LdsPtr;
typedef const __attribute__((address_space(3))) v4i* LdsFragment;

constexpr int TILE_BLOCK_BYTES = 128;   // of a row, per step of the contraction

// One operand of a workgroup's tile: rows `first` .. of a row-major matrix.  Rows at or past `rows` are
// read as the last row, bytes past `last_chunk` (a multiple of 16) of a row as its last chunk: the
// results that come of them are not stored, or meet zeros of the other operand.
struct TileOperand {
    const char* base;
    long long ld;           // bytes from row to row
    long long rows;
    long long first;
    long long last_chunk;   // below 2^31
    int turn = 1 << 30;     // blocks of a row (of B): from there on they are read again from the first
};

// A workgroup of WM x WN wavefronts computes BM x BN numbers over the blocks [kb0, kb1) of the contraction.
// acc[i][j] of a wavefront is the 16x16 piece (i, j) of its BM/WM x BN/WN part.  Rows of D (register index) run
// along B when ROWS_B, along A otherwise: the caller picks what its stores want contiguous in a lane.
//
// A ring of STAGES blocks in LDS: while one is worked on, the next STAGES - 1 are on their way, straight from memory into
// LDS (16 bytes a lane, no registers in between; the exchange of chunks is made in the address a lane reads, since a
// wavefront's 1,024 bytes land in LDS in lane order).  A load takes about 1 us, a block's products 0.6 us (128 x 128) to
// 1.2 us (128 x 256): what is in flight hides the difference, within a workgroup by stages and on a CU by several
// workgroups.  The stages are distinct objects, so reads of one need not wait for loads into another.  One barrier per
// block: it says that the block has landed for every wavefront and that the block before it has been read by all.
template <class Math, int BM, int BN, int WM, int WN, int STAGES, bool ROWS_B>
struct TileProduct {
    static constexpr int THREADS = 64 * WM * WN, DEPTH = STAGES;
    static constexpr int TM = BM / WM / 16, TN = BN / WN / 16;
    static constexpr int HALF = (BM + BN) * TILE_BLOCK_BYTES;
    static constexpr int WAVES = WM * WN;
    static constexpr int LA = BM / 8 / WAVES, LB = BN / 8 / WAVES;   // 1,024-byte loads (8 rows) of a wavefront per block
    static_assert(BM % (8 * WAVES) == 0 && BN % (8 * WAVES) == 0, "whole loads");
    static_assert(STAGES >= 2 && STAGES <= 4, "a ring of two to four");
    using Acc = typename Math::Acc;

    static __device__ __forceinline__ void block(LdsPtr s, int abase, int bbase, int c0, int c1, Acc (&acc)[TM][TN]) {
        v4i fb[TN][2];
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            fb[j][0] = *(LdsFragment)(s + bbase + j * 16 * TILE_BLOCK_BYTES + c0);
            fb[j][1] = *(LdsFragment)(s + bbase + j * 16 * TILE_BLOCK_BYTES + c1);
        }
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            v4i fa[2];
            fa[0] = *(LdsFragment)(s + abase + i * 16 * TILE_BLOCK_BYTES + c0);
            fa[1] = *(LdsFragment)(s + abase + i * 16 * TILE_BLOCK_BYTES + c1);
            mma_row<Math, ROWS_B, 0, TN>(acc[i], fa, fb);
        }
    }

    // all but the N youngest loads of this wavefront have landed and its LDS reads are done; then every wavefront's
    template <int N> static __device__ __forceinline__ void landed() {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 7 << 4);      // vmcnt(N) lgkmcnt(0), expcnt as it is
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    }

    static __device__ __forceinline__ void run(const TileOperand& A, const TileOperand& B, int kb0, int kb1, const LdsPtr (&ring)[4],
                                               Acc (&acc)[TM][TN]) {
        const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
        const int group = __builtin_amdgcn_readfirstlane(wave) * 8;       // of 8 rows, every WAVES-th is this wavefront's
        const int row = group + (lane >> 3);
        const int chunk = ((lane & 7) ^ (lane >> 3)) << 4;
        const int last_a = (int)A.last_chunk, last_b = (int)B.last_chunk;
        const char *pa[LA], *pb[LB];
#pragma unroll
        for (int i = 0; i < LA; ++i) {
            const long long r = A.first + row + i * 8 * WAVES;
            pa[i] = A.base + (r < A.rows ? r : A.rows - 1) * A.ld;
        }
#pragma unroll
        for (int i = 0; i < LB; ++i) {
            const long long r = B.first + row + i * 8 * WAVES;
            pb[i] = B.base + (r < B.rows ? r : B.rows - 1) * B.ld;
        }
        auto to_lds = [](const char* from, LdsPtr to) {
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                             (__attribute__((address_space(3))) void*)to, 16, 0, 0);
        };
        auto load = [&](LdsPtr s, int kb) {
            const int off = kb * TILE_BLOCK_BYTES + chunk;
            const int offb = (kb < B.turn ? kb : kb - B.turn) * TILE_BLOCK_BYTES + chunk;
            const int oa = off < last_a ? off : last_a, ob = offb < last_b ? offb : last_b;
#pragma unroll
            for (int i = 0; i < LA; ++i) to_lds(pa[i] + oa, s + (group + i * 8 * WAVES) * TILE_BLOCK_BYTES);
#pragma unroll
            for (int i = 0; i < LB; ++i) to_lds(pb[i] + ob, s + (BM + group + i * 8 * WAVES) * TILE_BLOCK_BYTES);
        };
        const int wm = wave / WN, wn = wave % WN;
        const int lr = lane & 15, lq = lane >> 4;
        const int c0 = (lq ^ (lr & 7)) << 4, c1 = ((4 + lq) ^ (lr & 7)) << 4;
        const int abase = (wm * (BM / WM) + lr) * TILE_BLOCK_BYTES;
        const int bbase = (BM + wn * (BN / WN) + lr) * TILE_BLOCK_BYTES;
        if (kb0 >= kb1) return;
        // Loads past the last block bring it in once more and are not used: every load of the loop is issued, so what is on
        // its way at any point is known when this is compiled (a load behind a branch makes the compiler wait for all).
        const int end = kb1 - 1;
#pragma unroll
        for (int u = 0; u < STAGES - 1; ++u) load(ring[u], kb0 + u < end ? kb0 + u : end);
        int kb = kb0;
        for (; kb + STAGES <= kb1; kb += STAGES) {
#pragma unroll
            for (int u = 0; u < STAGES; ++u) {
                landed<(STAGES - 2) * (LA + LB)>();       // this block; STAGES - 2 more are behind it
                const int next = kb + u + STAGES - 1;
                load(ring[(u + STAGES - 1) % STAGES], next < end ? next : end);
                block(ring[u], abase, bbase, c0, c1, acc);
            }
        }
        landed<0>();
#pragma unroll
        for (int u = 0; u < STAGES - 1; ++u)
            if (kb + u < kb1) block(ring[u], abase, bbase, c0, c1, acc);
    }
};

// the ring of a kernel whose TileProduct is T (up to four stages)
#define YH_TILE_RING(T)                                                                                              \
    __shared__ __align__(1024) char ring0[T::HALF], ring1[T::HALF], ring2[T::DEPTH > 2 ? T::HALF : 16],              \
        ring3[T::DEPTH > 3 ? T::HALF : 16];                                                                          \
    const LdsPtr ring[4] = {(LdsPtr)ring0, (LdsPtr)ring1, (LdsPtr)ring2, (LdsPtr)ring3};

// Where a lane's four numbers of piece (i, j) lie in the tile: `along` is the first of the four consecutive
// indices on the operand that supplies D's rows, `across` the index on the other one.
__device__ __forceinline__ int piece_along(int lane) { return (lane >> 4) * 4; }
__device__ __forceinline__ int piece_across(int lane) { return lane & 15; }

// Sixteen rows of a wavefront's result, PIECES * 16 columns, turned through LDS so that neighbouring lanes hold
// neighbouring columns: a lane by itself holds four numbers of a row, and stores of 8 bytes in every row cost a third of
// a large product's time.  v[p] are the lane's four numbers of piece p; emit(row, column, numbers) is called with WIDTH
// neighbouring numbers of a row.  `turn` is LDS of this wavefront alone (TURN_BYTES<PIECES>).
template <int PIECES> constexpr int TURN_LINE = PIECES * 64 + 16;
template <int PIECES> constexpr int TURN_BYTES = 16 * TURN_LINE<PIECES>;

template <int PIECES>
__device__ __forceinline__ void turn_in(LdsPtr turn, const float (&v)[PIECES][4]) {
    const int lane = threadIdx.x & 63;
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int p = 0; p < PIECES; ++p)
        *(__attribute__((address_space(3))) v4f*)(turn + piece_across(lane) * TURN_LINE<PIECES> + (p * 16 + piece_along(lane)) * 4) =
            v4f{v[p][0], v[p][1], v[p][2], v[p][3]};
    __builtin_amdgcn_wave_barrier();
}

template <int PIECES, int WIDTH, class Emit>
__device__ __forceinline__ void turn_out(LdsPtr turn, Emit&& emit) {
    constexpr int PER_ROW = PIECES * 16 / WIDTH, ITEMS = 16 * PER_ROW;
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int base = 0; base < ITEMS; base += 64) {
        const int item = base + lane, row = item / PER_ROW, col = item % PER_ROW * WIDTH;
        if (ITEMS % 64 != 0 && item >= ITEMS) break;
        float v[WIDTH];
        if constexpr (WIDTH >= 4) {
#pragma unroll
            for (int e = 0; e < WIDTH; e += 4) {
                const v4f t = *(const __attribute__((address_space(3))) v4f*)(turn + row * TURN_LINE<PIECES> + (col + e) * 4);
                v[e] = t[0];
                v[e + 1] = t[1];
                v[e + 2] = t[2];
                v[e + 3] = t[3];
            }
        } else {
#pragma unroll
            for (int e = 0; e < WIDTH; ++e)
                v[e] = *(const __attribute__((address_space(3))) float*)(turn + row * TURN_LINE<PIECES> + (col + e) * 4);
        }
        emit(row, col, v);
    }
}

// workgroup -> tile so that the workgroups of one XCD (every eighth of the launch order) take neighbouring
// tiles and share their operands in that XCD's L2
__device__ __forceinline__ long long xcd_order(long long b, long long n) {
    const long long per = n / 8, extra = n % 8, x = b % 8, i = b / 8;
    return x * per + (x < extra ? x : extra) + i;
}

}  // namespace yh
