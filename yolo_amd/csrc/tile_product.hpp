// Tile products on the matrix cores (gfx950): D = A * B' for two operands whose rows lie along the
// contraction, 128 bytes of a row at a time.  Two arithmetics share the data path, since a lane's
// share of a fragment is 16 bytes in both:
//
//   MathI8     a 128-byte block of a row is 128 signed bytes; two 16x16x64 products per 16x16
//              piece of D, exact in int32.
//   MathSplit  a block is 32 numbers in two halves: 64 bytes of their leading parts (fp16), then 64
//              bytes of what fp16 leaves over (fp16 again): x = hi + lo to 22 bits.  Three 16x16x32
//              products, hi*hi + hi*lo + lo*hi, in fp32; lo*lo is below 2^-22 of the product.
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
    static __device__ __forceinline__ void mma(Acc& d, const v4i (&p)[2], const v4i (&q)[2]) {
        d = __builtin_amdgcn_mfma_i32_16x16x64_i8(p[0], q[0], d, 0, 0, 0);
        d = __builtin_amdgcn_mfma_i32_16x16x64_i8(p[1], q[1], d, 0, 0, 0);
    }
};

struct MathSplit {
    using Acc = v4f;
    static __device__ __forceinline__ v8h h(v4i x) { return __builtin_bit_cast(v8h, x); }
    static __device__ __forceinline__ void mma(Acc& d, const v4i (&p)[2], const v4i (&q)[2]) {
        d = __builtin_amdgcn_mfma_f32_16x16x32_f16(h(p[0]), h(q[1]), d, 0, 0, 0);
        d = __builtin_amdgcn_mfma_f32_16x16x32_f16(h(p[1]), h(q[0]), d, 0, 0, 0);
        d = __builtin_amdgcn_mfma_f32_16x16x32_f16(h(p[0]), h(q[0]), d, 0, 0, 0);
    }
};

constexpr int TILE_BLOCK_BYTES = 128;   // of a row, per step of the contraction

// One operand of a workgroup's tile: rows `first` .. of a row-major matrix.  Rows at or past `rows` are
// read as the last row, bytes past `last_chunk` (a multiple of 16) of a row as its last chunk: the
// results that come of them are not stored, or meet zeros of the other operand.
struct TileOperand {
    const char* base;
    long long ld;           // bytes from row to row
    long long rows;
    long long first;
    long long last_chunk;
};

// A workgroup of WM x WN wavefronts computes BM x BN numbers over the blocks [kb0, kb1) of the contraction.
// acc[i][j] of a wavefront is the 16x16 piece (i, j) of its BM/WM x BN/WN part.  Rows of D (register index) run
// along B when ROWS_B, along A otherwise: the caller picks what its stores want contiguous in a lane.
// lds: 2 * (BM + BN) * 128 bytes.  The next block's bytes travel in registers while a block is worked on
// (double-buffered LDS, one barrier per block).
template <class Math, int BM, int BN, int WM, int WN, bool ROWS_B>
struct TileProduct {
    static constexpr int THREADS = 64 * WM * WN;
    static constexpr int TM = BM / WM / 16, TN = BN / WN / 16;
    static constexpr int LDS_BYTES = 2 * (BM + BN) * TILE_BLOCK_BYTES;
    static constexpr int LA = BM * 8 / THREADS, LB = BN * 8 / THREADS;   // 16-byte loads per thread
    using Acc = typename Math::Acc;

    static __device__ __forceinline__ void run(const TileOperand& A, const TileOperand& B, long long kb0, long long kb1,
                                               char* lds, Acc (&acc)[TM][TN]) {
        const int t = threadIdx.x, chunk = t & 7, row0 = t >> 3;
        constexpr int STEP = THREADS / 8;
        const char* pa[LA];
        const char* pb[LB];
#pragma unroll
        for (int i = 0; i < LA; ++i) {
            const long long r = A.first + row0 + i * STEP;
            pa[i] = A.base + (r < A.rows ? r : A.rows - 1) * A.ld;
        }
#pragma unroll
        for (int i = 0; i < LB; ++i) {
            const long long r = B.first + row0 + i * STEP;
            pb[i] = B.base + (r < B.rows ? r : B.rows - 1) * B.ld;
        }
        v4i ra[LA], rb[LB];
        auto fetch = [&](long long kb) {
            const long long off = kb * TILE_BLOCK_BYTES + chunk * 16;
            const long long oa = off < A.last_chunk ? off : A.last_chunk, ob = off < B.last_chunk ? off : B.last_chunk;
#pragma unroll
            for (int i = 0; i < LA; ++i) ra[i] = *(const v4i*)(pa[i] + oa);
#pragma unroll
            for (int i = 0; i < LB; ++i) rb[i] = *(const v4i*)(pb[i] + ob);
        };
        auto park = [&](char* s) {
#pragma unroll
            for (int i = 0; i < LA; ++i) {
                const int r = row0 + i * STEP;
                *(v4i*)(s + r * TILE_BLOCK_BYTES + ((chunk ^ (r & 7)) << 4)) = ra[i];
            }
#pragma unroll
            for (int i = 0; i < LB; ++i) {
                const int r = row0 + i * STEP;
                *(v4i*)(s + (BM + r) * TILE_BLOCK_BYTES + ((chunk ^ (r & 7)) << 4)) = rb[i];
            }
        };
        const int lane = t & 63, wave = t >> 6;
        const int wm = wave / WN, wn = wave % WN;
        const int lr = lane & 15, lq = lane >> 4;
        const int c0 = (lq ^ (lr & 7)) << 4, c1 = ((4 + lq) ^ (lr & 7)) << 4;
        const int abase = (wm * (BM / WM) + lr) * TILE_BLOCK_BYTES;
        const int bbase = (BM + wn * (BN / WN) + lr) * TILE_BLOCK_BYTES;
        constexpr int HALF = (BM + BN) * TILE_BLOCK_BYTES;
        if (kb0 >= kb1) return;
        fetch(kb0);
        park(lds);
        __syncthreads();
        int cur = 0;
        for (long long kb = kb0; kb < kb1; ++kb) {
            const bool more = kb + 1 < kb1;
            if (more) fetch(kb + 1);
            const char* s = lds + cur * HALF;
            v4i fb[TN][2];
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                fb[j][0] = *(const v4i*)(s + bbase + j * 16 * TILE_BLOCK_BYTES + c0);
                fb[j][1] = *(const v4i*)(s + bbase + j * 16 * TILE_BLOCK_BYTES + c1);
            }
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                v4i fa[2];
                fa[0] = *(const v4i*)(s + abase + i * 16 * TILE_BLOCK_BYTES + c0);
                fa[1] = *(const v4i*)(s + abase + i * 16 * TILE_BLOCK_BYTES + c1);
#pragma unroll
                for (int j = 0; j < TN; ++j) {
                    if (ROWS_B) Math::mma(acc[i][j], fb[j], fa);
                    else Math::mma(acc[i][j], fa, fb[j]);
                }
            }
            if (more) park(lds + (cur ^ 1) * HALF);
            __syncthreads();
            cur ^= 1;
        }
    }
};

// Where a lane's four numbers of piece (i, j) lie in the tile: `along` is the first of the four consecutive
// indices on the operand that supplies D's rows, `across` the index on the other one.
__device__ __forceinline__ int piece_along(int lane) { return (lane >> 4) * 4; }
__device__ __forceinline__ int piece_across(int lane) { return lane & 15; }

// workgroup -> tile so that the workgroups of one XCD (every eighth of the launch order) take neighbouring
// tiles and share their operands in that XCD's L2
__device__ __forceinline__ long long xcd_order(long long b, long long n) {
    const long long per = n / 8, extra = n % 8, x = b % 8, i = b / 8;
    return x * per + (x < extra ? x : extra) + i;
}

}  // namespace yh
