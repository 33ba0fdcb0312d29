// Newton-Schulz orthogonalisation of a matrix, and the weight step built on it.
//
//   X_0 = G / (|G| + eps) (Frobenius norm),   X_{j+1} = (a + b A_j + c A_j^2) X_j,   A_j = X_j X_j'
//
// taken on the short side: X is l x n with l <= n (G itself, or its transpose).  Every factor is a polynomial in
// A_0, so all of them commute and are symmetric, and a group of steps needs X only twice -- for one A = X X' and for
// one product with the finished polynomial Q:
//
//   R = b A + c A^2,   P = a + R,   A <- P A P = a T + T R with T = P A = a A + R A,
//   Q <- P Q:  Q = q + S with  S <- a S + q R + R S,  q <- a q
//
// (q is a number; the multiple of the identity never goes through a matrix.)  That is 3 l^2 n + (4 s - 3) l^3
// multiply-adds for a group of s steps with half a product for each symmetric result, against s (3 l^2 n + l^3)
// step by step.
//
// Precision.  A small singular value of G grows by a in every step (485 times in five steps with a = 3.4445) and so
// does what leaks into its direction out of the large ones, so numbers of 8 or 11 bits lose it: against 64 bits,
// bf16 matrices end 1e-2 to 3e-1 off and fp16 ones 1e-3 to 4e-2 (noise; a few strong directions over noise).
// Every matrix is therefore held as two fp16 numbers, hi + lo: 22 bits, three matrix-core products for one, fp32
// sums.  An error of A grows by a^2 a step, which limits how many steps one A may serve: five end 1e-5 to 2e-4 off,
// three and two with a fresh A in between 3e-6 to 3e-5, an A for every step 2e-6 to 2e-5 -- the last is what fp32
// arithmetic gives.  The entry points form a new A when a^steps would pass 64 (fp32 results) or 512 (16-bit
// results, whose own rounding is 2e-3).
//
// A matrix of this file, "split": rows of 128-byte blocks, 32 numbers each, 64 bytes of hi and 64 bytes of lo, times
// a power of two that keeps lo out of the subnormal range; zeros fill a row's last block.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "linear_i8_kernels.hpp"
#include "tile_product.hpp"

namespace yh {

constexpr int NS_MAX_LIST = 32;      // matrices of one call that are handed over as a list of pointers
constexpr int NS_NORM_BLOCKS = 256;  // partial sums of squares of a matrix, at most

// G: one strided batch, or a list of pointers
struct NsSource {
    const void* base;
    long long stride_b, stride_r;            // in elements
    const void* g[NS_MAX_LIST];
    float* buf[NS_MAX_LIST];                 // momentum; the list form only
    float momentum;
    int nesterov;
};

struct NsShape {
    long long rows, cols;    // of G
    long long l, n;          // short and long side
    long long lk, nk;        // padded to whole blocks of 32
    int tall;                // rows > cols: X is G'
    int count;
};

__device__ __forceinline__ long long split_at(long long row, long long ld, long long col) {   // byte of hi; lo is 64 further
    return row * ld + (col >> 5) * 128 + (col & 31) * 2;
}

__device__ __forceinline__ void split_of(float v, _Float16& hi, _Float16& lo) {
    hi = (_Float16)v;
    lo = (_Float16)(v - (float)hi);
}

// sum over a workgroup of 256, to every thread
__device__ __forceinline__ double block_sum(double v, double* part) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = (part[0] + part[1]) + (part[2] + part[3]);
    __syncthreads();
    return v;
}

// ---------------------------------------------------------------- norm (and momentum)
// Squares are added in 64 bits: no gradient in fp32 range overflows or vanishes.  One partial sum per workgroup, added
// in order by whoever needs the norm: the same bits from run to run.
template <int DT, bool LIST>
__global__ __launch_bounds__(256) void ns_norm_kernel(NsSource src, NsShape sh, double* __restrict__ parts) {
    __shared__ double part[4];
    const int mat = blockIdx.y;
    const long long total = sh.rows * sh.cols;
    typedef typename Elem<DT>::T T;
    const T* g = LIST ? (const T*)src.g[mat] : (const T*)src.base + mat * src.stride_b;
    const bool flat = LIST || src.stride_r == sh.cols;
    double sum = 0.0;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        long long at = i;
        if (!flat) {
            const long long r = i / sh.cols;
            at = r * src.stride_r + (i - r * sh.cols);
        }
        float v = Elem<DT>::get(g[at]);
        if (LIST) {
            const float m = src.momentum * src.buf[mat][i] + v;
            src.buf[mat][i] = m;
            v = src.nesterov ? v + src.momentum * m : m;
        }
        sum += (double)v * (double)v;
    }
    sum = block_sum(sum, part);
    if (threadIdx.x == 0) parts[(long long)mat * gridDim.x + blockIdx.x] = sum;
}

// ---------------------------------------------------------------- G -> X and X', split
// 64 x 64 numbers of G per workgroup; `nat` gets G's own rows, `tra` its columns, both times scale / (|G| + eps)
template <int DT, bool LIST>
__global__ __launch_bounds__(256) void ns_convert_kernel(NsSource src, NsShape sh, const double* __restrict__ parts, int nparts,
                                                         double eps, double scale, char* __restrict__ nat, long long nat_mat,
                                                         char* __restrict__ tra, long long tra_mat) {
    typedef typename Elem<DT>::T T;
    __shared__ float tile[64][65];
    __shared__ double part[4];
    const int mat = blockIdx.y, t = threadIdx.x;
    const double sq = block_sum(t < nparts ? parts[(long long)mat * nparts + t] : 0.0, part);
    const double inv = scale / (sqrt(sq) + eps);
    const T* g = LIST ? (const T*)src.g[mat] : (const T*)src.base + mat * src.stride_b;
    const long long stride = LIST ? sh.cols : src.stride_r;
    const long long ncp = (sh.cols + 31) & ~31ll, nrp = (sh.rows + 31) & ~31ll;
    const unsigned across = (unsigned)((sh.cols + 63) / 64);
    const long long r0 = (long long)(blockIdx.x / across) * 64, c0 = (long long)(blockIdx.x % across) * 64;
    for (int i = t; i < 4096; i += 256) {
        const int r = i >> 6, c = i & 63;
        float v = 0.0f;
        if (r0 + r < sh.rows && c0 + c < sh.cols) {
            v = Elem<DT>::get(g[(r0 + r) * stride + c0 + c]);
            if (LIST) {
                const float m = src.buf[mat][(r0 + r) * sh.cols + c0 + c];
                v = src.nesterov ? v + src.momentum * m : m;
            }
            v = (float)((double)v * inv);
        }
        tile[r][c] = v;
    }
    __syncthreads();
    const int line = t >> 2, at = (t & 3) * 16;      // 16 numbers of a line of the tile
    union Pack {
        v4i w[2];
        _Float16 h[16];
    } hi, lo;
    if (r0 + line < sh.rows && c0 + at < ncp) {
#pragma unroll
        for (int e = 0; e < 16; ++e) split_of(tile[line][at + e], hi.h[e], lo.h[e]);
        char* p = nat + mat * nat_mat + split_at(r0 + line, ncp * 4, c0 + at);
        *(v4i*)p = hi.w[0];
        *(v4i*)(p + 16) = hi.w[1];
        *(v4i*)(p + 64) = lo.w[0];
        *(v4i*)(p + 80) = lo.w[1];
    }
    if (c0 + line < sh.cols && r0 + at < nrp) {
#pragma unroll
        for (int e = 0; e < 16; ++e) split_of(tile[at + e][line], hi.h[e], lo.h[e]);
        char* p = tra + mat * tra_mat + split_at(c0 + line, nrp * 4, r0 + at);
        *(v4i*)p = hi.w[0];
        *(v4i*)(p + 16) = hi.w[1];
        *(v4i*)(p + 64) = lo.w[0];
        *(v4i*)(p + 80) = lo.w[1];
    }
}

// ---------------------------------------------------------------- symmetric products
// out = k0 * (P Q') + k1 * E1 + k2 * E2, symmetric (P and Q commute, or are one matrix): the tiles on and below the
// diagonal are computed and every number below it is stored on both sides.
struct NsProduct {
    const char *P, *Q, *E1, *E2;
    char* out;
    long long p_mat, out_mat;       // bytes from matrix to matrix of P and Q; of E1, E2 and out
    long long ldp;                  // bytes from row to row of P and Q; lk * 4 in E1, E2 and out
    float k0, k1, k2;
    int blocks;                     // of 32 numbers along the contraction
};
struct NsProducts {
    NsProduct job[2];
    long long l, lk;
    int count, tiles;               // tiles on and below the diagonal
    int slices, per_slice;          // the contraction in slices, when partial sums are joined
    float* partial;
};

__device__ __forceinline__ float split_get(const char* p) {
    return (float)*(const _Float16*)p + (float)*(const _Float16*)(p + 64);
}
__device__ __forceinline__ void split_put(char* p, float v) {
    _Float16 hi, lo;
    split_of(v, hi, lo);
    *(_Float16*)p = hi;
    *(_Float16*)(p + 64) = lo;
}

__device__ __forceinline__ void triangle(int t, int& i, int& j) {
    i = (int)((sqrtf(8.0f * (float)t + 1.0f) - 1.0f) * 0.5f);
    while ((i + 1) * (i + 2) / 2 <= t) ++i;
    while (i * (i + 1) / 2 > t) --i;
    j = t - i * (i + 1) / 2;
}

// four numbers (m, n .. n + 3) of a product
__device__ __forceinline__ void ns_store_sym(const NsProduct& p, const NsProducts& a, long long mat, long long m, long long n,
                                             const v4f& d) {
    if (m >= a.lk || n >= a.l || n > m) return;
    const long long ld = a.lk * 4;
    char* out = p.out + mat * p.out_mat;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const long long c = n + r;
        if (c >= a.l || c > m) continue;
        float v = 0.0f;
        if (m < a.l) {
            const long long at = split_at(m, ld, c);
            v = p.k0 * d[r];
            if (p.E1) v += p.k1 * split_get(p.E1 + mat * p.out_mat + at);
            if (p.E2) v += p.k2 * split_get(p.E2 + mat * p.out_mat + at);
            split_put(out + at, v);
        }
        split_put(out + split_at(c, ld, m), v);      // the other side; zeros past the matrix
    }
}

template <int BM, int WM, int WN, int STAGES>
__global__ __launch_bounds__(64 * WM * WN, 2) void ns_product_kernel(NsProducts a) {
    typedef TileProduct<MathSplit, BM, BM, WM, WN, STAGES, true> T;
    YH_TILE_RING(T)
    const NsProduct p = a.job[blockIdx.y];
    const long long per = (long long)a.tiles * a.count;
    const long long id = xcd_order(blockIdx.x, per * a.slices);
    const int slice = (int)(id / per);
    const long long mt = id - slice * per;
    const long long mat = mt / a.tiles;
    int ti, tj;
    triangle((int)(mt - mat * a.tiles), ti, tj);
    typename T::Acc acc[T::TM][T::TN] = {};
    const TileOperand A = {p.P + mat * p.p_mat, p.ldp, a.l, (long long)ti * BM, p.ldp - 16};
    const TileOperand B = {p.Q + mat * p.p_mat, p.ldp, a.l, (long long)tj * BM, p.ldp - 16};
    const int k0 = slice * a.per_slice;
    const int k1 = k0 + a.per_slice < p.blocks ? k0 + a.per_slice : p.blocks;
    T::run(A, B, k0, k1, ring, acc);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long m0 = (long long)ti * BM + (wave / WN) * (BM / WM) + piece_across(lane);
    const long long n0 = (long long)tj * BM + (wave % WN) * (BM / WN) + piece_along(lane);
    float* part = a.partial + id * (BM * BM) + threadIdx.x * 4;
#pragma unroll
    for (int i = 0; i < T::TM; ++i)
#pragma unroll
        for (int j = 0; j < T::TN; ++j) {
            if (a.slices == 1) ns_store_sym(p, a, mat, m0 + i * 16, n0 + j * 16, acc[i][j]);
            else *(v4f*)(part + (i * T::TN + j) * T::THREADS * 4) = acc[i][j];
        }
}

// the slices of ns_product_kernel added in order, same geometry
template <int BM, int WM, int WN, int STAGES>
__global__ __launch_bounds__(64 * WM * WN, 2) void ns_join_kernel(NsProducts a) {
    typedef TileProduct<MathSplit, BM, BM, WM, WN, STAGES, true> T;
    const NsProduct p = a.job[0];
    const long long per = (long long)a.tiles * a.count;
    const long long mt = blockIdx.x;
    const long long mat = mt / a.tiles;
    int ti, tj;
    triangle((int)(mt - mat * a.tiles), ti, tj);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long m0 = (long long)ti * BM + (wave / WN) * (BM / WM) + piece_across(lane);
    const long long n0 = (long long)tj * BM + (wave % WN) * (BM / WN) + piece_along(lane);
    const float* part = a.partial + mt * (BM * BM) + threadIdx.x * 4;
#pragma unroll
    for (int i = 0; i < T::TM; ++i)
#pragma unroll
        for (int j = 0; j < T::TN; ++j) {
            v4f d = {0.0f, 0.0f, 0.0f, 0.0f};
            for (int s = 0; s < a.slices; ++s)
                d += *(const v4f*)(part + (long long)s * per * (BM * BM) + (i * T::TN + j) * T::THREADS * 4);
            ns_store_sym(p, a, mat, m0 + i * 16, n0 + j * 16, d);
        }
}

// ---------------------------------------------------------------- Y = q X + S X
enum { NS_OUT_RESULT = 0, NS_OUT_WEIGHT = 1, NS_OUT_SPLIT = 2 };

struct NsApply {
    const char *S, *X, *Xt;
    long long s_mat, x_mat, xt_mat;
    NsShape sh;
    float k0, k1;                    // Y = k0 * (S X) + k1 * X
    // NS_OUT_RESULT
    void* out;
    long long out_b, out_r;          // elements from matrix to matrix and row to row
    int whole;                       // four neighbours of a row may be stored at once
    // NS_OUT_WEIGHT
    void* param[NS_MAX_LIST];
    float decay, step;               // p = decay * p - step * Y
    // NS_OUT_SPLIT: Y times `again`
    char *Yn, *Yt;
    float again;
};

template <int DT, int OUT, bool TALL, int BM, int BN, int WM, int WN, int STAGES>
__global__ __launch_bounds__(64 * WM * WN, 2) void ns_apply_kernel(NsApply a) {
    // a lane's four numbers lie along a row of the result: along n, or along l when X is G'
    typedef TileProduct<MathSplit, BM, BN, WM, WN, STAGES, !TALL> T;
    typedef typename Elem<DT>::T E;
    YH_TILE_RING(T)
    const NsShape& sh = a.sh;
    const int tl = (int)((sh.l + BM - 1) / BM);
    const long long tn = (sh.n + BN - 1) / BN, per = tl * tn;
    const long long id = xcd_order(blockIdx.x, per * sh.count);
    const long long mat = id / per, tile = id - mat * per;
    const long long ti = tile % tl, tj = tile / tl;
    typename T::Acc acc[T::TM][T::TN] = {};
    const long long ld = sh.lk * 4, ldn = sh.nk * 4;
    const TileOperand A = {a.S + mat * a.s_mat, ld, sh.l, ti * BM, ld - 16};
    const TileOperand B = {a.Xt + mat * a.xt_mat, ld, sh.n, tj * BN, ld - 16};
    T::run(A, B, 0, (int)(sh.lk / 32), ring, acc);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const char* x = TALL ? a.Xt + mat * a.xt_mat : a.X + mat * a.x_mat;
    const long long ldx = TALL ? ld : ldn;
    const long long along_end = TALL ? sh.l : sh.n, across_end = TALL ? sh.n : sh.l, along_pad = TALL ? sh.lk : sh.nk;
#pragma unroll
    for (int i = 0; i < T::TM; ++i)
#pragma unroll
        for (int j = 0; j < T::TN; ++j) {
            const long long m = ti * BM + (wave / WN) * (BM / WM) + i * 16, n = tj * BN + (wave % WN) * (BN / WN) + j * 16;
            const long long row = (TALL ? n : m) + piece_across(lane), col = (TALL ? m : n) + piece_along(lane);
            if (OUT == NS_OUT_SPLIT && row >= across_end && row < sh.lk) {      // a row of X' ends in zeros
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (col + r < along_end) split_put(a.Yt + mat * a.xt_mat + split_at(col + r, ld, row), 0.0f);
            }
            if (row >= across_end || col >= along_pad) continue;
            const char* px = x + split_at(row, ldx, col);      // whole blocks of four: inside the padding
            const v4h hi = *(const v4h*)px, lo = *(const v4h*)(px + 64);
            float y[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) y[r] = a.k0 * acc[i][j][r] + a.k1 * ((float)hi[r] + (float)lo[r]);
            const int left = along_end - col < 4 ? (int)(along_end - col) : 4;
            if (OUT == NS_OUT_RESULT) {
                if (left > 0) put4<DT>((E*)a.out + mat * a.out_b + row * a.out_r + col, y, left, a.whole);
            } else if (OUT == NS_OUT_WEIGHT) {
                E* p = (E*)a.param[mat] + row * along_end + col;
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (r < left) p[r] = Elem<DT>::put(a.decay * Elem<DT>::get(p[r]) - a.step * y[r]);
            } else {
                // !TALL here: rows of X along n, rows of X' along l
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float v = r < left ? y[r] * a.again : 0.0f;
                    split_put(a.Yn + mat * a.x_mat + split_at(row, ldn, col + r), v);
                    if (r < left) split_put(a.Yt + mat * a.xt_mat + split_at(col + r, ld, row), v);
                }
            }
        }
}

}  // namespace yh
