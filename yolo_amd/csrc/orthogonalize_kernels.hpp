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
// sums.  An error of A grows by a^2 a step, which limits how many steps one A may serve: measured over 16 x 16 to
// 4096 x 9216 and spectra from noise to one strong direction over 1 % of it, five end 6e-6 to 8e-4 off, three and two
// with a fresh A in between 2e-6 to 5.5e-5, where fp32 arithmetic with an A for every step ends 7e-7 to 7.4e-5 off.
// The entry points form a new A when a^steps would pass 64, or 511 for bf16 results, whose own rounding is 1.7e-3.
//
// X is held as a matrix of Frobenius norm `scale` and the factor |G| / (|G| + eps) / scale beside it, a number of its own for
// each matrix: a gradient far below eps keeps its bits.  What is held grows with the steps, by `growth` as long as the singular
// values are small and until they reach `top`, so each group of steps begins at a scale (and factor) with room for that.
//
// Where G and the result have 16-bit numbers, X needs no lo ("half": rows of fp16 numbers, zeros up to a multiple of 64): it
// is G times a power of two, held as fp16 without a rounding (numbers 2^14 below the mean are off by 2^-25 of the mean at
// most, as in hi + lo), and the factor takes the rest.  X X' is one product instead of three, S X two (S as the planes hi
// and lo of a row, X' read twice), and X is half the bytes: 4096 x 50,176 9.5 -> 7.2 ms.
//
// A matrix of this file, "split": rows of 128-byte blocks, 32 numbers each, 64 bytes of hi and 64 bytes of lo, times
// a power of two that keeps lo out of the subnormal range; zeros fill a row's last block.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "linear_i8_kernels.hpp"
#include "tile_product.hpp"

namespace yh {

constexpr int NS_MAX_GROUPS = 64;
struct NsHold {
    int groups;
    double scale;                    // of the first group
    // before group g, powers of two: small singular values have grown by less than growth[g], none has reached top[g]
    short growth[NS_MAX_GROUPS], top[NS_MAX_GROUPS];
};

constexpr int NS_MAX_LIST = 32;      // matrices of one call that are handed over as a list of pointers
constexpr int NS_NORM_BLOCKS = 1024; // partial sums of squares of a matrix, at most

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
    long long lh, nh;        // padded to whole blocks of 64 ("half")
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
// in order by whoever needs the norm: the same bits from run to run.  vec: matrices without gaps between rows, on 16 bytes
// and of a multiple of eight numbers; a thread then takes eight at a time.  411 MB of bf16: 85 us (4.8 TB/s);
// with momentum (38 M numbers, 375 MB): 62 us.
template <int DT, bool LIST>
__global__ __launch_bounds__(256) void ns_norm_kernel(NsSource src, NsShape sh, double* __restrict__ parts, int vec) {
    __shared__ double part[4];
    const int mat = blockIdx.y;
    const long long total = sh.rows * sh.cols, stride = (long long)gridDim.x * 256;
    typedef typename Elem<DT>::T T;
    const T* g = LIST ? (const T*)src.g[mat] : (const T*)src.base + mat * src.stride_b;
    float* buf = LIST ? src.buf[mat] : nullptr;
    double sum = 0.0;
    auto one = [&](float v, float* m) {
        if (LIST) {
            *m = src.momentum * *m + v;
            v = src.nesterov ? v + src.momentum * *m : *m;
        }
        sum += (double)v * (double)v;
    };
    if (vec) {
        constexpr int V = 16 / (int)sizeof(T);
        typedef T TV __attribute__((ext_vector_type(V)));
#pragma unroll 2
        for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i * 8 < total; i += stride) {
            TV v[8 / V];
            v4f m[2];
#pragma unroll
            for (int p = 0; p < 8 / V; ++p) v[p] = *(const TV*)(g + i * 8 + p * V);
            if (LIST) {
                m[0] = *(const v4f*)(buf + i * 8);
                m[1] = *(const v4f*)(buf + i * 8 + 4);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float x = LIST ? m[e / 4][e % 4] : 0.0f;
                one(Elem<DT>::get(v[e / V][e % V]), &x);
                if (LIST) m[e / 4][e % 4] = x;
            }
            if (LIST) {
                *(v4f*)(buf + i * 8) = m[0];
                *(v4f*)(buf + i * 8 + 4) = m[1];
            }
        }
    } else {
        const bool flat = LIST || src.stride_r == sh.cols;
        for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += stride) {
            long long at = i;
            if (!flat) {
                const long long r = i / sh.cols;
                at = r * src.stride_r + (i - r * sh.cols);
            }
            one(Elem<DT>::get(g[at]), buf + i);
        }
    }
    sum = block_sum(sum, part);
    if (threadIdx.x == 0) parts[(long long)mat * gridDim.x + blockIdx.x] = sum;
}

// eight neighbours of a split row
struct Split8 {
    v4i hi, lo;
};
__device__ __forceinline__ Split8 split8_of(const float (&v)[8]) {
    union {
        v4i w;
        _Float16 h[8];
    } hi, lo;
#pragma unroll
    for (int e = 0; e < 8; ++e) split_of(v[e], hi.h[e], lo.h[e]);
    return {hi.w, lo.w};
}
__device__ __forceinline__ void split8_put(char* p, const float (&v)[8]) {
    const Split8 x = split8_of(v);
    *(v4i*)p = x.hi;
    *(v4i*)(p + 64) = x.lo;
}
// the same of v[from .. to) only
__device__ __forceinline__ void split8_put_some(char* p, const float (&v)[8], long long from, long long to) {
    if (from <= 0 && to >= 8) {
        split8_put(p, v);
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (e >= from && e < to) {
            _Float16 hi, lo;
            split_of(v[e], hi, lo);
            *(_Float16*)(p + 2 * e) = hi;
            *(_Float16*)(p + 2 * e + 64) = lo;
        }
}
// N (a power of two up to 8) neighbours, from a multiple of N on
template <int N>
__device__ __forceinline__ void split_get_n(const char* p, float (&v)[N]) {
    typedef _Float16 H __attribute__((ext_vector_type(N)));
    if constexpr (N == 1) {
        v[0] = (float)*(const _Float16*)p + (float)*(const _Float16*)(p + 64);
    } else {
        const H hi = *(const H*)p, lo = *(const H*)(p + 64);
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = (float)hi[e] + (float)lo[e];
    }
}

template <int N>
__device__ __forceinline__ void half_get_n(const char* p, float (&v)[N]) {
    if constexpr (N == 1) {
        v[0] = (float)*(const _Float16*)p;
    } else {
        typedef _Float16 H __attribute__((ext_vector_type(N)));
        const H h = *(const H*)p;
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = (float)h[e];
    }
}

// ---------------------------------------------------------------- G -> X and X', split or half
// 64 x 64 numbers of G per workgroup; `nat` gets G's own rows, `tra` its columns, both times scale / |G|.  vec: rows
// of G (and of the momentum) on 16 bytes and of a multiple of eight numbers.  4096 x 50,176 bf16, fp16 alone: 286 us
// for 1.23 GB (4.3 TB/s); 4 x 1024 x 9216 with momentum, split: 117 us for 528 MB (4.5 TB/s).
template <int DT, bool LIST, bool HALF>
__global__ __launch_bounds__(256) void ns_convert_kernel(NsSource src, NsShape sh, const double* __restrict__ parts, int nparts,
                                                         double eps, NsHold hold, char* __restrict__ nat, long long nat_mat,
                                                         char* __restrict__ tra, long long tra_mat, float* __restrict__ factor,
                                                         float* __restrict__ hop, int vec) {
    typedef typename Elem<DT>::T T;
    __shared__ float tile[64][65];
    __shared__ double part[4];
    const int mat = blockIdx.y, t = threadIdx.x;
    const T* g = LIST ? (const T*)src.g[mat] : (const T*)src.base + mat * src.stride_b;
    const float* buf = LIST ? src.buf[mat] : nullptr;
    const long long stride = LIST ? sh.cols : src.stride_r;
    constexpr long long PAD = HALF ? 63 : 31;
    const long long ncp = (sh.cols + PAD) & ~PAD, nrp = (sh.rows + PAD) & ~PAD;
    auto place = [](long long row, long long padded, long long col) {
        return HALF ? row * padded * 2 + col * 2 : split_at(row, padded * 4, col);
    };
    const unsigned across = (unsigned)((sh.cols + 63) / 64);
    const long long r0 = (long long)(blockIdx.x / across) * 64, c0 = (long long)(blockIdx.x % across) * 64;
    const int line = t >> 2, at = (t & 3) * 16;      // 16 numbers of a line of the tile
    float v[16], m[16];
    const bool row_in = r0 + line < sh.rows;
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = m[e] = 0.0f;
    if (vec) {
        constexpr int V = 16 / (int)sizeof(T);
        typedef T TV __attribute__((ext_vector_type(V)));
#pragma unroll
        for (int e = 0; e < 16; e += 8)
            if (row_in && c0 + at + e < sh.cols) {
#pragma unroll
                for (int p = 0; p < 8; p += V) {
                    const TV x = *(const TV*)(g + (r0 + line) * stride + c0 + at + e + p);
#pragma unroll
                    for (int k = 0; k < V; ++k) v[e + p + k] = Elem<DT>::get(x[k]);
                }
                if (LIST) {
#pragma unroll
                    for (int p = 0; p < 8; p += 4) {
                        const v4f x = *(const v4f*)(buf + (r0 + line) * sh.cols + c0 + at + e + p);
#pragma unroll
                        for (int k = 0; k < 4; ++k) m[e + p + k] = x[k];
                    }
                }
            }
    } else {
#pragma unroll
        for (int e = 0; e < 16; ++e)
            if (row_in && c0 + at + e < sh.cols) {
                v[e] = Elem<DT>::get(g[(r0 + line) * stride + c0 + at + e]);
                if (LIST) m[e] = buf[(r0 + line) * sh.cols + c0 + at + e];
            }
    }
    double some = 0.0;
    for (int i = t; i < nparts; i += 256) some += parts[(long long)mat * nparts + i];
    const double sq = block_sum(some, part);
    const double norm = sqrt(sq);
    double inv = norm == 0.0 ? 0.0 : hold.scale / norm;
    if (HALF && norm > 0.0 && norm < 1e300) {
        int e;
        frexp(inv, &e);
        inv = ldexp(1.0, e - 1);                 // the power of two at or below
    }
    if (blockIdx.x == 0 && t < hold.groups) {
        // X_g = factor[g] times what is held; hop[g]: from what is held in group g - 1 to what is held in group g
        const double unit = norm / (norm + eps);                   // |X_0|
        auto scale_of = [&](int g) {
            const int most = hold.top[g] - ilogb(unit);
            return ldexp(1.0, 15 - (hold.growth[g] < most ? hold.growth[g] : most));
        };
        const double now = t == 0 ? inv * norm : scale_of(t), before = t == 1 ? inv * norm : t > 1 ? scale_of(t - 1) : now;
        factor[t * sh.count + mat] = norm == 0.0 ? 0.0f : (float)(unit / now);
        hop[t * sh.count + mat] = norm == 0.0 ? 0.0f : (float)(now / before);
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        if (LIST) v[e] = src.nesterov ? v[e] + src.momentum * m[e] : m[e];
        v[e] = (float)((double)v[e] * inv);
        tile[line][at + e] = v[e];
    }
    auto put = [&](char* p, const float (&x)[16]) {
        if constexpr (HALF) {
            v8h a, b;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                a[e] = (_Float16)x[e];
                b[e] = (_Float16)x[8 + e];
            }
            *(v8h*)p = a;
            *(v8h*)(p + 16) = b;
            return;
        }
        float a[8], b[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            a[e] = x[e];
            b[e] = x[8 + e];
        }
        split8_put(p, a);
        split8_put(p + 16, b);
    };
    if (row_in && c0 + at < ncp) put(nat + mat * nat_mat + place(r0 + line, ncp, c0 + at), v);
    __syncthreads();
    if (c0 + line < sh.cols && r0 + at < nrp) {
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = tile[at + e][line];
        put(tra + mat * tra_mat + place(c0 + line, nrp, r0 + at), v);
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
    const float* factor;            // of each matrix, or null: k0 times its square
    float k0, k1, k2;
    int blocks;                     // of 128 bytes along the contraction
    int first, tiles;               // of the tiles on and below the diagonal: this job's
};
struct NsProducts {
    NsProduct job[2];               // the second may have no tiles
    long long l, lk;
    int count;
    int slices, per_slice;          // the contraction in slices, when partial sums are joined
    float* partial;
};

__device__ __forceinline__ void triangle(int t, int& i, int& j) {
    i = (int)((sqrtf(8.0f * (float)t + 1.0f) - 1.0f) * 0.5f);
    while ((i + 1) * (i + 2) / 2 <= t) ++i;
    while (i * (i + 1) / 2 > t) --i;
    j = t - i * (i + 1) / 2;
}

// The wavefront's part of a tile: its rows from m0 and columns from n0 on, turned through LDS 16 rows at a time: eight
// neighbours of a row to their place, eight neighbours of a column to the other side.  Of a tile on the diagonal only what
// is on and below it is taken: both sides hold the same bits.  (They have to.  A product here takes the rows of its second
// factor for columns, so what is not symmetric would enter the next step with its sign turned round, where it grows
// by a - R = 6 instead of a + R = 0.7: two sides that differ in their last bit ended 2e-3 off.)
template <class T>
__device__ __forceinline__ void ns_store_sym(const NsProduct& p, const NsProducts& a, long long mat, long long m0, long long n0,
                                             bool diagonal, LdsPtr turn, const typename T::Acc (&acc)[T::TM][T::TN]) {
    const long long ld = a.lk * 4;
    char* out = p.out + mat * p.out_mat;
    const char* E1 = p.E1 ? p.E1 + mat * p.out_mat : nullptr;
    const char* E2 = p.E2 ? p.E2 + mat * p.out_mat : nullptr;
    const int lane = threadIdx.x & 63;
    const float k0 = p.factor ? p.k0 * p.factor[mat] * p.factor[mat] : p.k0;
#pragma unroll
    for (int i = 0; i < T::TM; ++i) {
        float d[T::TN][4];
#pragma unroll
        for (int j = 0; j < T::TN; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) d[j][r] = k0 * acc[i][j][r];
        turn_in<T::TN>(turn, d);
        turn_out<T::TN, 8>(turn, [&](int row, int col, float (&v)[8]) {
            const long long m = m0 + i * 16 + row, n = n0 + col;
            const bool inside = m < a.l && n < a.lk;
            const long long at = split_at(m, ld, n);
            float e[8];
            if (inside && E1) {
                split_get_n<8>(E1 + at, e);
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] += p.k1 * e[k];
            }
            if (inside && E2) {
                split_get_n<8>(E2 + at, e);
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] += p.k2 * e[k];
            }
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (m >= a.l || n + k >= a.l) v[k] = 0.0f;      // zeros past the matrix
            if (inside) split8_put_some(out + at, v, 0, diagonal ? m - n + 1 : 8);
#pragma unroll
            for (int k = 0; k < 8; k += 4)
                *(__attribute__((address_space(3))) v4f*)(turn + row * TURN_LINE<T::TN> + (col + k) * 4) = v4f{v[k], v[k + 1], v[k + 2], v[k + 3]};
        });
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int c = lane; c < T::TN * 32; c += 64) {        // (column, half of the 16 rows)
            const int col = c % (T::TN * 16), half = c / (T::TN * 16) * 8;
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k)
                v[k] = *(const __attribute__((address_space(3))) float*)(turn + (half + k) * TURN_LINE<T::TN> + col * 4);
            const long long n = n0 + col, m = m0 + i * 16 + half;
            if (n < a.l && m < a.lk) split8_put_some(out + split_at(n, ld, m), v, diagonal ? n - m + 1 : 0, 8);
        }
    }
}

template <class Math, int BM, int WM, int WN, int STAGES>
__global__ __launch_bounds__(64 * WM * WN, 2) void ns_product_kernel(NsProducts a) {
    typedef TileProduct<Math, BM, BM, WM, WN, STAGES, true> T;
    YH_TILE_RING(T)
    const long long before = (long long)a.job[0].tiles * a.count * a.slices;
    long long id = xcd_order(blockIdx.x, before + (long long)a.job[1].tiles * a.count);      // slices only of a job by itself
    const int second = id >= before;
    const NsProduct p = a.job[second];
    if (second) id -= before;
    const long long per = (long long)p.tiles * a.count;
    const int slice = (int)(id / per);
    const long long mt = id - slice * per;
    const long long mat = mt / p.tiles;
    int ti, tj;
    triangle(p.first + (int)(mt - mat * p.tiles), ti, tj);
    typename T::Acc acc[T::TM][T::TN] = {};
    const TileOperand A = {p.P + mat * p.p_mat, p.ldp, a.l, (long long)ti * BM, p.ldp - 16};
    const TileOperand B = {p.Q + mat * p.p_mat, p.ldp, a.l, (long long)tj * BM, p.ldp - 16};
    const int k0 = slice * a.per_slice;
    const int k1 = k0 + a.per_slice < p.blocks ? k0 + a.per_slice : p.blocks;
    T::run(A, B, k0, k1, ring, acc);
    const int wave = threadIdx.x >> 6;
    if (a.slices > 1) {
        float* part = a.partial + id * (BM * BM) + threadIdx.x * 4;
#pragma unroll
        for (int i = 0; i < T::TM; ++i)
#pragma unroll
            for (int j = 0; j < T::TN; ++j) *(v4f*)(part + (i * T::TN + j) * T::THREADS * 4) = acc[i][j];
        return;
    }
    __syncthreads();
    LdsPtr turn = (wave & 1 ? ring[1] : ring[0]) + (wave >> 1) * TURN_BYTES<T::TN>;
    ns_store_sym<T>(p, a, mat, (long long)ti * BM + (wave / WN) * (BM / WM), (long long)tj * BM + (wave % WN) * (BM / WN), ti == tj,
                    turn, acc);
}

// the slices of ns_product_kernel added in order, same geometry
template <int BM, int WM, int WN, int STAGES>
__global__ __launch_bounds__(64 * WM * WN, 2) void ns_join_kernel(NsProducts a) {
    typedef TileProduct<MathSplit, BM, BM, WM, WN, STAGES, true> T;
    __shared__ __align__(16) char lds[T::WAVES * TURN_BYTES<T::TN>];
    const NsProduct p = a.job[0];
    const long long per = (long long)p.tiles * a.count;
    const long long mt = blockIdx.x;
    const long long mat = mt / p.tiles;
    int ti, tj;
    triangle((int)(mt - mat * p.tiles), ti, tj);
    const int wave = threadIdx.x >> 6;
    const float* part = a.partial + mt * (BM * BM) + threadIdx.x * 4;
    typename T::Acc acc[T::TM][T::TN] = {};
    for (int s = 0; s < a.slices; ++s)
#pragma unroll
        for (int i = 0; i < T::TM; ++i)
#pragma unroll
            for (int j = 0; j < T::TN; ++j)
                acc[i][j] += *(const v4f*)(part + (long long)s * per * (BM * BM) + (i * T::TN + j) * T::THREADS * 4);
    ns_store_sym<T>(p, a, mat, (long long)ti * BM + (wave / WN) * (BM / WM), (long long)tj * BM + (wave % WN) * (BM / WN), ti == tj,
                    (LdsPtr)lds + wave * TURN_BYTES<T::TN>, acc);
}

// ---------------------------------------------------------------- a group of steps on a small A, in one launch
// l <= SIDE: a workgroup per matrix runs the group from A to S.  The matrices stay in registers as fp32 (a wavefront owns a
// block of T x T pieces on or below the diagonal), a product's two factors go through LDS in split form, written on both
// sides of the diagonal from the one value below it.  13 to 17 products of which each as a launch of its own costs 3.5 us
// take 9 us (30 rows), 16 us (64), 35 us (90), 53 us (128); LDS reads and the split writes share that time.
struct NsChain {
    const char* A;
    char* S;
    long long mat;           // bytes from matrix to matrix of A and S
    long long l, lk;
    float a, b, c;
    int steps;
    float scale_a, scale_r, scale_s;     // of the matrices in LDS; A comes at scale_a, S leaves at scale_s (scale_r after one step)
};

template <int SIDE, int T>
struct ChainGrid {
    static constexpr int ROWS = SIDE / (16 * T), WAVES = ROWS * (ROWS + 1) / 2, THREADS = WAVES * 64;
};

template <int SIDE, int T>
__global__ __launch_bounds__((ChainGrid<SIDE, T>::THREADS)) void ns_chain_kernel(NsChain p) {
    constexpr int LINE = SIDE * 4, THREADS = ChainGrid<SIDE, T>::THREADS;
    __shared__ __align__(1024) char left[SIDE * LINE], right[SIDE * LINE];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    int wi, wj;
    triangle(wave, wi, wj);
    const int m0 = wi * 16 * T + piece_across(lane), n0 = wj * 16 * T + piece_along(lane);     // of piece (0, 0)
    const int l = (int)p.l;
    typedef float Block[T][T][4];
    auto at = [](int row, int col) {       // byte of hi in LDS; lo is the chunk four further on
        const int chunk = (col & 31) >> 3;
        return row * LINE + (col >> 5) * 128 + ((chunk ^ (row & 7)) << 4) + (col & 7) * 2;
    };
    auto four = [](char* to, int q, const unsigned (&w)[4]) {        // words of hi (low half) and lo to two places of 8 bytes
        typedef unsigned v2u __attribute__((ext_vector_type(2)));
        *(v2u*)(to + q) = v2u{__builtin_amdgcn_perm(w[1], w[0], 0x05040100u), __builtin_amdgcn_perm(w[3], w[2], 0x05040100u)};
        *(v2u*)(to + (q ^ 64)) = v2u{__builtin_amdgcn_perm(w[1], w[0], 0x07060302u), __builtin_amdgcn_perm(w[3], w[2], 0x07060302u)};
    };
    // A lane's four neighbours of a row go to their place at once; four lanes of neighbouring rows exchange theirs (a 4x4
    // transposition, the lane one further, then the lane two further) and write four neighbours of a column to the other side.
    auto put = [&](char* to, const Block& v, float scale) {
        const bool odd = lane & 1, high = lane & 2;
#pragma unroll
        for (int i = 0; i < T; ++i)
#pragma unroll
            for (int j = 0; j < T; ++j) {
                const int m = m0 + i * 16, n = n0 + j * 16, mq = m & ~3;
                unsigned d[4], x[4], c[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    _Float16 hi, lo;
                    split_of(m < l && n + r < l ? v[i][j][r] * scale : 0.0f, hi, lo);
                    d[r] = (unsigned)__builtin_bit_cast(unsigned short, hi) | (unsigned)__builtin_bit_cast(unsigned short, lo) << 16;
                }
#pragma unroll
                for (int r = 0; r < 4; r += 2) {
                    const unsigned got = (unsigned)__builtin_amdgcn_mov_dpp((int)(odd ? d[r] : d[r + 1]), 0xB1, 0xF, 0xF, true);
                    x[r] = odd ? got : d[r];
                    x[r + 1] = odd ? d[r + 1] : got;
                }
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const unsigned got = (unsigned)__builtin_amdgcn_mov_dpp((int)(high ? x[r] : x[r + 2]), 0x4E, 0xF, 0xF, true);
                    c[r] = high ? got : x[r];
                    c[r + 2] = high ? x[r + 2] : got;
                }
                if (n < mq) {
                    four(to, at(m, n), d);
                    four(to, at(n + (m & 3), mq), c);
                } else if (n == mq) {                 // the 4x4 block on the diagonal: each side from below it
#pragma unroll
                    for (int r = 0; r < 4; ++r) d[r] = r <= (m & 3) ? d[r] : c[r];
                    four(to, at(m, n), d);
                }
            }
    };
    // out = k * (P Q'), this wavefront's block
    auto product = [&](const char* P, const char* Q, float k, Block& out) {
        v4f acc[T][T] = {};
        const int lr = lane & 15, lq = lane >> 4;
        const int c0 = (lq ^ (lr & 7)) << 4, c1 = ((4 + lq) ^ (lr & 7)) << 4;
        const int pb = (wi * 16 * T + lr) * LINE, qb = (wj * 16 * T + lr) * LINE;
#pragma unroll
        for (int kb = 0; kb < SIDE / 32; ++kb) {
            v4i fb[T][2];
#pragma unroll
            for (int j = 0; j < T; ++j) {
                fb[j][0] = *(const v4i*)(Q + qb + j * 16 * LINE + kb * 128 + c0);
                fb[j][1] = *(const v4i*)(Q + qb + j * 16 * LINE + kb * 128 + c1);
            }
#pragma unroll
            for (int i = 0; i < T; ++i) {
                v4i fa[2];
                fa[0] = *(const v4i*)(P + pb + i * 16 * LINE + kb * 128 + c0);
                fa[1] = *(const v4i*)(P + pb + i * 16 * LINE + kb * 128 + c1);
                mma_row<MathSplit, true, 0, T>(acc[i], fa, fb);
            }
        }
#pragma unroll
        for (int i = 0; i < T; ++i)
#pragma unroll
            for (int j = 0; j < T; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) out[i][j][r] = k * acc[i][j][r];
    };
    auto mix = [&](Block& v, float x, const Block& u) {        // v += x * u
#pragma unroll
        for (int i = 0; i < T; ++i)
#pragma unroll
            for (int j = 0; j < T; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) v[i][j][r] += x * u[i][j][r];
    };
    Block A, R, X, S;
    const char* ga = p.A + blockIdx.x * p.mat;
    const long long ld = p.lk * 4;
#pragma unroll
    for (int i = 0; i < T; ++i)
#pragma unroll
        for (int j = 0; j < T; ++j) {
            const int m = m0 + i * 16, n = n0 + j * 16;
            float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (m < l && n < p.lk) split_get_n<4>(ga + split_at(m, ld, n), v);
#pragma unroll
            for (int r = 0; r < 4; ++r) A[i][j][r] = v[r] / p.scale_a;
        }
    float q = p.a;
    for (int step = 0; step < p.steps; ++step) {
        const bool last = step + 1 == p.steps;
        put(left, A, p.scale_a);
        __syncthreads();
        product(left, left, p.c / (p.scale_a * p.scale_a), R);
        mix(R, p.b, A);
        put(right, R, p.scale_r);
        __syncthreads();
        if (!last) {
            product(right, left, 1.0f / (p.scale_r * p.scale_a), X);
            mix(X, p.a, A);
        }
        if (step == 0) {
#pragma unroll
            for (int i = 0; i < T; ++i)
#pragma unroll
                for (int j = 0; j < T; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) S[i][j][r] = R[i][j][r];
        } else {
            __syncthreads();
            put(left, S, p.scale_s);
            __syncthreads();
            Block N;
            product(right, left, 1.0f / (p.scale_r * p.scale_s), N);
            mix(N, p.a, S);
            mix(N, q, R);
            q *= p.a;
#pragma unroll
            for (int i = 0; i < T; ++i)
#pragma unroll
                for (int j = 0; j < T; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) S[i][j][r] = N[i][j][r];
        }
        __syncthreads();
        if (!last) {
            put(left, X, p.scale_a);
            __syncthreads();
            product(left, right, 1.0f / (p.scale_a * p.scale_r), A);
            mix(A, p.a, X);
            __syncthreads();
        }
    }
    put(left, S, p.steps == 1 ? p.scale_r : p.scale_s);
    __syncthreads();
    char* gs = p.S + blockIdx.x * p.mat;
    const int row_chunks = (int)(p.lk / 4);          // of 16 bytes
    for (int i = t; i < l * row_chunks; i += THREADS) {
        const int row = i / row_chunks, chunk = i - row * row_chunks;
        *(v4i*)(gs + row * ld + chunk * 16) = *(const v4i*)(left + row * LINE + (chunk >> 3) * 128 + (((chunk & 7) ^ (row & 7)) << 4));
    }
}

// S split -> the planes hi and lo of each row, lh numbers each.  4096 x 4096: 25 us (134 MB); 4 x 512 x 512: 4 us, a launch.
static __global__ __launch_bounds__(256) void ns_planes_kernel(const char* __restrict__ S, long long s_mat, char* __restrict__ planes,
                                                               long long planes_mat, NsShape sh) {
    const long long eights = sh.lh / 8, total = sh.l * eights;
    const char* from = S + blockIdx.y * s_mat;
    char* to = planes + blockIdx.y * planes_mat;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const long long row = i / eights, col = (i - row * eights) * 8;
        v4i hi = {0, 0, 0, 0}, lo = hi;
        if (col < sh.lk) {
            const char* p = from + split_at(row, sh.lk * 4, col);
            hi = *(const v4i*)p;
            lo = *(const v4i*)(p + 64);
        }
        char* q = to + row * sh.lh * 4 + col * 2;
        *(v4i*)q = hi;
        *(v4i*)(q + sh.lh * 2) = lo;
    }
}

// ---------------------------------------------------------------- Y = q X + S X
enum { NS_OUT_RESULT = 0, NS_OUT_WEIGHT = 1, NS_OUT_SPLIT = 2 };

struct NsApply {
    const char *S, *X, *Xt;
    long long s_mat, x_mat, xt_mat;
    NsShape sh;
    const float* factor;             // of each matrix: Y times it (NS_OUT_SPLIT: to what is held next)
    float k0, k1;                    // Y = k0 * (S X) + k1 * X
    // NS_OUT_RESULT
    void* out;
    long long out_b, out_r;          // elements from matrix to matrix and row to row
    int store;                       // how a row of the result, or of the weights, is stored
    // NS_OUT_WEIGHT
    void* param[NS_MAX_LIST];
    float decay, step;               // p = decay * p - step * Y
    // NS_OUT_SPLIT
    char *Yn, *Yt;
};

template <int DT, int OUT, bool TALL, bool HALF, int BM, int BN, int WM, int WN, int STAGES>
__global__ __launch_bounds__(64 * WM * WN, 2) void ns_apply_kernel(NsApply a) {
    // a lane's four numbers lie along a row of the result: along n, or along l when X is G'
    typedef typename std::conditional<HALF, MathHalf, MathSplit>::type Math;
    typedef TileProduct<Math, BM, BN, WM, WN, STAGES, !TALL> T;
    typedef typename Elem<DT>::T E;
    YH_TILE_RING(T)
    const NsShape& sh = a.sh;
    const int tl = (int)((sh.l + BM - 1) / BM);
    const long long tn = (sh.n + BN - 1) / BN, per = tl * tn;
    const long long id = xcd_order(blockIdx.x, per * sh.count);
    const long long mat = id / per, tile = id - mat * per;
    const long long ti = tile % tl, tj = tile / tl;
    typename T::Acc acc[T::TM][T::TN] = {};
    const long long ld = HALF ? sh.lh * 2 : sh.lk * 4, ldn = HALF ? sh.nh * 2 : sh.nk * 4;
    const long long lds = HALF ? sh.lh * 4 : ld;         // S: both planes of a row
    const TileOperand A = {a.S + mat * a.s_mat, lds, sh.l, ti * BM, lds - 16};
    const TileOperand B = {a.Xt + mat * a.xt_mat, ld, sh.n, tj * BN, ld - 16, HALF ? (int)(sh.lh / 64) : 1 << 30};
    T::run(A, B, 0, (int)(lds / TILE_BLOCK_BYTES), ring, acc);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const char* x = TALL ? a.Xt + mat * a.xt_mat : a.X + mat * a.x_mat;
    const long long ldx = TALL ? ld : ldn;
    const long long cols = TALL ? sh.l : sh.n, rows = TALL ? sh.n : sh.l, cols_pad = TALL ? sh.lk : sh.nk;
    const long long mw = ti * BM + (wave / WN) * (BM / WM), nw = tj * BN + (wave % WN) * (BN / WN);
    constexpr int ACROSS = TALL ? T::TN : T::TM, ALONG = TALL ? T::TM : T::TN;
    static_assert((T::WAVES + 1) / 2 * TURN_BYTES<ALONG> <= T::HALF, "fits two stages");
    __syncthreads();
    LdsPtr turn = (wave & 1 ? ring[1] : ring[0]) + (wave >> 1) * TURN_BYTES<ALONG>;
    const float factor = a.factor[mat];
    const float k0 = a.k0 * factor, k1 = a.k1 * factor;
#pragma unroll
    for (int i = 0; i < ACROSS; ++i) {
        float d[ALONG][4];
#pragma unroll
        for (int j = 0; j < ALONG; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) d[j][r] = k0 * (TALL ? acc[j][i][r] : acc[i][j][r]);
        turn_in<ALONG>(turn, d);
        const long long r0 = (TALL ? nw : mw) + i * 16, c0 = TALL ? mw : nw;
        // v += k1 * X; false where there is nothing
        auto add = [&](long long row, long long col, auto& v) {
            constexpr int W = (int)(sizeof(v) / sizeof(float));
            if (row >= rows || col >= cols_pad) return false;
            float e[W];
            if constexpr (HALF) half_get_n<W>(x + row * ldx + col * 2, e);
            else split_get_n<W>(x + split_at(row, ldx, col), e);
#pragma unroll
            for (int k = 0; k < W; ++k) v[k] += k1 * e[k];
            return true;
        };
        if constexpr (OUT == NS_OUT_SPLIT) {
            turn_out<ALONG, 8>(turn, [&](int r, int c, float (&v)[8]) {
                const long long row = r0 + r, col = c0 + c;
                const bool in = add(row, col, v);
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (!in || col + k >= cols) v[k] = 0.0f;
                if (in) split8_put(a.Yn + mat * a.x_mat + split_at(row, ldn, col), v);
#pragma unroll
                for (int k = 0; k < 8; k += 4)
                    *(__attribute__((address_space(3))) v4f*)(turn + r * TURN_LINE<ALONG> + (c + k) * 4) = v4f{v[k], v[k + 1], v[k + 2], v[k + 3]};
            });
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int c = lane; c < ALONG * 32; c += 64) {        // rows of X', eight neighbours along l; they end in zeros
                const int col = c % (ALONG * 16), half = c / (ALONG * 16) * 8;
                float v[8];
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    v[k] = *(const __attribute__((address_space(3))) float*)(turn + (half + k) * TURN_LINE<ALONG> + col * 4);
                if (c0 + col < cols && r0 + half < sh.lk) split8_put(a.Yt + mat * a.xt_mat + split_at(c0 + col, ld, r0 + half), v);
            }
        } else {
            auto emit = [&](int r, int c, auto& v) {
                constexpr int W = (int)(sizeof(v) / sizeof(float));
                const long long row = r0 + r, col = c0 + c;
                if (!add(row, col, v)) return;
                if constexpr (OUT == NS_OUT_RESULT) {
                    put_row<DT, W>((E*)a.out + mat * a.out_b, row, col, rows, cols, a.out_r, v);
                } else {
                    E* p = (E*)a.param[mat];
                    float w[W];
                    get_row<DT, W>(p, row, col, cols, w);
#pragma unroll
                    for (int k = 0; k < W; ++k) w[k] = a.decay * w[k] - a.step * v[k];
                    put_row<DT, W>(p, row, col, rows, cols, cols, w);
                }
            };
            if (a.store == STORE_16) turn_out<ALONG, 16 / (int)sizeof(E)>(turn, emit);
            else if (sizeof(E) == 2 && a.store == STORE_PAIR) turn_out<ALONG, 2>(turn, emit);
            else turn_out<ALONG, 1>(turn, emit);
        }
    }
}

}  // namespace yh
