// The product of a linear layer in 8-bit integers: y = s_m t_n sum_k q_mk w_nk + bias_n, with a scale for
// every row of x (an image's features) and every row of w (an output channel).
//   s_m  = amax_k |x_mk| / 127          q_mk = round_half_even(127 x_mk / amax_m)   (the exact quotient)
// The sum is exact in int32 (|q|, |w| <= 128 and K <= 131,071), so no order of additions changes a bit
// of it; the scales and the bias are applied in fp32 and the result is rounded once to its type.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "tile_product.hpp"

namespace yh {

enum { DT_F32 = 0, DT_F16 = 1, DT_BF16 = 2, DT_I8 = 3 };

__device__ __forceinline__ float bf16_to_f32(unsigned short u) { return __uint_as_float((unsigned)u << 16); }
// round to nearest even; a NaN stays one
__device__ __forceinline__ unsigned short f32_to_bf16(float f) {
    const unsigned u = __float_as_uint(f);
    if ((u & 0x7fffffffu) > 0x7f800000u) return (unsigned short)((u >> 16) | 0x40u);
    return (unsigned short)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}

template <int DT> struct Elem;
template <> struct Elem<DT_F32> {
    using T = float;
    static __device__ __forceinline__ float get(T v) { return v; }
    static __device__ __forceinline__ T put(float f) { return f; }
};
template <> struct Elem<DT_F16> {
    using T = _Float16;
    static __device__ __forceinline__ float get(T v) { return (float)v; }
    static __device__ __forceinline__ T put(float f) { return (_Float16)f; }
};
template <> struct Elem<DT_BF16> {
    using T = unsigned short;
    static __device__ __forceinline__ float get(T v) { return bf16_to_f32(v); }
    static __device__ __forceinline__ T put(float f) { return f32_to_bf16(f); }
};

// four consecutive numbers to p (aligned to their size when `whole`)
template <int DT>
__device__ __forceinline__ void put4(typename Elem<DT>::T* p, const float (&v)[4], int n, bool whole) {
    typedef typename Elem<DT>::T T;
    typedef T T4 __attribute__((ext_vector_type(4)));
    if (whole && n >= 4) {
        T4 o;
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r] = Elem<DT>::put(v[r]);
        *(T4*)p = o;
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (r < n) p[r] = Elem<DT>::put(v[r]);
    }
}

// ---------------------------------------------------------------- quantisation
// 127 x / amax to the nearest whole number, ties to even, as the exact quotient has it.  t is off by at most
// 2^-44; a quotient of two 24-bit numbers that is no tie is at least 2^-34 away from one, so rounding t to a
// multiple of 2^-38 first (adding and taking away 1.5 * 2^14: 52 - 14 = 38 bits stay behind the point) brings
// every tie back to where it is and moves nothing across one.
__device__ __forceinline__ int quantize_one(float x, double inv) {
    double t = (double)x * inv;
    t = (t + 24576.0) - 24576.0;
    return (int)__builtin_rint(t);
}

// One workgroup per row; VEC: 16-byte loads (ldx and x allow them).  The row is read twice, the second time out
// of L2.  A row that holds a NaN or an infinity gets the scale NaN and zeros, so every y of it is NaN.
// Zeros are written from K to Kz (the padding the product's blocks of 128 bytes read).
template <int DT, int THREADS>
__global__ __launch_bounds__(THREADS) void quantize_rows_kernel(const typename Elem<DT>::T* __restrict__ x,
                                                                long long ldx, int8_t* __restrict__ q, long long ldq,
                                                                float* __restrict__ scale, int K, int Kz, int vec) {
    typedef typename Elem<DT>::T T;
    constexpr int V = 16 / (int)sizeof(T);
    typedef T TV __attribute__((ext_vector_type(V)));
    const T* row = x + (long long)blockIdx.x * ldx;
    int8_t* out = q + (long long)blockIdx.x * ldq;
    const int t = threadIdx.x;
    __shared__ unsigned part[THREADS / 64];
    // |x| as an integer orders as the number does, with infinities and NaNs above all numbers
    unsigned top = 0;
    if (vec) {
        const int nv = K / V;
        for (int i = t; i < nv; i += THREADS) {
            const TV v = ((const TV*)row)[i];
#pragma unroll
            for (int e = 0; e < V; ++e) top = max(top, __float_as_uint(Elem<DT>::get(v[e])) & 0x7fffffffu);
        }
        for (int i = nv * V + t; i < K; i += THREADS) top = max(top, __float_as_uint(Elem<DT>::get(row[i])) & 0x7fffffffu);
    } else {
        for (int i = t; i < K; i += THREADS) top = max(top, __float_as_uint(Elem<DT>::get(row[i])) & 0x7fffffffu);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, o));
    if ((t & 63) == 0) part[t >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) top = max(top, part[w]);
    const float amax = __uint_as_float(top);
    const bool finite = top < 0x7f800000u;
    if (t == 0) scale[blockIdx.x] = finite ? amax / 127.0f : __uint_as_float(0x7fc00000u);
    const double inv = finite && amax > 0.0f ? 127.0 / (double)amax : 0.0;
    // 16 results at a time (q and ldq are multiples of 16 bytes)
    for (int i = t * 16; i < Kz; i += THREADS * 16) {
        float v[16];
        if (vec && i + 16 <= K) {
#pragma unroll
            for (int c = 0; c < 16 / V; ++c) {
                const TV u = *(const TV*)(row + i + c * V);
#pragma unroll
                for (int e = 0; e < V; ++e) v[c * V + e] = Elem<DT>::get(u[e]);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] = i + e < K ? Elem<DT>::get(row[i + e]) : 0.0f;
        }
        union {
            v4i w;
            int8_t b[16];
        } o;
#pragma unroll
        for (int e = 0; e < 16; ++e) o.b[e] = (int8_t)(finite ? quantize_one(v[e], inv) : 0);
        if (i + 16 <= Kz) *(v4i*)(out + i) = o.w;
        else
            for (int e = 0; e < Kz - i; ++e) out[i + e] = o.b[e];
    }
}

// rows of 8-bit integers whose bytes past K are anything -> rows padded with zeros to Kz
static __global__ __launch_bounds__(256) void repack_rows_kernel(const int8_t* __restrict__ x, long long ldx,
                                                          int8_t* __restrict__ q, long long ldq, int K, int Kz) {
    const int8_t* row = x + (long long)blockIdx.x * ldx;
    int8_t* out = q + (long long)blockIdx.x * ldq;
    for (int i = threadIdx.x * 4; i < Kz; i += 1024) {
        unsigned w = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) w |= (i + e < K ? (unsigned)(uint8_t)row[i + e] : 0u) << (8 * e);
        *(unsigned*)(out + i) = w;
    }
}

// ---------------------------------------------------------------- the product
struct LinearI8Args {
    const int8_t* q;        // (M, >= Kp) zeros past K
    const int8_t* w;
    const float *sx, *sw, *bias;
    void* y;
    int* partial;           // (slices, M, N) when the contraction is split
    long long ldq, ldw, ldy, M, N;
    int last_w;             // start of the last 16-byte chunk of a row of w
    int blocks;             // of 128 bytes along K
    int slices, per_slice;  // the contraction in slices of per_slice blocks
    int tiles_m, tiles_n;
    int whole;              // four neighbours of a row of y may be stored at once
};

template <int DT>
__device__ __forceinline__ void linear_store(const LinearI8Args& a, long long m, long long n, const v4i& d) {
    if (m >= a.M || n >= a.N) return;
    const float s = a.sx[m];
    const int left = a.N - n < 4 ? (int)(a.N - n) : 4;
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int r = 0; r < 4; ++r)
        if (r < left) {
            v[r] = (float)d[r] * s * a.sw[n + r];
            if (a.bias) v[r] += a.bias[n + r];
        }
    put4<DT>((typename Elem<DT>::T*)a.y + m * a.ldy + n, v, left, a.whole);
}

template <int DT, int BM, int BN, int WM, int WN, int STAGES>
__global__ __launch_bounds__(64 * WM * WN, 2) void linear_i8_tile_kernel(LinearI8Args a) {
    typedef TileProduct<MathI8, BM, BN, WM, WN, STAGES, true> P;
    YH_TILE_RING(P)
    const long long tiles = (long long)a.tiles_m * a.tiles_n;
    const long long id = xcd_order(blockIdx.x, tiles * a.slices);
    const int slice = (int)(id / tiles);
    const long long tile = id - slice * tiles;
    // groups of eight tile rows, column by column: neighbours share both operands
    const long long per_group = 8ll * a.tiles_n;
    const long long g = tile / per_group, in = tile - g * per_group;
    const int rows = a.tiles_m - g * 8 < 8 ? (int)(a.tiles_m - g * 8) : 8;
    const long long tm = g * 8 + in % rows, tn = in / rows;
    typename P::Acc acc[P::TM][P::TN] = {};
    const TileOperand A = {(const char*)a.q, a.ldq, a.M, tm * BM, (long long)a.blocks * 128 - 16};
    const TileOperand B = {(const char*)a.w, a.ldw, a.N, tn * BN, a.last_w};
    const int k0 = slice * a.per_slice;
    const int k1 = k0 + a.per_slice < a.blocks ? k0 + a.per_slice : a.blocks;
    P::run(A, B, k0, k1, ring, acc);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long m0 = tm * BM + (wave / WN) * (BM / WM) + piece_across(lane);
    const long long n0 = tn * BN + (wave % WN) * (BN / WN) + piece_along(lane);
#pragma unroll
    for (int i = 0; i < P::TM; ++i)
#pragma unroll
        for (int j = 0; j < P::TN; ++j) {
            const long long m = m0 + i * 16, n = n0 + j * 16;
            if (a.slices == 1) {
                linear_store<DT>(a, m, n, acc[i][j]);
            } else if (m < a.M) {
                int* p = a.partial + ((long long)slice * a.M + m) * a.N + n;
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (n + r < a.N) p[r] = acc[i][j][r];
            }
        }
}

// the slices' sums (integers: any order gives the same), scales, bias
template <int DT>
__global__ __launch_bounds__(256) void linear_i8_join_kernel(LinearI8Args a) {
    const long long quads = (a.N + 3) / 4, total = a.M * quads, plane = a.M * a.N;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const long long m = i / quads, n = (i - m * quads) * 4;
        v4i d = {0, 0, 0, 0};
        for (int s = 0; s < a.slices; ++s) {
            const int* p = a.partial + s * plane + m * a.N + n;
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (n + r < a.N) d[r] += p[r];
        }
        linear_store<DT>(a, m, n, d);
    }
}

}  // namespace yh
