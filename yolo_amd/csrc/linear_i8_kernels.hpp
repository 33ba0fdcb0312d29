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
template <> struct Elem<DT_I8> {
    using T = int8_t;
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

// |x| as an integer orders as the number does, with infinities and NaNs above all numbers
__device__ __forceinline__ unsigned magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// N numbers: x * inv in fp32 is off by at most 127 * 2^-23, so its nearest whole number is the right one unless it lies
// that close to the middle of two; then (one number in 5,000, three groups of 16 in a thousand, and where numbers are halves of
// the largest) the group is done again in 64 bits, by the whole wavefront: one of its passes in five.  A pass without it
// takes a third of the cycles of 64 bits throughout, so the mean is about half.
template <int N>
__device__ __forceinline__ void quantize_some(const float (&x)[N], double inv, int8_t (&q)[N]) {
    const float f = (float)inv;
    bool near = false;
    float r[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
        const float t = x[e] * f;
        r[e] = __builtin_rintf(t);
        near |= fabsf(t - r[e]) > 0.4999f;
    }
    // inv outside fp32's normal range (rows of tiny numbers) goes the exact way too
    if (near || !(f > 1e-37f && f < 1e37f)) {
#pragma unroll
        for (int e = 0; e < N; ++e) r[e] = (float)quantize_one(x[e], inv);
    }
#pragma unroll
    for (int e = 0; e < N; ++e) q[e] = (int8_t)(int)r[e];
}

// 16 numbers of a row from i on, zeros past K; vec: the row lies on 16 bytes
template <int DT>
__device__ __forceinline__ void load16(const typename Elem<DT>::T* row, int i, int K, bool vec, float (&f)[16]) {
    typedef typename Elem<DT>::T T;
    constexpr int V = 16 / (int)sizeof(T);
    typedef T TV __attribute__((ext_vector_type(V)));
    if (vec && i + 16 <= K) {
#pragma unroll
        for (int p = 0; p < 16 / V; ++p) {
            const TV v = *(const TV*)(row + i + p * V);
#pragma unroll
            for (int e = 0; e < V; ++e) f[p * V + e] = Elem<DT>::get(v[e]);
        }
    } else {
        // every load is issued (the last number again past the end): loads behind conditions wait for each other
        T v[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = row[i + e < K ? i + e : K - 1];
#pragma unroll
        for (int e = 0; e < 16; ++e) f[e] = i + e < K ? Elem<DT>::get(v[e]) : 0.0f;
    }
}

template <int THREADS>
__device__ __forceinline__ unsigned row_top(unsigned top, unsigned* part) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, o));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) top = max(top, part[w]);
    return top;
}

// scale of the row and 127 / amax (0 where there is nothing to scale).  A row that holds a NaN or an infinity gets the
// scale NaN and zeros, so every y of it is NaN.
__device__ __forceinline__ double row_scale(unsigned top, float* scale) {
    const float amax = __uint_as_float(top);
    const bool finite = top < 0x7f800000u;
    if (threadIdx.x == 0) *scale = finite ? amax / 127.0f : __uint_as_float(0x7fc00000u);
    return finite && top ? 127.0 / (double)amax : 0.0;
}

union Quantized {
    v4i w;
    int8_t b[16];
};

// One workgroup per row, a thread 16 numbers at a time, held in registers between the maximum and the division
// (K <= THREADS * 16 * CHUNKS): every byte is read once and a row costs one trip to memory.  Zeros are written from K to
// Kz, a multiple of 16: the padding the product's blocks of 128 bytes read.  8,192 rows of 4,096 bf16: 23 to 28 us,
// 3.6 to 4.3 TB/s; 4,096 rows of 4,096 fp32: 15 us, 5.5 TB/s.
template <int DT, int THREADS, int CHUNKS>
__global__ __launch_bounds__(THREADS) void quantize_rows_kernel(const typename Elem<DT>::T* __restrict__ x, long long ldx,
                                                                int8_t* __restrict__ q, long long ldq,
                                                                float* __restrict__ scale, int K, int Kz, int vec) {
    __shared__ unsigned part[THREADS / 64];
    const typename Elem<DT>::T* row = x + (long long)blockIdx.x * ldx;
    int8_t* out = q + (long long)blockIdx.x * ldq;
    float v[CHUNKS][16];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) load16<DT>(row, (c * THREADS + (int)threadIdx.x) * 16, K, vec, v[c]);
    unsigned top = 0;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
        for (int e = 0; e < 16; ++e) top = max(top, magnitude(v[c][e]));
    const double inv = row_scale(row_top<THREADS>(top, part), scale + blockIdx.x);
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        const int at = (c * THREADS + (int)threadIdx.x) * 16;
        if (at >= Kz) break;
        Quantized o;
        o.w = v4i{0, 0, 0, 0};
        if (inv > 0.0) quantize_some(v[c], inv, o.b);
        *(v4i*)(out + at) = o.w;
    }
}

// Few long rows: a CU alone takes 4 us to bring in 100 KB, so PARTS workgroups share a row in two launches, the largest
// magnitudes of the parts first (tops: rows x PARTS).  64 rows of 50,176: 4.4 to 4.8 us each instead of
// 11 us.
constexpr int QUANT_PARTS = 16;

template <int DT>
__global__ __launch_bounds__(256) void quantize_top_kernel(const typename Elem<DT>::T* __restrict__ x, long long ldx,
                                                           unsigned* __restrict__ tops, int K, int span) {
    __shared__ unsigned part[4];
    const typename Elem<DT>::T* row = x + (long long)blockIdx.y * ldx;
    const int from = (int)blockIdx.x * span, to = from + span < K ? from + span : K;
    unsigned top = 0;
    for (int i = from + (int)threadIdx.x * 16; i < to; i += 4096) {
        float f[16];
        load16<DT>(row, i, K, true, f);
#pragma unroll
        for (int e = 0; e < 16; ++e) top = max(top, magnitude(f[e]));
    }
    top = row_top<256>(top, part);
    if (threadIdx.x == 0) tops[blockIdx.y * QUANT_PARTS + blockIdx.x] = top;
}

template <int DT>
__global__ __launch_bounds__(256) void quantize_part_kernel(const typename Elem<DT>::T* __restrict__ x, long long ldx,
                                                            int8_t* __restrict__ q, long long ldq, float* __restrict__ scale,
                                                            const unsigned* __restrict__ tops, int K, int Kz, int span) {
    const typename Elem<DT>::T* row = x + (long long)blockIdx.y * ldx;
    int8_t* out = q + (long long)blockIdx.y * ldq;
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < QUANT_PARTS; ++i) top = max(top, tops[blockIdx.y * QUANT_PARTS + i]);
    const float amax = __uint_as_float(top);
    const bool finite = top < 0x7f800000u;
    if (blockIdx.x == 0 && threadIdx.x == 0) scale[blockIdx.y] = finite ? amax / 127.0f : __uint_as_float(0x7fc00000u);
    const double inv = finite && top ? 127.0 / (double)amax : 0.0;
    const int from = (int)blockIdx.x * span, to = from + span < Kz ? from + span : Kz;
    for (int i = from + (int)threadIdx.x * 16; i < to; i += 4096) {
        Quantized o;
        o.w = v4i{0, 0, 0, 0};
        if (inv > 0.0) {
            float f[16];
            load16<DT>(row, i, K, true, f);
            quantize_some(f, inv, o.b);
        }
        *(v4i*)(out + i) = o.w;
    }
}

// rows of any length: read twice, the second time out of L2
template <int DT>
__global__ __launch_bounds__(1024) void quantize_long_rows_kernel(const typename Elem<DT>::T* __restrict__ x, long long ldx,
                                                                 int8_t* __restrict__ q, long long ldq,
                                                                 float* __restrict__ scale, int K, int Kz) {
    __shared__ unsigned part[16];
    const typename Elem<DT>::T* row = x + (long long)blockIdx.x * ldx;
    int8_t* out = q + (long long)blockIdx.x * ldq;
    unsigned top = 0;
    for (int i = threadIdx.x; i < K; i += 1024) top = max(top, magnitude(Elem<DT>::get(row[i])));
    const double inv = row_scale(row_top<1024>(top, part), scale + blockIdx.x);
    for (int i = threadIdx.x * 4; i < Kz; i += 4096) {
        unsigned o = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (i + e < K && inv > 0.0) o |= (unsigned)(uint8_t)(int8_t)quantize_one(Elem<DT>::get(row[i + e]), inv) << (8 * e);
        *(unsigned*)(out + i) = o;
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
    int store;              // how a row of y is stored
};

enum { STORE_ONE = 0, STORE_PAIR = 1, STORE_16 = 2 };   // rows lie on their numbers' size, on twice that, on 16 bytes

// WIDTH neighbouring numbers of a row of y (rows x cols), as one store where they are all inside
template <int DT, int WIDTH>
__device__ __forceinline__ void put_row(typename Elem<DT>::T* y, long long row, long long col, long long rows, long long cols,
                                        long long ld, const float (&v)[WIDTH]) {
    typedef typename Elem<DT>::T T;
    if (row >= rows) return;
    T* p = y + row * ld + col;
    if (col + WIDTH <= cols) {
        if constexpr (WIDTH == 1) {
            *p = Elem<DT>::put(v[0]);
        } else {
            typedef T TV __attribute__((ext_vector_type(WIDTH)));
            TV o;
#pragma unroll
            for (int e = 0; e < WIDTH; ++e) o[e] = Elem<DT>::put(v[e]);
            *(TV*)p = o;
        }
    } else {
#pragma unroll
        for (int e = 0; e < WIDTH; ++e)
            if (col + e < cols) p[e] = Elem<DT>::put(v[e]);
    }
}

// the same from a matrix without gaps between rows; zeros past its columns
template <int DT, int WIDTH>
__device__ __forceinline__ void get_row(const typename Elem<DT>::T* y, long long row, long long col, long long cols, float (&v)[WIDTH]) {
    typedef typename Elem<DT>::T T;
    const T* p = y + row * cols + col;
    if constexpr (WIDTH > 1) {
        if (col + WIDTH <= cols) {
            typedef T TV __attribute__((ext_vector_type(WIDTH)));
            const TV o = *(const TV*)p;
#pragma unroll
            for (int e = 0; e < WIDTH; ++e) v[e] = Elem<DT>::get(o[e]);
            return;
        }
    }
#pragma unroll
    for (int e = 0; e < WIDTH; ++e) v[e] = col + e < cols ? Elem<DT>::get(p[e]) : 0.0f;
}

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
    put4<DT>((typename Elem<DT>::T*)a.y + m * a.ldy + n, v, left, a.store == STORE_16);
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
    const long long mw = tm * BM + (wave / WN) * (BM / WM), nw = tn * BN + (wave % WN) * (BN / WN);
    const long long m0 = mw + piece_across(lane), n0 = nw + piece_along(lane);
    if (a.slices > 1) {
#pragma unroll
        for (int i = 0; i < P::TM; ++i)
#pragma unroll
            for (int j = 0; j < P::TN; ++j) {
                const long long m = m0 + i * 16, n = n0 + j * 16;
                if (m >= a.M) continue;
                int* p = a.partial + ((long long)slice * a.M + m) * a.N + n;
                if (a.N % 4 == 0) {
                    if (n < a.N) *(v4i*)p = acc[i][j];
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (n + r < a.N) p[r] = acc[i][j][r];
                }
            }
        return;
    }
    typedef typename Elem<DT>::T T;
    float w[P::TN][4], b[P::TN][4];
#pragma unroll
    for (int j = 0; j < P::TN; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const long long n = n0 + j * 16 + r < a.N ? n0 + j * 16 + r : a.N - 1;
            w[j][r] = a.sw[n];
            b[j][r] = a.bias ? a.bias[n] : 0.0f;
        }
    __syncthreads();
    static_assert((P::WAVES + 1) / 2 * TURN_BYTES<P::TN> <= P::HALF, "fits two stages");
    LdsPtr turn = (wave & 1 ? ring[1] : ring[0]) + (wave >> 1) * TURN_BYTES<P::TN>;
#pragma unroll
    for (int i = 0; i < P::TM; ++i) {
        const long long m = m0 + i * 16;
        const float s = a.sx[m < a.M ? m : a.M - 1];
        float v[P::TN][4];
#pragma unroll
        for (int j = 0; j < P::TN; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                v[j][r] = (float)acc[i][j][r] * s * w[j][r];
                if (a.bias) v[j][r] += b[j][r];
            }
        turn_in<P::TN>(turn, v);
        auto emit = [&](int row, int col, const auto& x) { put_row<DT>((T*)a.y, mw + i * 16 + row, nw + col, a.M, a.N, a.ldy, x); };
        if (a.store == STORE_16) turn_out<P::TN, 16 / (int)sizeof(T)>(turn, emit);
        else if (sizeof(T) == 2 && a.store == STORE_PAIR) turn_out<P::TN, 2>(turn, emit);
        else turn_out<P::TN, 1>(turn, emit);
    }
}

// Up to 16 rows a workgroup (blockIdx.y: which): the weight is read once, straight into registers, and that is what bounds
// it.  A workgroup of 16 wavefronts takes 16 channels; a wavefront takes every 16th block of 128 bytes of their rows, four
// blocks (8 KB) on their way while four are worked on; the 16 sums meet in LDS.  STAGE: every workgroup brings the rows of x
// into LDS for itself, quantised where they are not 8-bit already and padded with zeros, while its first weights are on
// their way: for few rows that is less than a launch of its own.  Otherwise a.q holds the padded rows.  1 x 4096 -> 1470:
// 7 us (6.0 MB; the host's part of a call is 11); 1 x 50,176 -> 4096: 44 to 46 us, 4.5 to 4.7 TB/s of weights (copies reach 5.1).  Loads past the end of
// a row, the same line from every wavefront, took 1 x 4096 to 13 us: none is issued.
template <int DTX, int DT, bool STAGE>
__global__ __launch_bounds__(1024) void linear_i8_rows_kernel(LinearI8Args a, const typename Elem<DTX>::T* __restrict__ x,
                                                              long long ldx, int K, int vec) {
    typedef typename Elem<DTX>::T T;
    constexpr int AHEAD = 4, WAVES = 16;
    extern __shared__ __align__(16) char rows_lds[];        // STAGE: the rows, a.blocks * 128 bytes each
    __shared__ __align__(16) v4i sums[WAVES][64];
    __shared__ unsigned part[WAVES];
    __shared__ float row_s[16];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int lr = lane & 15, lq = (lane >> 4) * 16;
    const long long n0 = (long long)blockIdx.x * 16, m0 = (long long)blockIdx.y * 16;
    const int M = a.M - m0 < 16 ? (int)(a.M - m0) : 16;
    const char* w = (const char*)a.w + (n0 + lr < a.N ? n0 + lr : a.N - 1) * a.ldw;
    const int m = lr < M ? lr : M - 1;
    const int row_bytes = a.blocks * 128;
    const char* q = (const char*)a.q + (m0 + m) * a.ldq;
    const int last = a.blocks - 1;
    v4i wr[2][AHEAD][2];
    auto fetch = [&](v4i (&r)[AHEAD][2], int kb) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
            if (kb + u * WAVES <= last) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int off = (kb + u * WAVES) * 128 + h * 64 + lq;
                    r[u][h] = *(const v4i*)(w + (off < a.last_w ? off : a.last_w));
                }
            }
    };
    fetch(wr[0], wave);
    if constexpr (STAGE) {
        // 1024 / rows threads (rounded down to a power of two) to a row, 16 numbers at a time
        int per = 1024;
        while (per * M > 1024) per >>= 1;
        const int row = t / per, at0 = (t & (per - 1)) * 16;
        const bool mine = row < M;
        const T* xr = x + (m0 + (mine ? row : 0)) * ldx;
        const int end = mine ? K : 0, pad = mine ? row_bytes : 0;
        if constexpr (DTX == DT_I8) {
            if (mine && at0 == 0) row_s[row] = a.sx[m0 + row];
            for (int i = at0; i < pad; i += per * 16) {
                Quantized o;
                if (vec && i + 16 <= end) {
                    o.w = *(const v4i*)(xr + i);
                } else {
#pragma unroll
                    for (int e = 0; e < 16; ++e) o.b[e] = i + e < end ? xr[i + e] : (int8_t)0;
                }
                *(v4i*)(rows_lds + row * row_bytes + i) = o.w;
            }
        } else {
            unsigned top = 0;
            float held[16];                              // short rows are read once
            const bool once = K <= per * 16;
            load16<DTX>(xr, mine ? at0 : K, K, vec, held);
#pragma unroll
            for (int e = 0; e < 16; ++e) top = max(top, magnitude(held[e]));
#pragma unroll 4
            for (int i = at0 + per * 16; i < end; i += per * 16) {
                float f[16];
                load16<DTX>(xr, i, K, vec, f);
#pragma unroll
                for (int e = 0; e < 16; ++e) top = max(top, magnitude(f[e]));
            }
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, o));
            if (lane == 0) part[wave] = top;
            __syncthreads();
            const int span = per / 64, first = (wave / span) * span;      // per is 64 at least: M <= 16
            for (int i = 0; i < span; ++i) top = max(top, part[first + i]);
            const float amax = __uint_as_float(top);
            const bool finite = top < 0x7f800000u;
            const double inv = finite && top ? 127.0 / (double)amax : 0.0;
            if (mine && at0 == 0) row_s[row] = finite ? amax / 127.0f : __uint_as_float(0x7fc00000u);
#pragma unroll 4
            for (int i = at0; i < pad; i += per * 16) {
                Quantized o;
                o.w = v4i{0, 0, 0, 0};
                if (inv > 0.0) {
                    if (!once) load16<DTX>(xr, i, K, vec, held);
                    quantize_some(held, inv, o.b);
                }
                *(v4i*)(rows_lds + row * row_bytes + i) = o.w;
            }
        }
        __syncthreads();
    }
    v4i acc = {0, 0, 0, 0};
    auto work = [&](const v4i (&r)[AHEAD][2], int kb) {
        v4i xr[AHEAD][2];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int b = kb + u * WAVES < last ? kb + u * WAVES : last;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int off = b * 128 + h * 64 + lq;
                xr[u][h] = *(const v4i*)(STAGE ? rows_lds + m * row_bytes + off : q + off);
            }
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
            if (kb + u * WAVES <= last) {
                MathI8::mma<0>(acc, r[u], xr[u]);
                MathI8::mma<1>(acc, r[u], xr[u]);
            }
    };
    for (int kb = wave; kb <= last; kb += 2 * AHEAD * WAVES) {
        fetch(wr[1], kb + AHEAD * WAVES);
        work(wr[0], kb);
        fetch(wr[0], kb + 2 * AHEAD * WAVES);
        work(wr[1], kb + AHEAD * WAVES);
    }
    sums[wave][lane] = acc;
    __syncthreads();
    if (t < 64) {       // the channels lie along a lane's registers
        v4i d = sums[0][lane];
#pragma unroll
        for (int i = 1; i < WAVES; ++i) d += sums[i][lane];
        if (lr < M) {
            LinearI8Args b = a;
            if (STAGE) b.sx = row_s - m0;
            linear_store<DT>(b, m0 + lr, n0 + piece_along(lane), d);
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
#pragma unroll 8
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
