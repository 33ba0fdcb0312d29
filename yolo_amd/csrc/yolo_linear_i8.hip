// yh_quantize_rows and yh_linear_i8: the 8-bit product entry points of include/yolo_head.h.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/yolo_head.h"
#include "linear_i8_kernels.hpp"

namespace {

using namespace yh;

inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }
inline size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }
inline int launch_status() {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? YH_OK : (int)e;
}
inline size_t dtype_bytes(int dt) { return dt == YH_F32 ? 4 : dt == YH_I8 ? 1 : 2; }

constexpr int64_t kMaxRows = YH_MAX_I8_ROWS;      // a grid holds fewer than 2^32 threads, a row takes up to 1,024

// tops: rows * QUANT_PARTS words for the shared form, or null (yh_quantize_rows has no workspace)
template <int DT>
void quantize_launch(const void* x, int64_t ldx, int8_t* q, int64_t ldq, float* scale, unsigned* tops, int64_t rows, int K,
                     int Kz, hipStream_t st) {
    typedef typename Elem<DT>::T T;
    const dim3 grid((unsigned)rows);
    const T* p = (const T*)x;
    const int vec = aligned(x, 16) && (rows == 1 || (ldx * sizeof(T)) % 16 == 0);
    if (K > 65536)
        hipLaunchKernelGGL((quantize_long_rows_kernel<DT>), grid, dim3(1024), 0, st, p, ldx, q, ldq, scale, K, Kz);
    else if (tops && vec && rows < 256 && K > 8192) {
        const int span = ((Kz + QUANT_PARTS - 1) / QUANT_PARTS + 15) & ~15;
        const dim3 parts(QUANT_PARTS, (unsigned)rows);
        hipLaunchKernelGGL((quantize_top_kernel<DT>), parts, dim3(256), 0, st, p, ldx, tops, K, span);
        hipLaunchKernelGGL((quantize_part_kernel<DT>), parts, dim3(256), 0, st, p, ldx, q, ldq, scale, (const unsigned*)tops, K,
                           Kz, span);
    } else if (K <= 1024)
        hipLaunchKernelGGL((quantize_rows_kernel<DT, 64, 1>), grid, dim3(64), 0, st, p, ldx, q, ldq, scale, K, Kz, vec);
    else if (K <= 4096)
        hipLaunchKernelGGL((quantize_rows_kernel<DT, 256, 1>), grid, dim3(256), 0, st, p, ldx, q, ldq, scale, K, Kz, vec);
    else if (K <= 16384)
        hipLaunchKernelGGL((quantize_rows_kernel<DT, 1024, 1>), grid, dim3(1024), 0, st, p, ldx, q, ldq, scale, K, Kz, vec);
    else
        hipLaunchKernelGGL((quantize_rows_kernel<DT, 1024, 4>), grid, dim3(1024), 0, st, p, ldx, q, ldq, scale, K, Kz, vec);
}

int quantize(const void* x, int dt, int64_t ldx, int8_t* q, int64_t ldq, float* scale, unsigned* tops, int64_t rows, int K,
             int Kz, hipStream_t st) {
    if (dt == YH_F32) quantize_launch<DT_F32>(x, ldx, q, ldq, scale, tops, rows, K, Kz, st);
    else if (dt == YH_F16) quantize_launch<DT_F16>(x, ldx, q, ldq, scale, tops, rows, K, Kz, st);
    else quantize_launch<DT_BF16>(x, ldx, q, ldq, scale, tops, rows, K, Kz, st);
    return launch_status();
}

// How the product is cut: tiles of one of four sizes, and slices of the contraction.
//
//   tile      wavefronts  stages  LDS     workgroups a CU   us for a block of 128 bytes: one workgroup on a CU, each more
//   256x128   8           3       144 KB  1                 1.08
//   128x128   8           4       128 KB  1                 0.65
//   64x64     4           4        64 KB  2                 0.30, 0.14
//   32x32     4           4        32 KB  5                 0.14, 0.08
//
// A larger tile reads less per product (a CU takes in about 64 bytes a cycle), a smaller one fills the card when
// there are few rows or channels.  The choice is the least time of: rounds of workgroups over the 256 CUs, times the
// blocks of a slice (+ 3 us to start and end), or the operands at 5 TB/s; plus, when the sums are joined, a launch and
// the traffic of the partial sums.  Measured (us, 32x32 / 64x64 / 128x128 / 256x128, each with its best slices):
// 64 x 4096 -> 1470 7.4 / 11.1 / 13.4 / -, 256 x 4096 -> 1470 8.4 / 10.3 / 17.9 / 26.3, 1024 x 4096 -> 4096 49.7 / 29.6 /
// 23.5 / 31.7, 512 x 50,176 -> 4096 353 / 205 / 132 / 119, 8192 x 4096 -> 4096 369 / 225 / 182 / 148.
struct Tile {
    int bm, bn, per_cu;
    double block, more;
};
constexpr int kTileKinds = 4;
constexpr Tile kTiles[kTileKinds] = {{256, 128, 1, 1.08, 0.0}, {128, 128, 1, 0.65, 0.0}, {64, 64, 2, 0.30, 0.14}, {32, 32, 5, 0.14, 0.08}};

struct Plan {
    int tile, tiles_m, tiles_n, slices, per_slice, blocks;
    size_t q_off, s_off, t_off, p_off, total;
};

Plan plan_for(int64_t M, int64_t N, int64_t K) {
    Plan p = {};
    p.blocks = (int)((K + 127) / 128);
    double best = 0.0;
    const double operands = ((double)N + (double)M) * (double)K / 5e6;
    for (int t = 0; t < kTileKinds; ++t) {
        const Tile& c = kTiles[t];
        const int64_t tm = (M + c.bm - 1) / c.bm, tn = (N + c.bn - 1) / c.bn, tiles = tm * tn;
        for (int s = 1; s <= 16 && s <= p.blocks; s *= 2) {
            if (s > 1 && tiles * s > 2048) break;
            const int64_t wgs = tiles * s, at_once = 256 * (int64_t)c.per_cu;
            const int per = (p.blocks + s - 1) / s;
            const int64_t together = wgs >= at_once ? c.per_cu : (wgs + 255) / 256;
            double us = (double)((wgs + at_once - 1) / at_once) * (per * (c.block + c.more * (double)(together - 1)) + 3.0);
            if (us < operands + 3.0) us = operands + 3.0;
            if (s > 1) us += 4.0 + (double)(s + 1) * (double)M * (double)N * 4.0 / 3e6;
            if (best == 0.0 || us < best) {
                best = us;
                p.tile = t;
                p.tiles_m = (int)tm;
                p.tiles_n = (int)tn;
                p.per_slice = per;
                p.slices = (p.blocks + per - 1) / per;
            }
        }
    }
    p.q_off = 0;
    p.s_off = up256((size_t)M * p.blocks * 128);
    p.t_off = p.s_off + up256((size_t)M * 4);
    p.p_off = p.t_off + (M < 256 ? up256((size_t)M * QUANT_PARTS * 4) : 0);
    p.total = p.p_off + (p.slices > 1 ? up256((size_t)p.slices * M * N * 4) : 0);
    return p;
}

constexpr int kRows = 16;      // rows of a workgroup of linear_i8_rows_kernel
// It brings the rows into LDS itself when that is less than a launch by itself (bf16 rows, kernel times in us of calls on one
// weight, with / without, the latter both launches: 1 x 4096 -> 1470 6.8 / 7.6, 4 x 4096 7.8 / 8.3, 16 x 4096 14.0 / 9.6, 1 x
// 50,176 -> 4096 39.2 / 43.7): up to 12,288 numbers or one row (8-bit rows, which are only copied: 65,536 bytes), and one
// workgroup a CU (64 x 700 -> 1470, 368 workgroups: 19.7 / 7.9).
inline bool stages_itself(int x_dtype, int64_t M, int64_t N, int64_t blocks) {
    const int64_t rows = M < kRows ? M : kRows;
    if (((M + kRows - 1) / kRows) * ((N + 15) / 16) > 256) return M <= kRows && M * blocks <= 96;
    return x_dtype == YH_I8 ? rows * blocks <= 512 && M <= kRows : blocks <= 512 && (M == 1 || rows * blocks <= 96);
}

template <int DTX, int DT, bool STAGE>
int few_rows(const LinearI8Args& a, const void* x, int64_t ldx, int K, hipStream_t st) {
    const int64_t rows = a.M < kRows ? a.M : kRows;
    const int vec = aligned(x, 16) && (a.M == 1 || (ldx * sizeof(typename Elem<DTX>::T)) % 16 == 0);
    hipLaunchKernelGGL((linear_i8_rows_kernel<DTX, DT, STAGE>), dim3((unsigned)((a.N + 15) / 16), (unsigned)((a.M + kRows - 1) / kRows)),
                       dim3(1024), STAGE ? (size_t)rows * a.blocks * 128 : 0, st, a, (const typename Elem<DTX>::T*)x, ldx, K, vec);
    return launch_status();
}

template <int DT>
int few_rows_of(const LinearI8Args& a, const void* x, int x_dtype, int64_t ldx, int K, hipStream_t st) {
    if (!x) return few_rows<DT_I8, DT, false>(a, nullptr, 0, K, st);      // a.q holds the rows
    if (x_dtype == YH_F32) return few_rows<DT_F32, DT, true>(a, x, ldx, K, st);
    if (x_dtype == YH_F16) return few_rows<DT_F16, DT, true>(a, x, ldx, K, st);
    if (x_dtype == YH_BF16) return few_rows<DT_BF16, DT, true>(a, x, ldx, K, st);
    return few_rows<DT_I8, DT, true>(a, x, ldx, K, st);
}

template <int DT, int BM, int BN, int WM, int WN, int STAGES>
void tiles(const LinearI8Args& a, hipStream_t st) {
    const unsigned grid = (unsigned)((int64_t)a.tiles_m * a.tiles_n * a.slices);
    hipLaunchKernelGGL((linear_i8_tile_kernel<DT, BM, BN, WM, WN, STAGES>), dim3(grid), dim3(64 * WM * WN), 0, st, a);
}

template <int DT>
int product(int tile, const LinearI8Args& a, hipStream_t st) {
    if (tile == 0) tiles<DT, 256, 128, 4, 2, 3>(a, st);
    else if (tile == 1) tiles<DT, 128, 128, 2, 4, 4>(a, st);
    else if (tile == 2) tiles<DT, 64, 64, 2, 2, 4>(a, st);
    else tiles<DT, 32, 32, 2, 2, 4>(a, st);
    if (const int rc = launch_status()) return rc;
    if (a.slices > 1) {
        int64_t b = (a.M * ((a.N + 3) / 4) + 255) / 256;
        if (b > 4096) b = 4096;
        hipLaunchKernelGGL((linear_i8_join_kernel<DT>), dim3((unsigned)b), dim3(256), 0, st, a);
    }
    return launch_status();
}

int check_sizes(int64_t M, int64_t N, int64_t K) {
    if (M < 0 || N < 0 || K < 1 || K > YH_MAX_I8_K || M > kMaxRows || N > kMaxRows) return YH_ERR_SHAPE;
    if (((M + 31) / 32) * ((N + 31) / 32) >= ((int64_t)1 << 24)) return YH_ERR_SHAPE;      // 256 threads a tile
    return YH_OK;
}

}  // namespace

extern "C" {

int yh_quantize_rows(const void* x, int x_dtype, int64_t ldx, int8_t* q, int64_t ldq, float* scale, int64_t rows,
                     int64_t K, void* stream) {
    if (rows < 0 || rows > kMaxRows || K < 1 || K > YH_MAX_I8_K || ldx < K || ldq < K) return YH_ERR_SHAPE;
    if (x_dtype != YH_F32 && x_dtype != YH_F16 && x_dtype != YH_BF16) return YH_ERR_ARG;
    if (rows == 0) return YH_OK;
    if (!x || !q || !scale) return YH_ERR_NULL;
    if (!aligned(x, dtype_bytes(x_dtype)) || !aligned(scale, 4) || !aligned(q, 16) || ldq % 16 != 0) return YH_ERR_ALIGN;
    int64_t Kz = (K + 127) / 128 * 128;
    if (Kz > ldq) Kz = ldq;
    return quantize(x, x_dtype, ldx, q, ldq, scale, nullptr, rows, (int)K, (int)Kz, (hipStream_t)stream);
}

size_t yh_linear_i8_workspace_bytes(int x_dtype, int64_t M, int64_t N, int64_t K) {
    if (check_sizes(M, N, K) != YH_OK || M == 0 || N == 0) return 0;
    return stages_itself(x_dtype, M, N, (K + 127) / 128) ? 0 : plan_for(M, N, K).total;
}

int yh_linear_i8(const void* x, int x_dtype, int64_t ldx, const float* x_scale, const int8_t* w, int64_t ldw,
                 const float* w_scale, const float* bias, void* y, int y_dtype, int64_t ldy, int64_t M, int64_t N,
                 int64_t K, void* workspace, size_t workspace_bytes, void* stream) {
    if (const int rc = check_sizes(M, N, K)) return rc;
    if (ldx < K || ldw < K || ldy < N) return YH_ERR_SHAPE;
    if (x_dtype < YH_F32 || x_dtype > YH_I8 || y_dtype < YH_F32 || y_dtype > YH_BF16) return YH_ERR_ARG;
    if ((x_dtype == YH_I8) != (x_scale != nullptr)) return YH_ERR_ARG;
    if (M == 0 || N == 0) return YH_OK;
    if (!x || !w || !w_scale || !y) return YH_ERR_NULL;
    const bool itself = stages_itself(x_dtype, M, N, (K + 127) / 128);
    Plan p = {};
    if (itself) p.blocks = (int)((K + 127) / 128);
    else p = plan_for(M, N, K);
    if (p.total && (!workspace || workspace_bytes < p.total)) return YH_ERR_WORKSPACE;
    if (!aligned(x, dtype_bytes(x_dtype)) || !aligned(x_scale, 4) || !aligned(w, 16) || ldw % 16 != 0 ||
        !aligned(w_scale, 4) || !aligned(bias, 4) || !aligned(y, dtype_bytes(y_dtype)) || !aligned(workspace, 256))
        return YH_ERR_ALIGN;
    hipStream_t st = (hipStream_t)stream;
    char* ws = (char*)workspace;
    LinearI8Args a = {};
    a.q = (const int8_t*)(ws + p.q_off);
    a.ldq = (long long)p.blocks * 128;
    a.sx = (const float*)(ws + p.s_off);
    a.w = w;
    a.ldw = ldw;
    a.sw = w_scale;
    a.bias = bias;
    a.y = y;
    a.ldy = ldy;
    a.partial = (int*)(ws + p.p_off);
    a.M = M;
    a.N = N;
    a.last_w = (int)((K + 15) / 16 * 16 - 16);
    a.blocks = p.blocks;
    a.slices = p.slices;
    a.per_slice = p.per_slice;
    a.tiles_m = p.tiles_m;
    a.tiles_n = p.tiles_n;
    const size_t e = dtype_bytes(y_dtype);
    a.store = (ldy * e) % 16 == 0 && aligned(y, 16) ? STORE_16 : ldy % 2 == 0 && aligned(y, 2 * e) ? STORE_PAIR : STORE_ONE;
    if (itself) {
        a.sx = x_scale;
        if (y_dtype == YH_F32) return few_rows_of<DT_F32>(a, x, x_dtype, ldx, (int)K, st);
        if (y_dtype == YH_F16) return few_rows_of<DT_F16>(a, x, x_dtype, ldx, (int)K, st);
        return few_rows_of<DT_BF16>(a, x, x_dtype, ldx, (int)K, st);
    }
    if (x_dtype != YH_I8) {
        const int rc = quantize(x, x_dtype, ldx, (int8_t*)(ws + p.q_off), a.ldq, (float*)(ws + p.s_off),
                                (unsigned*)(ws + p.t_off), M, (int)K,
                                (int)a.ldq, st);
        if (rc) return rc;
    } else {
        a.sx = x_scale;
        if (K % 128 == 0 && ldx % 16 == 0 && aligned(x, 16)) {
            a.q = (const int8_t*)x;
            a.ldq = ldx;
        } else {
            hipLaunchKernelGGL(repack_rows_kernel, dim3((unsigned)M), dim3(256), 0, st, (const int8_t*)x, ldx,
                               (int8_t*)(ws + p.q_off), a.ldq, (int)K, (int)a.ldq);
            if (const int rc = launch_status()) return rc;
        }
    }
    if (M <= kRows) {
        if (y_dtype == YH_F32) return few_rows_of<DT_F32>(a, nullptr, YH_I8, 0, (int)K, st);
        if (y_dtype == YH_F16) return few_rows_of<DT_F16>(a, nullptr, YH_I8, 0, (int)K, st);
        return few_rows_of<DT_BF16>(a, nullptr, YH_I8, 0, (int)K, st);
    }
    if (y_dtype == YH_F32) return product<DT_F32>(p.tile, a, st);
    if (y_dtype == YH_F16) return product<DT_F16>(p.tile, a, st);
    return product<DT_BF16>(p.tile, a, st);
}

}  // extern "C"
