// yh_orthogonalize and yh_muon_step: the entry points of the orthogonalised update (include/yolo_head.h).
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/yolo_head.h"
#include "orthogonalize_kernels.hpp"

namespace {

using namespace yh;

inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }
inline size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }
inline int launch_status() {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? YH_OK : (int)e;
}
inline size_t dtype_bytes(int dt) { return dt == YH_F32 ? 4 : 2; }

constexpr int64_t kMaxShort = 32768, kMaxLong = (int64_t)1 << 24, kMaxNumbers = (int64_t)1 << 38;
// Tiles of the products: us for a block of 32 numbers of the contraction with one workgroup on a CU, and for each more that
// fits; `start` us to begin and end.  The choice is the least time of its rounds over the 256 CUs.
// Symmetric products (us, 192 / 128 / 96 / 64 / 32; l = contraction unless stated, matrices in brackets): 192 22 / 9.9 / 12.8 / 6.2 /
// 4.4, 512 (4) 31 / 15 / 17.7 / 8.9 / 8.6, 1024 44 / 22 / 23 / 12.1 / 12.2, 1024 (4) 49 / 26 / 34 / 28 / 33, 1470 59 / 30 / 31 / 21 / 30,
// 2048 77 / 41 / 43 / 46 / 77, 2048 (2) - / 83 / 67 / 80 / -, 4096 183 / 239 / 238 / 339 / -, 4096 over 50,176 1974 / 2521 / - / 4531 / -:
// 4096 is 253 tiles of 192, one for each CU, but 528 of 128, two and a bit; two of 2048 are 506 tiles of 96, two for each.
// The times are those of split matrices, three products a block; X in fp16 alone, two a block, is cut by the same ones.
struct TileKind {
    int bm, bn, per_cu;
    double block, more, start;
};
enum { TILE_LARGE = 0, TILE_128 = 1, TILE_64 = 2, TILE_32 = 3, TILE_KINDS = 4, TILE_96 = 4, PRODUCT_KINDS = 5 };
constexpr TileKind kTiles[PRODUCT_KINDS] = {
    {192, 192, 1, 1.30, 0.0, 6.0}, {128, 128, 1, 0.58, 0.0, 4.3}, {64, 64, 2, 0.23, 0.14, 4.3}, {32, 32, 5, 0.10, 0.11, 3.8}, {96, 96, 2, 0.60, 0.375, 4.3}};
// Y = q X + S X (us, 128x256 / 128 / 64 / 32): 64 x 9000 9.5 / 6.5 / 4.8 / 5.0, 192 x 576 13.4 / 8.4 / 5.0 / 4.3, 512 x 2304 (4)
// 25.7 / 30.0 / 24.6 / 32.0, 1024 x 9216 (4) 232 / 265 / 330 / 573, 1470 x 4096 52 / 59 / 70 / 153, 4096 x 50,176 3869 / 4547 /
// 7632 / 13944 (256x128: 4078); written over X in split form 1024 x 9216 (4) 310 / 298 / 385 / 615.
constexpr TileKind kApplyTiles[TILE_KINDS] = {
    {128, 256, 1, 1.18, 0.0, 4.0}, {128, 128, 1, 0.69, 0.0, 4.3}, {64, 64, 2, 0.25, 0.18, 4.3}, {32, 32, 5, 0.10, 0.13, 3.8}};

// us for `wgs` workgroups of `blocks` blocks each: their rounds, or what they take in at 14 TB/s (the caches: 1056 workgroups of 64 over
// 64 blocks 79.5 us, 1128 over 94 138, 2080 over 128 340)
double tile_time(const TileKind& k, int64_t wgs, int64_t blocks) {
    const int64_t at_once = 256 * (int64_t)k.per_cu;
    const int64_t together = wgs >= at_once ? k.per_cu : (wgs + 255) / 256;
    const double rounds = (double)((wgs + at_once - 1) / at_once) * ((double)blocks * (k.block + k.more * (double)(together - 1)) + k.start);
    const double intake = (double)(wgs * blocks) * (double)((k.bm + k.bn) * TILE_BLOCK_BYTES) / 14e6;
    return rounds > intake ? rounds : intake;
}

// powers of two the split matrices are held at: A, R and T up to 120, S up to 1022 (steps_in_groups)
constexpr float kScaleA = 512.0f, kScaleR = 512.0f, kScaleS = 64.0f;

NsShape shape_of(int64_t rows, int64_t cols, int count) {
    NsShape s = {};
    s.rows = rows;
    s.cols = cols;
    s.tall = rows > cols;
    s.l = s.tall ? cols : rows;
    s.n = s.tall ? rows : cols;
    s.lk = (s.l + 31) & ~31ll;
    s.nk = (s.n + 31) & ~31ll;
    s.lh = (s.l + 63) & ~63ll;
    s.nh = (s.n + 63) & ~63ll;
    s.count = count;
    return s;
}

int check_sizes(int64_t count, int64_t rows, int64_t cols) {
    if (count < 0 || count > 65535 || rows < 1 || cols < 1) return YH_ERR_SHAPE;
    const int64_t l = rows < cols ? rows : cols, n = rows < cols ? cols : rows;
    if (l > kMaxShort || n > kMaxLong || l * n > kMaxNumbers) return YH_ERR_SHAPE;
    // workgroups of a launch (256 threads each; a grid holds fewer than 2^32 threads)
    if (count > kMaxNumbers / (l * n) || (count < 1 ? 1 : count) * ((l + 31) / 32) * ((n + 31) / 32) >= ((int64_t)1 << 24))
        return YH_ERR_SHAPE;
    return YH_OK;
}

struct Layout {
    size_t parts, factor, hop, x, xt, xt2, a, r0, r1, t, s0, s1, partial, total;      // the planes of S go where xt2 would be
    long long x_mat, xt_mat, sq_mat;
    int norm_blocks;
    bool half;
    int gram, tiles, slices, per_slice;      // X X': kind of tile, tiles on and below the diagonal, slices
    int square, square_tiles;                // an l x l product by itself
    int shared, shared_tiles, shares;        // and with a share of S: of how many
};

inline int triangle_tiles(int64_t l, int b) {
    const int64_t side = (l + b - 1) / b;
    return (int)(side * (side + 1) / 2);
}

// half: X in fp16 alone
Layout layout_for(const NsShape& s, bool half) {
    Layout w = {};
    w.half = half;
    int64_t nb = (s.rows * s.cols + 4095) / 4096;
    w.norm_blocks = (int)(nb < 1 ? 1 : nb > NS_NORM_BLOCKS ? NS_NORM_BLOCKS : nb);
    w.x_mat = half ? s.l * s.nh * 2 : s.l * s.nk * 4;
    w.xt_mat = half ? s.n * s.lh * 2 : s.n * s.lk * 4;
    w.sq_mat = s.l * s.lk * 4;
    // the contraction of X X' is cut when the tiles alone do not fill the card
    const int64_t blocks = half ? s.nh / 64 : s.nk / 32;
    double best = 0.0, best_square = 0.0, best_shared = 0.0;
    for (int k = 0; k < PRODUCT_KINDS; ++k) {
        const int t = triangle_tiles(s.l, kTiles[k].bm);
        const int64_t wgs = (int64_t)t * s.count;
        for (int cut = 1; cut <= 16 && cut * 4 <= blocks + 3; ++cut) {
            if (cut > 1 && wgs * cut > 4096) break;
            const int64_t per = (blocks + cut - 1) / cut;
            double us = tile_time(kTiles[k], wgs * cut, per);
            if (cut > 1) us += 4.0 + (double)(wgs * (cut + 1)) * kTiles[k].bm * kTiles[k].bm * 4.0 / 3e6;
            if (best == 0.0 || us < best) {
                best = us;
                w.gram = k;
                w.tiles = t;
                w.per_slice = (int)per;
                w.slices = (int)((blocks + per - 1) / per);
            }
        }
        const double us = tile_time(kTiles[k], wgs, s.lk / 32);
        if (best_square == 0.0 || us < best_square) {
            best_square = us;
            w.square = k;
            w.square_tiles = t;
        }
    }
    // S of a step is not needed before the next step's: it goes along with T alone, or in shares with T, the next A and the next R,
    // so that a launch fills the card without beginning another round (a call in us, with T alone / as chosen: 1470x4096 440 / 425,
    // 1024x1024 225 / 205, four of them 497 / 447, 2048x2048 754 / 700, 3000x5000 2380 / 2007, 512x512 115 / 116)
    for (int k = 0; k < PRODUCT_KINDS; ++k) {
        const int t = triangle_tiles(s.l, kTiles[k].bm);
        for (int shares = 1; shares <= 3; ++shares) {
            const double us = shares * tile_time(kTiles[k], (int64_t)(t + (t + shares - 1) / shares) * s.count, s.lk / 32) +
                              (3 - shares) * best_square;
            if (best_shared == 0.0 || us < best_shared) {
                best_shared = us;
                w.shared = k;
                w.shared_tiles = t;
                w.shares = shares;
            }
        }
    }
    size_t off = 0;
    auto take = [&](size_t bytes) { const size_t at = off; off += up256(bytes); return at; };
    w.parts = take((size_t)s.count * w.norm_blocks * 8);
    w.factor = take((size_t)s.count * NS_MAX_GROUPS * 4);
    w.hop = take((size_t)s.count * NS_MAX_GROUPS * 4);
    w.x = take((size_t)s.count * w.x_mat);
    w.xt = take((size_t)s.count * w.xt_mat);
    w.xt2 = take((size_t)s.count * (half ? s.l * s.lh * 4 : w.xt_mat));
    w.a = take((size_t)s.count * w.sq_mat);
    w.r0 = take((size_t)s.count * w.sq_mat);
    w.r1 = take((size_t)s.count * w.sq_mat);
    w.t = take((size_t)s.count * w.sq_mat);
    w.s0 = take((size_t)s.count * w.sq_mat);
    w.s1 = take((size_t)s.count * w.sq_mat);
    w.partial = take(w.slices > 1 ? (size_t)w.slices * w.tiles * s.count * kTiles[w.gram].bm * kTiles[w.gram].bm * 4 : 0);
    w.total = off;
    return w;
}

// where the result goes
struct Sink {
    int dtype;
    void* out;
    int64_t out_b, out_r;
    void* const* params;
    float decay, step;
};

template <int DT, int OUT, bool TALL, bool HALF, int BM, int BN, int WM, int WN, int STAGES>
void apply_tiles(const NsApply& a, hipStream_t st) {
    const int64_t tiles = ((a.sh.l + BM - 1) / BM) * ((a.sh.n + BN - 1) / BN) * a.sh.count;
    hipLaunchKernelGGL((ns_apply_kernel<DT, OUT, TALL, HALF, BM, BN, WM, WN, STAGES>), dim3((unsigned)tiles), dim3(64 * WM * WN), 0, st, a);
}

template <int DT, int OUT, bool TALL, bool HALF = false>
int apply(const NsApply& a, hipStream_t st) {
    int kind = 0;
    double best = 0.0;
    for (int k = 0; k < TILE_KINDS; ++k) {
        const TileKind& t = kApplyTiles[k];
        const int64_t wgs = ((a.sh.l + t.bm - 1) / t.bm) * ((a.sh.n + t.bn - 1) / t.bn) * a.sh.count;
        const double us = tile_time(t, wgs, a.sh.lk / 32);
        if (best == 0.0 || us < best) {
            best = us;
            kind = k;
        }
    }
    if (kind == TILE_LARGE) apply_tiles<DT, OUT, TALL, HALF, 128, 256, 2, 4, 3>(a, st);
    else if (kind == TILE_128) apply_tiles<DT, OUT, TALL, HALF, 128, 128, 2, 4, 4>(a, st);
    else if (kind == TILE_64) apply_tiles<DT, OUT, TALL, HALF, 64, 64, 2, 2, 4>(a, st);
    else apply_tiles<DT, OUT, TALL, HALF, 32, 32, 2, 2, 4>(a, st);
    return launch_status();
}

template <int OUT>
int apply_as(int dt, bool tall, const NsApply& a, hipStream_t st) {
    if (dt == YH_F32) return tall ? apply<DT_F32, OUT, true>(a, st) : apply<DT_F32, OUT, false>(a, st);
    if (dt == YH_F16) return tall ? apply<DT_F16, OUT, true>(a, st) : apply<DT_F16, OUT, false>(a, st);
    return tall ? apply<DT_BF16, OUT, true>(a, st) : apply<DT_BF16, OUT, false>(a, st);
}

// X in fp16 alone serves 16-bit results
int apply_half(int dt, bool tall, const NsApply& a, hipStream_t st) {
    if (dt == YH_F16) return tall ? apply<DT_F16, NS_OUT_RESULT, true, true>(a, st) : apply<DT_F16, NS_OUT_RESULT, false, true>(a, st);
    return tall ? apply<DT_BF16, NS_OUT_RESULT, true, true>(a, st) : apply<DT_BF16, NS_OUT_RESULT, false, true>(a, st);
}

template <class Math, int BM, int WM, int WN, int STAGES>
int products_of(const NsProducts& a, hipStream_t st) {
    const unsigned grid = (unsigned)(((int64_t)a.job[0].tiles * a.slices + a.job[1].tiles) * a.count);
    hipLaunchKernelGGL((ns_product_kernel<Math, BM, WM, WN, STAGES>), dim3(grid), dim3(64 * WM * WN), 0, st, a);
    if (const int rc = launch_status()) return rc;
    if (a.slices > 1)
        hipLaunchKernelGGL((ns_join_kernel<BM, WM, WN, STAGES>), dim3((unsigned)(a.job[0].tiles * a.count)), dim3(64 * WM * WN), 0, st, a);
    return launch_status();
}

template <class Math>
int products_in(int kind, const NsProducts& a, hipStream_t st) {
    if (kind == TILE_LARGE) return products_of<Math, 192, 2, 4, 3>(a, st);
    if (kind == TILE_128) return products_of<Math, 128, 2, 4, 4>(a, st);
    if (kind == TILE_96) return products_of<Math, 96, 2, 2, 3>(a, st);
    if (kind == TILE_64) return products_of<Math, 64, 2, 2, 4>(a, st);
    return products_of<Math, 32, 2, 2, 4>(a, st);
}

constexpr int kChainSide = 128;     // A up to this size is worked on by one workgroup

int chain(const NsChain& c, int count, hipStream_t st) {
    const dim3 grid((unsigned)count);
    if (c.l <= 32) hipLaunchKernelGGL((ns_chain_kernel<32, 1>), grid, dim3(ChainGrid<32, 1>::THREADS), 0, st, c);
    else if (c.l <= 64) hipLaunchKernelGGL((ns_chain_kernel<64, 1>), grid, dim3(ChainGrid<64, 1>::THREADS), 0, st, c);
    else if (c.l <= 96) hipLaunchKernelGGL((ns_chain_kernel<96, 2>), grid, dim3(ChainGrid<96, 2>::THREADS), 0, st, c);
    else hipLaunchKernelGGL((ns_chain_kernel<128, 2>), grid, dim3(ChainGrid<128, 2>::THREADS), 0, st, c);
    return launch_status();
}

template <int DT, bool LIST>
int load(const NsSource& src, const NsShape& s, const Layout& w, char* ws, double eps, const NsHold& hold, hipStream_t st) {
    bool on16 = LIST || (aligned(src.base, 16) && src.stride_r % 8 == 0 && src.stride_b % 8 == 0);
    if (LIST)
        for (int i = 0; i < s.count; ++i) on16 = on16 && aligned(src.g[i], 16) && aligned(src.buf[i], 16);
    const int vec = on16 && s.cols % 8 == 0;
    hipLaunchKernelGGL((ns_norm_kernel<DT, LIST>), dim3((unsigned)w.norm_blocks, (unsigned)s.count), dim3(256), 0, st, src, s,
                       (double*)(ws + w.parts), vec && (LIST || src.stride_r == s.cols));
    if (const int rc = launch_status()) return rc;
    char* x = ws + w.x;
    char* xt = ws + w.xt;
    const dim3 grid((unsigned)(((s.cols + 63) / 64) * ((s.rows + 63) / 64)), (unsigned)s.count);
    auto convert = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, src, s, (const double*)(ws + w.parts), w.norm_blocks, eps, hold,
                           s.tall ? xt : x, s.tall ? w.xt_mat : w.x_mat, s.tall ? x : xt, s.tall ? w.x_mat : w.xt_mat,
                           (float*)(ws + w.factor), (float*)(ws + w.hop), vec);
    };
    if constexpr (!LIST && DT != DT_F32) {
        if (w.half) {
            convert(ns_convert_kernel<DT, LIST, true>);
            return launch_status();
        }
    }
    convert(ns_convert_kernel<DT, LIST, false>);
    return launch_status();
}

template <bool LIST>
int load_as(int dt, const NsSource& src, const NsShape& s, const Layout& w, char* ws, double eps, const NsHold& hold, hipStream_t st) {
    if (dt == YH_F32) return load<DT_F32, LIST>(src, s, w, ws, eps, hold, st);
    if (dt == YH_F16) return load<DT_F16, LIST>(src, s, w, ws, eps, hold, st);
    return load<DT_BF16, LIST>(src, s, w, ws, eps, hold, st);
}

// The steps in groups, each on one X X'.  A singular value s of X becomes s (a + b s^2 + c s^4): from all of [0, 1] that gives
// the largest one before every step, and the largest factor of every step.  A group ends where the product of its factors
// would pass 64, or 511 for bf16 results (S within its range): the error of one X X' for five steps, 8e-4 at most, is
// below bf16's own rounding (1.7e-3) but not fp16's (2.1e-4).
struct Steps {
    NsHold hold;
    int len[NS_MAX_GROUPS];
};
constexpr double kMostA = 120.0;     // of A, R and T: fp16 at their scales ends at 127

// the power of two above x
inline short above(double x) { return (short)(x > 1e-30 ? ilogb(x) + 1 : -99); }

// false: coefficients and steps whose matrices would leave fp16's range
bool steps_in_groups(double a, double b, double c, int steps, int out_dtype, double scale, Steps& p) {
    const double limit = out_dtype == YH_BF16 ? 511.0 : 64.0;
    double top = 1.0, growth = 1.0, within = 1.0;
    bool full = true;
    p.hold.groups = 0;
    p.hold.scale = scale;
    for (int j = 0; j < steps; ++j) {
        const double most = top * top;                               // of A
        double r = fabs(b * most + c * most * most);                 // of |R|, and of |a + R|
        double factor = fmax(fabs(a), fabs(a + b * most + c * most * most));
        const double z = c != 0.0 ? -b / (2.0 * c) : -1.0;
        if (z > 0.0 && z < most) {
            r = fmax(r, fabs(b * z / 2.0));
            factor = fmax(factor, fabs(a + b * z / 2.0));
        }
        if (!(most <= kMostA && r <= kMostA && factor * most <= kMostA)) return false;
        if (full || within * factor > limit) {
            p.hold.growth[p.hold.groups] = above(growth);
            p.hold.top[p.hold.groups] = above(top);
            p.len[p.hold.groups++] = 0;
            within = 1.0;
        }
        within *= factor;
        growth *= factor;
        full = within > limit;
        ++p.len[p.hold.groups - 1];
        // the largest s (a + b s^2 + c s^4): at the end or where a + 3 b z + 5 c z^2 = 0 (z = s^2)
        auto at = [&](double x) { return x > 0.0 && x <= most ? sqrt(x) * fabs(a + b * x + c * x * x) : 0.0; };
        double next = at(most);
        if (c != 0.0) {
            const double d = 9.0 * b * b - 20.0 * a * c;
            if (d >= 0.0) next = fmax(next, fmax(at((-3.0 * b + sqrt(d)) / (10.0 * c)), at((-3.0 * b - sqrt(d)) / (10.0 * c))));
        } else if (b != 0.0) next = fmax(next, at(-a / (3.0 * b)));
        top = next;
    }
    return true;
}

// X in fp16 alone: 16-bit numbers, all steps on one X X', and enough of them to pay for the launch that lays S out in
// planes (a call in us with bf16 results, split / half: 192x576 85.6 / 90.1, 512x512 113 / 117, 256x4096 104.5 / 102.3, 512x2304 129 / 127,
// 4x512x2304 202 / 195, 1470x4096 475 / 443, 4x1024x9216 897 / 740, 4096x50,176 9520 / 7210)
bool half_for(const NsShape& s, int g_dtype, int out_dtype, const Steps& plan) {
    return g_dtype != YH_F32 && out_dtype != YH_F32 && s.l > 128 && plan.hold.groups == 1 &&
           (double)s.l * (double)s.n * s.count >= 1e6;
}

// G is in the workspace as X and X', factors beside them; the steps, and the result to `sink`
int run_steps(const NsShape& s, const Layout& w, char* ws, float a, float b, float c, const Steps& plan, const Sink& sink,
              hipStream_t st) {
    char *A = ws + w.a, *T = ws + w.t, *R[2] = {ws + w.r0, ws + w.r1}, *S[2] = {ws + w.s0, ws + w.s1};
    char *X = ws + w.x, *Xt = ws + w.xt, *Xt_next = ws + w.xt2;
    const int lb = (int)(s.lk / 32);
    NsProducts base = {};
    base.l = s.l;
    base.lk = s.lk;
    base.count = s.count;
    base.slices = 1;
    base.per_slice = lb;
    auto job = [&](const char* P, const char* Q, char* out, float k0, const char* E1, float k1, const char* E2, float k2) {
        NsProduct p = {};
        p.P = P;
        p.Q = Q;
        p.E1 = E1;
        p.E2 = E2;
        p.out = out;
        p.p_mat = p.out_mat = w.sq_mat;
        p.ldp = s.lk * 4;
        p.k0 = k0;
        p.k1 = k1;
        p.k2 = k2;
        p.blocks = lb;
        return p;
    };
    for (int group = 0; group < plan.hold.groups; ++group) {
        const int len = plan.len[group];
        const bool last_group = group + 1 == plan.hold.groups;
        const float* factor = (const float*)(ws + w.factor) + (size_t)group * s.count;
        // A = X X'
        NsProducts gram = base;
        gram.slices = w.slices;
        gram.per_slice = w.per_slice;
        gram.partial = (float*)(ws + w.partial);
        gram.job[0] = job(X, X, A, kScaleA, nullptr, 0.0f, nullptr, 0.0f);
        gram.job[0].factor = factor;
        gram.job[0].tiles = w.tiles;
        gram.job[0].p_mat = w.x_mat;
        gram.job[0].ldp = w.half ? s.nh * 2 : s.nk * 4;
        gram.job[0].blocks = (int)(gram.job[0].ldp / TILE_BLOCK_BYTES);
        if (const int rc = w.half ? products_in<MathHalf>(w.gram, gram, st) : products_in<MathSplit>(w.gram, gram, st)) return rc;
        double q = a;                          // Q = q + S
        const char* Q = nullptr;
        float sq = 0.0f;
        if (s.l <= kChainSide) {
            NsChain ch = {};
            ch.A = A;
            ch.S = S[0];
            ch.mat = w.sq_mat;
            ch.l = s.l;
            ch.lk = s.lk;
            ch.a = a;
            ch.b = b;
            ch.c = c;
            ch.steps = len;
            ch.scale_a = kScaleA;
            ch.scale_r = kScaleR;
            ch.scale_s = kScaleS;
            if (const int rc = chain(ch, s.count, st)) return rc;
            for (int j = 1; j < len; ++j) q *= a;
            Q = S[0];
            sq = len == 1 ? kScaleR : kScaleS;
        } else {
            NsProduct waiting = {};            // S of this step, not needed before the next one's
            int left = 0;
            auto launch = [&](const NsProduct& p) {
                NsProducts both = base;
                both.job[0] = p;
                both.job[0].tiles = left ? w.shared_tiles : w.square_tiles;
                if (!left) return products_in<MathSplit>(w.square, both, st);
                const int64_t share = w.shares - left--;
                both.job[1] = waiting;
                both.job[1].first = (int)(w.shared_tiles * share / w.shares);
                both.job[1].tiles = (int)(w.shared_tiles * (share + 1) / w.shares) - both.job[1].first;
                return products_in<MathSplit>(w.shared, both, st);
            };
            for (int j = 0; j < len; ++j) {
                char* Rj = j == 0 ? S[0] : R[j & 1];      // S_0 = R_0; neither is written while S of the step before is under way
                const bool last = j + 1 == len;
                if (const int rc = launch(job(A, A, Rj, c * kScaleR / (kScaleA * kScaleA), A, b * kScaleR / kScaleA, nullptr, 0.0f))) return rc;
                NsProduct next = {};
                if (j > 0) {
                    next = job(Rj, Q, S[j & 1], kScaleS / (kScaleR * sq), Q, a * kScaleS / sq, Rj, (float)(q * kScaleS / kScaleR));
                    q *= a;
                    Q = S[j & 1];
                    sq = kScaleS;
                } else {
                    Q = Rj;
                    sq = kScaleR;
                }
                if (last) {
                    if (j > 0)
                        if (const int rc = launch(next)) return rc;
                    break;
                }
                if (j > 0) {
                    waiting = next;
                    left = w.shares;
                }
                if (const int rc = launch(job(Rj, A, T, 1.0f / kScaleR, A, a, nullptr, 0.0f))) return rc;
                if (const int rc = launch(job(T, Rj, A, 1.0f / kScaleR, T, a, nullptr, 0.0f))) return rc;
            }
        }
        NsApply ap = {};
        ap.S = Q;
        ap.X = X;
        ap.Xt = Xt;
        ap.s_mat = w.sq_mat;
        ap.x_mat = w.x_mat;
        ap.xt_mat = w.xt_mat;
        ap.sh = s;
        ap.factor = last_group ? factor : (const float*)(ws + w.hop) + (size_t)(group + 1) * s.count;
        ap.k0 = (float)(1.0 / sq);
        ap.k1 = (float)q;
        if (!last_group) {
            ap.Yn = X;
            ap.Yt = Xt_next;
            if (const int rc = apply<DT_F32, NS_OUT_SPLIT, false>(ap, st)) return rc;
            char* swap = Xt;
            Xt = Xt_next;
            Xt_next = swap;
        } else if (sink.params) {
            bool on16 = (s.cols * (int64_t)dtype_bytes(sink.dtype)) % 16 == 0;
            for (int i = 0; i < s.count; ++i) {
                ap.param[i] = sink.params[i];
                on16 = on16 && aligned(sink.params[i], 16);
            }
            ap.store = on16 ? STORE_16 : STORE_ONE;
            ap.decay = sink.decay;
            ap.step = sink.step;
            if (const int rc = apply_as<NS_OUT_WEIGHT>(sink.dtype, s.tall, ap, st)) return rc;
        } else {
            ap.out = sink.out;
            ap.out_b = sink.out_b;
            ap.out_r = sink.out_r;
            const size_t e = dtype_bytes(sink.dtype);
            if (aligned(sink.out, 16) && (sink.out_r * e) % 16 == 0 && (sink.out_b * e) % 16 == 0) ap.store = STORE_16;
            else if (aligned(sink.out, 2 * e) && sink.out_r % 2 == 0 && sink.out_b % 2 == 0) ap.store = STORE_PAIR;
            else ap.store = STORE_ONE;
            if (w.half) {
                hipLaunchKernelGGL(ns_planes_kernel, dim3((unsigned)((s.l * s.lh / 8 + 1023) / 1024), (unsigned)s.count), dim3(256), 0, st, Q,
                                   w.sq_mat, Xt_next, (long long)(s.l * s.lh * 4), s);
                if (const int rc = launch_status()) return rc;
                ap.S = Xt_next;
                ap.s_mat = s.l * s.lh * 4;
                if (const int rc = apply_half(sink.dtype, s.tall, ap, st)) return rc;
            } else if (const int rc = apply_as<NS_OUT_RESULT>(sink.dtype, s.tall, ap, st)) return rc;
        }
    }
    return YH_OK;
}

// X_0 is held at about unit mean square, a spike in it still below fp16's largest number
double first_scale(const NsShape& s) {
    int e = (int)floor(0.5 * log2((double)s.rows * (double)s.cols));
    if (e > 15) e = 15;
    return ldexp(1.0, e);
}

bool known(int dt) { return dt == YH_F32 || dt == YH_F16 || dt == YH_BF16; }

}  // namespace

extern "C" {

size_t yh_orthogonalize_workspace_bytes(int64_t count, int64_t rows, int64_t cols) {
    if (check_sizes(count, rows, cols) != YH_OK || count == 0) return 0;
    const NsShape s = shape_of(rows, cols, (int)count);
    const size_t split = layout_for(s, false).total, half = layout_for(s, true).total;
    return split > half ? split : half;
}

int yh_orthogonalize(const void* g, int g_dtype, int64_t g_stride, int64_t ldg, void* out, int out_dtype, int64_t out_stride,
                     int64_t ldo, int64_t count, int64_t rows, int64_t cols, float a, float b, float c, int steps, float eps,
                     void* workspace, size_t workspace_bytes, void* stream) {
    if (const int rc = check_sizes(count, rows, cols)) return rc;
    if (ldg < cols || ldo < cols || (count > 1 && out_stride < (rows - 1) * ldo + cols)) return YH_ERR_SHAPE;
    if (!known(g_dtype) || !known(out_dtype)) return YH_ERR_ARG;
    if (!isfinite(a) || !isfinite(b) || !isfinite(c) || steps < 1 || steps > YH_MAX_NS_STEPS || !(eps >= 0.0f) || isinf(eps))
        return YH_ERR_ARG;
    if (count == 0) return YH_OK;
    if (!g || !out) return YH_ERR_NULL;
    const NsShape s = shape_of(rows, cols, (int)count);
    if (!workspace || workspace_bytes < yh_orthogonalize_workspace_bytes(count, rows, cols)) return YH_ERR_WORKSPACE;
    if (!aligned(g, dtype_bytes(g_dtype)) || !aligned(out, dtype_bytes(out_dtype)) || !aligned(workspace, 256)) return YH_ERR_ALIGN;
    Steps plan;
    if (!steps_in_groups(a, b, c, steps, out_dtype, first_scale(s), plan)) return YH_ERR_ARG;
    const Layout w = layout_for(s, half_for(s, g_dtype, out_dtype, plan));
    hipStream_t st = (hipStream_t)stream;
    char* ws = (char*)workspace;
    NsSource src = {};
    src.base = g;
    src.stride_b = g_stride;
    src.stride_r = ldg;
    if (const int rc = load_as<false>(g_dtype, src, s, w, ws, eps, plan.hold, st)) return rc;
    Sink sink = {};
    sink.dtype = out_dtype;
    sink.out = out;
    sink.out_b = out_stride;
    sink.out_r = ldo;
    return run_steps(s, w, ws, a, b, c, plan, sink, st);
}

int yh_muon_step(void* const* params, int p_dtype, const void* const* grads, int g_dtype, float* const* momenta, int count,
                 int64_t rows, int64_t cols, float lr, float momentum, int nesterov, float weight_decay, float scale, float a,
                 float b, float c, int steps, float eps, void* workspace, size_t workspace_bytes, void* stream) {
    if (count < 0 || count > YH_MUON_MAX_COUNT) return YH_ERR_SHAPE;
    if (const int rc = check_sizes(count, rows, cols)) return rc;
    if (!known(p_dtype) || !known(g_dtype)) return YH_ERR_ARG;
    if (!isfinite(lr) || !isfinite(momentum) || !isfinite(weight_decay) || !isfinite(scale) || !isfinite(a) || !isfinite(b) ||
        !isfinite(c) || steps < 1 || steps > YH_MAX_NS_STEPS || !(eps >= 0.0f) || isinf(eps))
        return YH_ERR_ARG;
    if (count == 0) return YH_OK;
    if (!params || !grads || !momenta) return YH_ERR_NULL;
    NsSource src = {};
    for (int i = 0; i < count; ++i) {
        if (!params[i] || !grads[i] || !momenta[i]) return YH_ERR_NULL;
        if (!aligned(params[i], dtype_bytes(p_dtype)) || !aligned(grads[i], dtype_bytes(g_dtype)) || !aligned(momenta[i], 4))
            return YH_ERR_ALIGN;
        src.g[i] = grads[i];
        src.buf[i] = momenta[i];
    }
    const NsShape s = shape_of(rows, cols, count);
    if (!workspace || workspace_bytes < yh_orthogonalize_workspace_bytes(count, rows, cols)) return YH_ERR_WORKSPACE;
    if (!aligned(workspace, 256)) return YH_ERR_ALIGN;
    Steps plan;
    if (!steps_in_groups(a, b, c, steps, p_dtype, first_scale(s), plan)) return YH_ERR_ARG;
    const Layout w = layout_for(s, false);
    src.momentum = momentum;
    src.nesterov = nesterov != 0;
    hipStream_t st = (hipStream_t)stream;
    char* ws = (char*)workspace;
    if (const int rc = load_as<true>(g_dtype, src, s, w, ws, eps, plan.hold, st)) return rc;
    Sink sink = {};
    sink.dtype = p_dtype;
    sink.params = params;
    sink.decay = (float)(1.0 - (double)lr * (double)weight_decay);
    sink.step = (float)((double)lr * (double)scale);
    return run_steps(s, w, ws, a, b, c, plan, sink, st);
}

}  // extern "C"
