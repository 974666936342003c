// Newton-Schulz orthogonalisation and the Muon step around it (entry points in include/ctattn.h).
//
//   X = G / (|G|_F + eps);   each step: A = X X^T, X <- a X + (b A + c A^2) X
//
// with X taken on its short side: r = min(rows, cols), c = max, X [r][c] (a tall G is worked on transposed).
// Every step is three products: A (symmetric: its lower tiles are computed and mirrored), B = a I + b A + c
// A A (likewise), X <- B X.
//
// Precision: an fp32 product on the fp32 matrix cores has a tenth of the 16-bit rate.  Here every factor
// is the sum of two fp16 numbers, hi = fp16(256 x) and lo = fp16(256 x - hi), 22 significant bits, and a
// product is hi hi + hi lo + lo hi in one fp32 accumulator: three 16-bit MFMAs, what is left out
// (lo lo) is 2^-22 of the product, below the fp32 sums' own rounding.  fp16's range is enough because X is
// normalised: |X|, |A| and |B| stay below 255.9, and 256 x keeps lo a normal number down to x of 2^-7
// of an entry's usual 1 / sqrt(c).  One fp16 term alone would not do: five steps amplify a
// direction by up to a^5 = 485, and its rounding with it.
//
// Layout: factors lie in rows of groups [32 hi | 32 lo] (128 bytes), so that one K step of a tile row is
// one 128-byte line; rows and columns are padded with zeros to 128 and no product checks a bound.
// X is kept in both orders (X for A, X^T for B X): each product's operands then have the contraction
// contiguous, and the writing product has the tile in registers in either order anyway.
#include "attn_bf16_tiles.h"
#include "attn_launch.h"
#include "capi_util.h"
#include "ctattn.h"

#include <algorithm>
#include <type_traits>

namespace ctattn {
namespace {

using namespace bf16tile;

constexpr float kScale = 256.f;   // of every stored factor
constexpr int kPad = 128;         // rows and columns are padded to it
constexpr int kGroup = 32;        // elements of a [hi | lo] group
constexpr int kRowBytes = 128;    // bytes of a group: one K step of a row
constexpr int kMaxMats = 64;      // matrices of a launch
constexpr int kNormBlocks = 64;   // partial sums of squares per matrix

// Matrices of one shape: in one buffer, `stride` elements apart, or by pointers.
struct Mats {
    void *base;
    int64_t stride;
    void *p[kMaxMats];
    template <typename T> __device__ T *at(int i) const {
        return base != nullptr ? static_cast<T *>(base) + i * stride : static_cast<T *>(p[i]);
    }
};

// How a product of the last step leaves: written as it is, or the step of an optimizer.
struct Update {
    int muon;                 // 0: out = X
    int nesterov;
    float momentum, keep, lr;  // p <- keep p - lr X
};

// hi and lo of 256 x.
__device__ __forceinline__ uint32_t split(float x) {
    const _Float16 hi = _Float16(x);
    const _Float16 lo = _Float16(x - float(hi));
    return uint32_t(__builtin_bit_cast(uint16_t, hi)) | uint32_t(__builtin_bit_cast(uint16_t, lo)) << 16;
}
__device__ __forceinline__ float joined(uint16_t hi, uint16_t lo) {
    return float(__builtin_bit_cast(_Float16, hi)) + float(__builtin_bit_cast(_Float16, lo));
}
// Byte offset of element (i, k)'s hi in a factor with `pitch` bytes a row; lo is 64 bytes on.
__device__ __forceinline__ int64_t factor_at(int64_t i, int64_t k, int64_t pitch) {
    return i * pitch + (k / kGroup) * kRowBytes + (k % kGroup) * 2;
}

// ---- the update and its norm ----
// The update's element: G itself, or Muon's g + mu m (m = mu m + g already written; nesterov) or m.
template <typename T>
__device__ __forceinline__ float update_value(const Update &u, const T *g, const float *m, int64_t i) {
    if (!u.muon) return to_f32(g[i]);
    return u.nesterov ? fmaf(u.momentum, m[i], to_f32(g[i])) : m[i];
}

// Sums of squares in fp64 (fp32 squares would overflow from 1.8e19 on), kNormBlocks a matrix; the Muon step
// advances its moment here.
template <typename T>
__global__ __launch_bounds__(256) void norm_kernel(Mats g, Mats m, Update u, int64_t n, double *__restrict__ part) {
    const int mat = blockIdx.y;
    const T *gp = g.at<const T>(mat);
    float *mp = u.muon ? m.at<float>(mat) : nullptr;
    double s = 0;
    for (int64_t i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; i < n; i += int64_t(gridDim.x) * blockDim.x) {
        if (u.muon) mp[i] = fmaf(u.momentum, mp[i], to_f32(gp[i]));
        const double x = update_value(u, gp, mp, i);
        s += x * x;
    }
    s = wave_sum(s);
    __shared__ double w[4];
    if (threadIdx.x % kWave == 0) w[threadIdx.x / kWave] = s;
    __syncthreads();
    if (threadIdx.x == 0) part[int64_t(mat) * kNormBlocks + blockIdx.x] = (w[0] + w[1]) + (w[2] + w[3]);
}

struct Shape {
    int64_t rows, cols;  // of G
    int64_t r, c;        // of X: r <= c
    int64_t rp, cp;      // padded
    int tall;            // X = G^T
};

// X and X^T as factors: one workgroup per 64 x 64 tile of X.
template <typename T>
__global__ __launch_bounds__(256) void split_kernel(Mats g, Mats m, Update u, Shape s, double eps,
                                                   const double *__restrict__ part, int blocks, char *__restrict__ x,
                                                   char *__restrict__ xt, int64_t bytes) {
    __shared__ uint32_t tile[64][65];
    __shared__ float inv_s;
    const int mat = blockIdx.z;
    if (threadIdx.x < kWave) {
        const double ss = wave_sum(int(threadIdx.x) < blocks ? part[int64_t(mat) * kNormBlocks + threadIdx.x] : 0.0);
        if (threadIdx.x == 0) inv_s = float(double(kScale) / (sqrt(ss) + eps));
    }
    __syncthreads();
    const float inv = inv_s;
    const T *gp = g.at<const T>(mat);
    const float *mp = u.muon ? m.at<const float>(mat) : nullptr;
    const int64_t i0 = int64_t(blockIdx.y) * 64, k0 = int64_t(blockIdx.x) * 64;  // row and column of X
    const int a = threadIdx.x % 64, b0 = threadIdx.x / 64;
    for (int b = b0; b < 64; b += 4) {
        const int i = s.tall ? a : b, k = s.tall ? b : a;  // along G's rows
        float v = 0.f;
        if (i0 + i < s.r && k0 + k < s.c)
            v = update_value(u, gp, mp, s.tall ? (k0 + k) * s.cols + i0 + i : (i0 + i) * s.cols + k0 + k) * inv;
        tile[i][k] = split(v);
    }
    __syncthreads();
    // Row `line` of the tile (of its transpose), 16 elements a thread: 32 bytes of hi, 32 of lo.
    const int line = threadIdx.x / 4, part16 = threadIdx.x % 4 * 16;
    for (int t = 0; t < 2; ++t) {
        u16x8 hi[2], lo[2];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const uint32_t w = t == 0 ? tile[line][part16 + e] : tile[part16 + e][line];
            hi[e / 8][e % 8] = uint16_t(w);
            lo[e / 8][e % 8] = uint16_t(w >> 16);
        }
        char *to = (t == 0 ? x : xt) + mat * bytes +
                   (t == 0 ? factor_at(i0 + line, k0 + part16, 4 * s.cp) : factor_at(k0 + line, i0 + part16, 4 * s.rp));
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            *reinterpret_cast<u16x8 *>(to + 16 * h) = hi[h];
            *reinterpret_cast<u16x8 *>(to + 64 + 16 * h) = lo[h];
        }
    }
}

// ---- products ----
enum Product { kGram = 0, kPoly, kApply, kLast };

struct Gemm {
    const char *a, *b;           // factors with rows of kp elements; tile (ti, tj): rows of a, rows of b
    int64_t a_bytes, b_bytes;    // from matrix to matrix
    int64_t kp;
    int tiles_m, tiles_n;        // kGram, kPoly: tiles_m (tiles_m + 1) / 2 lower tiles
    int mats, splits;
    float *part;                 // splits > 1: sums of a split's tiles, 128 x 128 each
    char *o, *ot;                // the product as a factor, and its transpose (kApply)
    int64_t o_bytes, o_pitch, ot_pitch;
    const char *gram;            // kPoly: A, for b A
    float pa, pb, pc;
    Mats out;                    // kLast
    Update u;
    Shape s;
};

constexpr int kTile = 128;

__device__ __forceinline__ void lower_tile(int t, int &ti, int &tj) {
    ti = int((sqrtf(8.f * float(t) + 1.f) - 1.f) * 0.5f);
    while (ti * (ti + 1) / 2 > t) --ti;
    while ((ti + 1) * (ti + 2) / 2 <= t) ++ti;
    tj = t - ti * (ti + 1) / 2;
}

// What a 32 x 32 block of sums becomes, by one wave.  sum(r): register r of lane (col, half) is row
// acc_row(r, half), column col.  buf: 32 x 33 words of the wave's own.  (i0, j0): the block's place in the product.
template <typename T, int P>
__device__ __forceinline__ void leave(const Gemm &g, int mat, const floatx16 &acc, int64_t i0, int64_t j0, bool mirror,
                                      uint32_t *buf, int lane) {
    const int col = lane & 31, half = lane >> 5;
    if constexpr (P == kLast) {
        float *f = reinterpret_cast<float *>(buf);
#pragma unroll
        for (int r = 0; r < 16; ++r) f[acc_row(r, half) * 33 + col] = acc[r] * (1.f / (kScale * kScale));
        __builtin_amdgcn_wave_barrier();
        T *out = g.out.at<T>(mat);
#pragma unroll
        for (int q = 0; q < 16; ++q) {
            const int line = 2 * q + half;
            // Along the output's rows: X's row i, or for a tall matrix X's column j.
            const int64_t i = g.s.tall ? i0 + col : i0 + line, j = g.s.tall ? j0 + line : j0 + col;
            const float v = g.s.tall ? f[col * 33 + line] : f[line * 33 + col];
            if (i < g.s.r && j < g.s.c) {
                T *to = out + (g.s.tall ? j * g.s.cols + i : i * g.s.cols + j);
                *to = from_f32<T>(g.u.muon ? fmaf(-g.u.lr, v, g.u.keep * to_f32(*to)) : v);
            }
        }
        __builtin_amdgcn_wave_barrier();
    } else {
        char *o = g.o + mat * g.o_bytes;
        uint32_t w[16];
        if constexpr (P == kPoly) {
            const char *A = g.gram + mat * g.o_bytes;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int64_t i = i0 + acc_row(r, half), j = j0 + col;
                const uint16_t *p = reinterpret_cast<const uint16_t *>(A + factor_at(i, j, g.o_pitch));
                float v = fmaf(g.pb, joined(p[0], p[32]), g.pc * (acc[r] * (1.f / kScale)));
                if (i == j && i < g.s.r) v += g.pa * kScale;
                w[r] = split(v);
            }
        } else {
#pragma unroll
            for (int r = 0; r < 16; ++r) w[r] = split(acc[r] * (1.f / kScale));
        }
        // Transposed, straight from the registers: 4 elements of row j0 + col.
        char *t = P == kApply ? g.ot + mat * g.o_bytes : o;
        const int64_t t_pitch = P == kApply ? g.ot_pitch : g.o_pitch;
        if (P == kApply || mirror) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                u16x4 hi, lo;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    hi[e] = uint16_t(w[4 * q + e]);
                    lo[e] = uint16_t(w[4 * q + e] >> 16);
                }
                char *to = t + factor_at(j0 + col, i0 + 8 * q + 4 * half, t_pitch);
                *reinterpret_cast<u16x4 *>(to) = hi;
                *reinterpret_cast<u16x4 *>(to + 64) = lo;
            }
        }
        // As it is, through LDS: 16 elements of a row a lane.
#pragma unroll
        for (int r = 0; r < 16; ++r) buf[acc_row(r, half) * 33 + col] = w[r];
        __builtin_amdgcn_wave_barrier();
        const int line = lane / 2, at = lane % 2 * 16;
        u16x8 hi[2], lo[2];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const uint32_t x = buf[line * 33 + at + e];
            hi[e / 8][e % 8] = uint16_t(x);
            lo[e / 8][e % 8] = uint16_t(x >> 16);
        }
        char *to = o + factor_at(i0 + line, j0 + at, g.o_pitch);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            *reinterpret_cast<u16x8 *>(to + 16 * h) = hi[h];
            *reinterpret_cast<u16x8 *>(to + 64 + 16 * h) = lo[h];
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// Work item: matrix, tile, split.  XCD x (workgroup b runs on XCD b % 8) takes contiguous items, which share
// operand rows in its L2.
__device__ __forceinline__ int64_t xcd_item(int64_t n) {
    const int64_t q = (n + 7) / 8;
    return (blockIdx.x % 8) * q + blockIdx.x / 8;
}

// A workgroup of 4 waves: a 128 x 128 tile of a b^T, wave (w / 2, w % 2) its 64 x 64 quarter, K in steps of
// 32 (rows of 128 bytes) through two LDS buffers.
template <typename T, int P>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void product_kernel(Gemm g) {
    constexpr int TB = kTile * kRowBytes;  // one operand's tile
    __shared__ __attribute__((aligned(1024))) char smem[4 * TB];
    const uint32_t L = lds_addr(smem);
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int wm = wave / 2, wn = wave % 2, col = lane & 31, half = lane >> 5;
    constexpr bool SYM = P == kGram || P == kPoly;
    const int tiles = SYM ? g.tiles_m * (g.tiles_m + 1) / 2 : g.tiles_m * g.tiles_n;
    const int64_t item = xcd_item(int64_t(g.mats) * tiles * g.splits);
    if (item >= int64_t(g.mats) * tiles * g.splits) return;
    const int split_i = int(item % g.splits);
    const int t = int(item / g.splits % tiles), mat = int(item / g.splits / tiles);
    int ti, tj;
    if (SYM) lower_tile(t, ti, tj);
    else ti = t % g.tiles_m, tj = t / g.tiles_m;

    const int64_t pitch = 4 * g.kp;
    const int steps_all = int(g.kp / kGroup);
    const int per = (steps_all + g.splits - 1) / g.splits;
    const int k0 = split_i * per, k1 = min(steps_all, k0 + per);
    const char *ga = g.a + mat * g.a_bytes + int64_t(ti) * kTile * pitch;
    const char *gb = g.b + mat * g.b_bytes + int64_t(tj) * kTile * pitch;
    // This lane's chunks: 4 of each operand's tile, rows 8 apart per wave load.
    constexpr int NL = TB / (4 * kWave * 16);
    int64_t src[NL];
#pragma unroll
    for (int i = 0; i < NL; ++i) {
        const int p = (wave * NL + i) * kWave + lane;
        src[i] = int64_t(p / 8) * pitch + 16 * ((p % 8) ^ Tile<64>::swz(p / 8));
    }
    auto issue = [&](int k) __attribute__((always_inline)) {
        const uint32_t to = L + uint32_t((k - k0) & 1) * 2 * TB;
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const uint32_t dst = to + uint32_t((wave * NL + i) * kWave * 16);
            const char *pa = ga + src[i] + int64_t(k) * kRowBytes, *pb = gb + src[i] + int64_t(k) * kRowBytes;
            asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(pa),
                         "s"(__builtin_amdgcn_readfirstlane(dst)) : "memory", "m0");
            asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(pb),
                         "s"(__builtin_amdgcn_readfirstlane(dst + TB)) : "memory", "m0");
        }
    };
    floatx16 acc[2][2];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int n = 0; n < 2; ++n) acc[m][n] = zero16();
    const uint32_t ra = uint32_t(Tile<64>::off(64 * wm + col, half)), rb = uint32_t(Tile<64>::off(64 * wn + col, half)) + TB;
    if (k0 < k1) issue(k0);
    for (int k = k0; k < k1; ++k) {
        wait_loads();
        lds_barrier();
        if (k + 1 < k1) issue(k + 1);
        const uint32_t base = L + uint32_t((k - k0) & 1) * 2 * TB;
#pragma unroll
        for (int s = 0; s < 2; ++s) {  // 16 of the contraction: chunks 2 s + half of hi, 4 more on of lo
            f16x8 ah[2], al[2], bh[2], bl[2];
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                const uint32_t pa = base + ra + uint32_t(32 * m * kRowBytes), pb = base + rb + uint32_t(32 * m * kRowBytes);
                ah[m] = lds_b128<f16x8>(pa ^ uint32_t(s << 5));
                al[m] = lds_b128<f16x8>(pa ^ uint32_t((s + 2) << 5));
                bh[m] = lds_b128<f16x8>(pb ^ uint32_t(s << 5));
                bl[m] = lds_b128<f16x8>(pb ^ uint32_t((s + 2) << 5));
            }
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    acc[m][n] = F16Fmt::mfma(al[m], bh[n], acc[m][n]);
                    acc[m][n] = F16Fmt::mfma(ah[m], bl[n], acc[m][n]);
                    acc[m][n] = F16Fmt::mfma(ah[m], bh[n], acc[m][n]);
                }
        }
    }
    if (g.splits > 1) {
        // This split's sums, in register order: the joining wave reads them back the same way.
        float *to = g.part + ((int64_t(mat) * tiles + t) * g.splits + split_i) * kTile * kTile + wave * 64 * 64;
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    *reinterpret_cast<floatx4 *>(to + (((m * 2 + n) * 4 + q) * kWave + lane) * 4) =
                        floatx4{acc[m][n][4 * q], acc[m][n][4 * q + 1], acc[m][n][4 * q + 2], acc[m][n][4 * q + 3]};
        return;
    }
    lds_barrier();  // every wave is done with the tiles
    uint32_t *buf = reinterpret_cast<uint32_t *>(smem) + wave * 32 * 33;
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int n = 0; n < 2; ++n)
            leave<T, P>(g, mat, acc[m][n], int64_t(ti) * kTile + 64 * wm + 32 * m, int64_t(tj) * kTile + 64 * wn + 32 * n,
                        SYM && ti != tj, buf, lane);
}

// Joins the splits' sums in order: one wave per 32 x 32 block of a tile.
template <typename T, int P>
__global__ __launch_bounds__(256) void join_product_kernel(Gemm g) {
    constexpr bool SYM = P == kGram || P == kPoly;
    __shared__ uint32_t buf[4][32 * 33];
    const int lane = threadIdx.x & (kWave - 1);
    const int tiles = SYM ? g.tiles_m * (g.tiles_m + 1) / 2 : g.tiles_m * g.tiles_n;
    const int64_t w = int64_t(blockIdx.x) * 4 + threadIdx.x / kWave;  // block 0 .. 15 of a tile
    const int t = int(w / 16 % tiles), mat = int(w / 16 / tiles), blk = int(w % 16);
    if (mat >= g.mats) return;
    int ti, tj;
    if (SYM) lower_tile(t, ti, tj);
    else ti = t % g.tiles_m, tj = t / g.tiles_m;
    const int wave = blk / 4, m = blk / 2 % 2, n = blk % 2;
    floatx16 acc = zero16();
    const float *from = g.part + (int64_t(mat) * tiles + t) * g.splits * kTile * kTile + wave * 64 * 64;
    for (int s = 0; s < g.splits; ++s, from += kTile * kTile)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const floatx4 x = *reinterpret_cast<const floatx4 *>(from + (((m * 2 + n) * 4 + q) * kWave + lane) * 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[4 * q + e] += x[e];
        }
    leave<T, P>(g, mat, acc, int64_t(ti) * kTile + 64 * (wave / 2) + 32 * m, int64_t(tj) * kTile + 64 * (wave % 2) + 32 * n,
                SYM && ti != tj, buf[threadIdx.x / kWave], lane);
}

// ---- sizes and launches ----
struct Layout {
    Shape s;
    int64_t x_bytes, a_bytes;  // one factor X (or X^T), one factor A
    int64_t off_norm, off_x, off_xt[2], off_a, off_b, off_part, bytes;
};

// Workgroups that a launch should have at least; K steps that a split should keep.
constexpr int kWantGroups = 512;
constexpr int kMinSteps = 8;

int splits_of(int64_t tiles, int64_t kp) {
    const int64_t steps = kp / kGroup;
    int64_t s = kWantGroups / std::max<int64_t>(tiles, 1);
    s = std::min(s, steps / kMinSteps);
    return int(std::max<int64_t>(1, std::min<int64_t>(s, 32)));
}

Layout layout(int64_t mats, int64_t rows, int64_t cols) {
    Layout l{};
    l.s.rows = rows;
    l.s.cols = cols;
    l.s.tall = rows > cols;
    l.s.r = std::min(rows, cols);
    l.s.c = std::max(rows, cols);
    auto pad = [](int64_t x) { return (x + kPad - 1) / kPad * kPad; };
    l.s.rp = pad(l.s.r);
    l.s.cp = pad(l.s.c);
    l.x_bytes = l.s.rp * l.s.cp * 4;
    l.a_bytes = l.s.rp * l.s.rp * 4;
    int64_t at = 0;
    auto take = [&](int64_t b) {
        const int64_t o = at;
        at += capi::align_up(b);
        return o;
    };
    l.off_norm = take(mats * kNormBlocks * 8);
    l.off_x = take(mats * l.x_bytes);
    l.off_xt[0] = take(mats * l.x_bytes);
    l.off_xt[1] = take(mats * l.x_bytes);
    l.off_a = take(mats * l.a_bytes);
    l.off_b = take(mats * l.a_bytes);
    const int64_t tm = l.s.rp / kTile, tn = l.s.cp / kTile, sym = mats * (tm * (tm + 1) / 2), full = mats * tm * tn;
    auto part = [&](int64_t tiles, int64_t kp) {
        const int s = splits_of(tiles, kp);
        return s > 1 ? tiles * s * kTile * kTile * int64_t(4) : 0;
    };
    l.off_part = take(std::max({part(sym, l.s.cp), part(sym, l.s.rp), part(full, l.s.rp)}));
    l.bytes = at;
    return l;
}

template <typename T, int P> hipError_t product(Gemm g, hipStream_t st) {
    constexpr bool SYM = P == kGram || P == kPoly;
    const int64_t tiles = int64_t(g.mats) * (SYM ? g.tiles_m * (g.tiles_m + 1) / 2 : g.tiles_m * g.tiles_n);
    g.splits = splits_of(tiles, g.kp);
    const int64_t groups = (tiles * g.splits + 7) / 8 * 8;
    if (!grid_fits(groups, 256) || !grid_fits(tiles * 4, 256)) return hipErrorInvalidValue;
    hipLaunchKernelGGL((product_kernel<T, P>), dim3(unsigned(groups)), dim3(256), 0, st, g);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || g.splits == 1) return e;
    hipLaunchKernelGGL((join_product_kernel<T, P>), dim3(unsigned(tiles * 4)), dim3(256), 0, st, g);
    return hipGetLastError();
}

struct Args {
    Mats g, m, out;
    Update u;
    int mats, steps;
    double a, b, c, eps;
};

template <typename T> hipError_t orthogonalise(const Args &x, const Layout &l, char *ws, hipStream_t st) {
    double *norm = reinterpret_cast<double *>(ws + l.off_norm);
    const int64_t n = l.s.rows * l.s.cols;
    const int blocks = int(std::min<int64_t>(kNormBlocks, (n + 1023) / 1024));
    hipLaunchKernelGGL(norm_kernel<T>, dim3(unsigned(blocks), unsigned(x.mats)), dim3(256), 0, st, x.g, x.m, x.u, n, norm);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(split_kernel<T>, dim3(unsigned(l.s.cp / 64), unsigned(l.s.rp / 64), unsigned(x.mats)), dim3(256), 0,
                       st, x.g, x.m, x.u, l.s, x.eps, norm, blocks, ws + l.off_x, ws + l.off_xt[0], l.x_bytes);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    Gemm g{};
    g.mats = x.mats;
    g.s = l.s;
    g.part = reinterpret_cast<float *>(ws + l.off_part);
    g.pa = float(x.a);
    g.pb = float(x.b);
    g.pc = float(x.c);
    g.out = x.out;
    g.u = x.u;
    for (int i = 0; i < x.steps; ++i) {
        const char *xt = ws + l.off_xt[i % 2];
        g.a = g.b = ws + l.off_x;
        g.a_bytes = g.b_bytes = l.x_bytes;
        g.kp = l.s.cp;
        g.tiles_m = g.tiles_n = int(l.s.rp / kTile);
        g.o = ws + l.off_a;
        g.o_bytes = l.a_bytes;
        g.o_pitch = 4 * l.s.rp;
        if ((e = product<T, kGram>(g, st)) != hipSuccess) return e;
        g.a = g.b = g.gram = ws + l.off_a;
        g.a_bytes = g.b_bytes = l.a_bytes;
        g.kp = l.s.rp;
        g.o = ws + l.off_b;
        if ((e = product<T, kPoly>(g, st)) != hipSuccess) return e;
        g.a = ws + l.off_b;
        g.b = xt;
        g.b_bytes = l.x_bytes;
        g.tiles_n = int(l.s.cp / kTile);
        g.o = ws + l.off_x;
        g.ot = ws + l.off_xt[(i + 1) % 2];
        g.o_bytes = l.x_bytes;
        g.o_pitch = 4 * l.s.cp;
        g.ot_pitch = 4 * l.s.rp;
        e = i + 1 == x.steps ? product<T, kLast>(g, st) : product<T, kApply>(g, st);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

hipError_t typed(int dtype, const Args &x, const Layout &l, char *ws, hipStream_t st) {
    switch (dtype) {
        case CTATTN_F32: return orthogonalise<float>(x, l, ws, st);
        case CTATTN_BF16: return orthogonalise<bf16_t>(x, l, ws, st);
        default: return orthogonalise<f16_t>(x, l, ws, st);
    }
}

using capi::fail;

int check(const char *fn, int dtype, int64_t mats, int64_t rows, int64_t cols, int steps, double a, double b, double c,
          double eps) {
    if (dtype == CTATTN_F64) return fail(hipErrorNotSupported, "%s: f64 is not supported", fn);
    if (dtype != CTATTN_F32 && dtype != CTATTN_BF16 && dtype != CTATTN_F16)
        return fail(hipErrorInvalidValue, "%s: unknown dtype %d (0 = f32, 1 = bf16, 2 = f16)", fn, dtype);
    if (mats < 0 || rows < 1 || cols < 1 || mats > 65535 || rows > (1 << 20) || cols > (1 << 20) ||
        double(std::max<int64_t>(mats, 1)) * double(rows + kPad) * double(cols + kPad) > double(int64_t(1) << 36))
        return fail(hipErrorInvalidValue, "%s: invalid sizes %lld x [%lld, %lld]", fn, (long long)mats, (long long)rows,
                    (long long)cols);
    if (steps < 1 || steps > 100) return fail(hipErrorInvalidValue, "%s: %d steps (1 to 100)", fn, steps);
    // Factors are held as fp16 of 256 times their value.  |X| starts at 1 at most; with these bounds the common
    // coefficients stay far inside, and others that make the iteration grow end in infinities.
    if (!(std::abs(a) <= 64 && std::abs(b) <= 64 && std::abs(c) <= 64))
        return fail(hipErrorInvalidValue, "%s: coefficients above 64 (%g, %g, %g)", fn, a, b, c);
    if (!(eps >= 0) || !(eps <= 1e30)) return fail(hipErrorInvalidValue, "%s: eps %g", fn, eps);
    return 0;
}

int check_workspace(const char *fn, const void *ws, int64_t bytes, int64_t need) {
    if (!ws || bytes < need)
        return fail(hipErrorInvalidValue, "%s: workspace too small (%lld bytes, %lld needed)", fn, (long long)bytes,
                    (long long)need);
    if (reinterpret_cast<uintptr_t>(ws) % 256 != 0)
        return fail(hipErrorInvalidValue, "%s: workspace must be 256-byte aligned", fn);
    return 0;
}

}  // namespace
}  // namespace ctattn

using namespace ctattn;
using ctattn::capi::finish;
using ctattn::capi::ok;

extern "C" {

int64_t ctattn_newton_schulz_workspace_bytes(int dtype, int64_t mats, int64_t rows, int64_t cols) {
    if (check("ctattn_newton_schulz_workspace_bytes", dtype, mats, rows, cols, 1, 0, 0, 0, 0) != 0) return -1;
    return mats == 0 ? 0 : layout(mats, rows, cols).bytes;
}

int ctattn_newton_schulz(int dtype, const void *x, void *out, void *workspace, int64_t workspace_bytes, int64_t mats,
                         int64_t rows, int64_t cols, int steps, double a, double b, double c, double eps, void *stream) {
    const char *fn = "ctattn_newton_schulz";
    if (int rc = check(fn, dtype, mats, rows, cols, steps, a, b, c, eps)) return rc;
    if (mats == 0) return ok();
    if (!x || !out) return fail(hipErrorInvalidValue, "%s: null pointer", fn);
    const Layout l = layout(mats, rows, cols);
    if (int rc = check_workspace(fn, workspace, workspace_bytes, l.bytes)) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    Args y{};
    y.g.base = const_cast<void *>(x);
    y.out.base = out;
    y.g.stride = y.out.stride = rows * cols;
    y.mats = int(mats);
    y.steps = steps;
    y.a = a;
    y.b = b;
    y.c = c;
    y.eps = eps;
    return finish(fn, typed(dtype, y, l, static_cast<char *>(workspace), st), st);
}

int64_t ctattn_muon_update_workspace_bytes(int dtype, int64_t count, int64_t rows, int64_t cols) {
    if (check("ctattn_muon_update_workspace_bytes", dtype, count, rows, cols, 1, 0, 0, 0, 0) != 0) return -1;
    return count == 0 ? 0 : layout(std::min<int64_t>(count, kMaxMats), rows, cols).bytes;
}

int ctattn_muon_update_multi(int dtype, int count, void *const *param, const void *const *grad, void *const *moment,
                             void *workspace, int64_t workspace_bytes, int64_t rows, int64_t cols, double lr,
                             double momentum, int nesterov, double weight_decay, double scale, int steps, double a,
                             double b, double c, double eps, void *stream) {
    const char *fn = "ctattn_muon_update_multi";
    if (int rc = check(fn, dtype, count, rows, cols, steps, a, b, c, eps)) return rc;
    if (count == 0) return ok();
    if (!param || !grad || !moment) return fail(hipErrorInvalidValue, "%s: null pointer table", fn);
    for (int i = 0; i < count; ++i)
        if (!param[i] || !grad[i] || !moment[i]) return fail(hipErrorInvalidValue, "%s: null pointer in matrix %d", fn, i);
    if (int rc = check_workspace(fn, workspace, workspace_bytes, layout(std::min(count, kMaxMats), rows, cols).bytes)) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    for (int i0 = 0; i0 < count; i0 += kMaxMats) {
        Args y{};
        y.mats = std::min(count - i0, kMaxMats);
        for (int i = 0; i < y.mats; ++i) {
            y.g.p[i] = const_cast<void *>(grad[i0 + i]);
            y.m.p[i] = moment[i0 + i];
            y.out.p[i] = param[i0 + i];
        }
        y.u = {1, nesterov != 0, float(momentum), float(1.0 - lr * weight_decay), float(lr * scale)};
        y.steps = steps;
        y.a = a;
        y.b = b;
        y.c = c;
        y.eps = eps;
        const hipError_t e = typed(dtype, y, layout(y.mats, rows, cols), static_cast<char *>(workspace), st);
        if (e != hipSuccess) return finish(fn, e, st);
    }
    return finish(fn, hipSuccess, st);
}

}  // extern "C"
