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
// normalised: |X|, |A| and |B| stay below 255.9, and lo is a normal number down to x = 2^-10 (an entry of X is
// about 1 / sqrt(c)); below that a factor is off by 2^-33 at most, whatever x.  One fp16 term alone would not
// do: five steps amplify a direction by up to a^5 = 485, and its rounding with it.
//
// Layout: a factor's 128 x 32 blocks lie one behind the other, each a run of 128 rows [32 hi | 32 lo] (128 bytes
// a row, 16 KiB), so that one K step of a tile is one contiguous read.  A product's 32 x 32
// block is then a run of 4 KiB as well.  Rows and columns are padded with zeros to 128 and no product checks a bound.
// X is kept transposed alone: X^T's rows are what B X contracts over, and A = X X^T, which contracts over
// its columns, reads them through transposing LDS reads (ds_read_b64_tr_b16).  Keeping X as well made B X write
// twice: 24 x 384 x 384 290 us, bf16 4096 x 1024 398, 2048 x 8192 1.96 ms for five steps.
//
// Measured: r 2048, c 8192: B X 171 us (1.2 PFLOP/s of fp16 MFMA, matrix cores 58 % busy), A 108 + 14 to join its splits (46 %),
// A A 51 (136 tiles on 256 CUs).  24 matrices of 384 x 384: 15 to 18 us a product, 7.5 of it 12 K steps, the rest a
// launch's first loads and last stores.
#include "attn_bf16_tiles.h"
#include "attn_launch.h"
#include "capi_util.h"
#include "ctattn.h"

#include <algorithm>
#include <exception>
#include <type_traits>
#include <vector>

namespace ctattn {
namespace {

using namespace bf16tile;

constexpr float kScale = 256.f;   // of every stored factor
constexpr int kPad = 128;         // rows and columns are padded to it
constexpr int kGroup = 32;        // elements of a [hi | lo] group
constexpr int kRowBytes = 128;    // bytes of a group: one K step of a row
constexpr int kMaxMats = 64;      // matrices of a launch
constexpr int kNormBlocks = 1024;  // partial sums of squares per matrix at most

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

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

// hi and lo of 4 values that hold 256 x.
struct Four {
    u16x4 hi, lo;
};
__device__ __forceinline__ Four split4(f32x4 x) {
    const f16x4 hi = __builtin_convertvector(x, f16x4);
    const f32x4 back = __builtin_convertvector(hi, f32x4);
    const f16x4 lo = __builtin_convertvector(x - back, f16x4);
    return {__builtin_bit_cast(u16x4, hi), __builtin_bit_cast(u16x4, lo)};
}
__device__ __forceinline__ f32x4 join4(u16x4 hi, u16x4 lo) {
    return __builtin_convertvector(__builtin_bit_cast(f16x4, hi), f32x4) +
           __builtin_convertvector(__builtin_bit_cast(f16x4, lo), f32x4);
}

// A 32 x 32 block of a factor in LDS: 32 rows [32 hi | 32 lo], chunks of 16 bytes swizzled as in Tile<64>
// (4 KiB, on 1 KiB).  put4: elements c .. c + 3 (c a multiple of 4) of a row.
__device__ __forceinline__ void block_put4(uint32_t blk, int row, int c, const Four &v) {
    const uint32_t in = uint32_t(2 * (c & 4));
    *(__attribute__((address_space(3))) u16x4 *)(uintptr_t)(blk + uint32_t(Tile<64>::off(row, c >> 3)) + in) = v.hi;
    *(__attribute__((address_space(3))) u16x4 *)(uintptr_t)(blk + uint32_t(Tile<64>::off(row, 4 + (c >> 3))) + in) = v.lo;
}
__device__ __forceinline__ void lds_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
// The block to a factor's 4 KiB run, whole lines at a time (stores of 8 or 16 bytes a row, straight from registers, were
// bound by their number: 24 x 384 x 384 19 us a product for 16).
__device__ __forceinline__ void block_store(uint32_t blk, char *to, int lane) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = 8 * i + lane / 8, chunk = lane % 8;
        *reinterpret_cast<u16x8 *>(to + row * kRowBytes + 16 * chunk) = lds_b128<u16x8>(blk + uint32_t(Tile<64>::off(row, chunk)));
    }
}
// The block's transpose into another: ds_read_b64_tr_b16 gives lane l of a group of 16 column l of 4 rows, so
// two of them are 8 elements of one row of the transpose.
__device__ __forceinline__ void block_transpose(uint32_t blk, uint32_t into, int lane) {
    const int s = lane & 15, half = lane >> 5;
    const int chunk = 2 * ((lane >> 4) & 1) + ((s & 3) >> 1);
#pragma unroll
    for (int part = 0; part < 2; ++part)  // hi, lo
#pragma unroll
        for (int r0 = 0; r0 < 32; r0 += 16) {
            i16x4 x[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int row = r0 + 8 * half + 4 * u + (s >> 2);
                const uint32_t at = blk + uint32_t(Tile<64>::off(row, chunk + 4 * part) + 8 * (s & 1));
                x[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4 *)(uintptr_t)at);
            }
            const i16x8 y = {x[0][0], x[0][1], x[0][2], x[0][3], x[1][0], x[1][1], x[1][2], x[1][3]};
            *(__attribute__((address_space(3))) i16x8 *)(uintptr_t)(into + uint32_t(Tile<64>::off(lane & 31, 4 * part + r0 / 8 + half))) = y;
        }
}
// Byte offset of element (i, k)'s hi in a factor of `groups` K steps a row; lo is 64 bytes on.
__device__ __forceinline__ int64_t factor_at(uint32_t i, uint32_t k, int groups) {
    return int64_t((i / kPad) * uint32_t(groups) + k / kGroup) * (kPad * kRowBytes) + (i % kPad) * kRowBytes + (k % kGroup) * 2;
}

// ---- the update and its norm ----
// The update's element: G itself, or Muon's g + mu m (m = mu m + g already written; nesterov) or m.
template <typename T>
__device__ __forceinline__ float update_value(const Update &u, const T *g, const float *m, int64_t i) {
    if (!u.muon) return to_f32(g[i]);
    return u.nesterov ? fmaf(u.momentum, m[i], to_f32(g[i])) : m[i];
}

// Sums of squares in fp64 (fp32 squares would overflow from 1.8e19 on), up to kNormBlocks a matrix; the Muon
// step advances its moment here.  Runs of 16 bytes of G where its matrices lie on them.
template <typename T, int VEC>
__global__ __launch_bounds__(256) void norm_kernel(Mats g, Mats m, Update u, int64_t n, double *__restrict__ part) {
    struct alignas(sizeof(T) * VEC) Run {
        T v[VEC];
    };
    const int mat = blockIdx.y;
    const T *gp = g.at<const T>(mat);
    float *mp = u.muon ? m.at<float>(mat) : nullptr;
    double s = 0;
    for (int64_t i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; i < n / VEC; i += int64_t(gridDim.x) * blockDim.x) {
        const Run r = reinterpret_cast<const Run *>(gp)[i];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const int64_t at = i * VEC + e;
            float x = to_f32(r.v[e]);
            if (u.muon) {
                const float mv = fmaf(u.momentum, mp[at], x);
                mp[at] = mv;
                x = u.nesterov ? fmaf(u.momentum, mv, x) : mv;
            }
            s += double(x) * double(x);
        }
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

// X^T as a factor: a wave per 32 x 32 block of G, whose rows it reads 4 elements a lane, 8 lanes a row.  Of a tall G
// they are X^T's rows; of another they are transposed in LDS.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void split_kernel(Mats g, Mats m, Update u, Shape s, double eps,
                                                   const double *__restrict__ part, int blocks,
                                                   char *__restrict__ xt, int64_t bytes) {
    __shared__ __attribute__((aligned(1024))) char smem[4 * 8192];
    // 256 / (|G| + eps) = inv_s 2^exp_s: by itself it may lie outside fp32 where every 256 X is inside.
    __shared__ float inv_s;
    __shared__ int exp_s;
    __shared__ double sums[4];
    const int mat = blockIdx.z, lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    {
        double ss = 0;
        for (int i = threadIdx.x; i < blocks; i += 256) ss += part[int64_t(mat) * kNormBlocks + i];
        ss = wave_sum(ss);
        if (lane == 0) sums[wave] = ss;
        __syncthreads();
        if (threadIdx.x == 0) {
            const double x = double(kScale) / (sqrt((sums[0] + sums[1]) + (sums[2] + sums[3])) + eps);
            int e = 0;
            inv_s = x < double(INFINITY) ? float(frexp(x, &e)) : float(x);  // G = 0 without an eps: 0 times an infinity
            exp_s = e;
        }
    }
    __syncthreads();
    const float inv = inv_s;
    const int inv_e = exp_s;
    const T *gp = g.at<const T>(mat);
    const float *mp = u.muon ? m.at<const float>(mat) : nullptr;
    // G's padded shape; its row blocks in y, four column blocks a workgroup in x.
    const int gcols = int(s.tall ? s.rp : s.cp);
    const int j0 = (int(blockIdx.x) * 4 + wave) * 32, i0 = int(blockIdx.y) * 32;
    if (j0 >= gcols) return;
    char *to = xt + mat * bytes + (s.tall ? factor_at(i0, j0, int(s.rp) / kGroup) : factor_at(j0, i0, int(s.rp) / kGroup));
    const uint32_t blk = lds_addr(smem) + uint32_t(wave * 8192);
    struct alignas(sizeof(T) * 4) Run {
        T v[4];
    };
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int line = 8 * q + lane / 8, c = 4 * (lane % 8);
        const int64_t i = i0 + line, j = j0 + c, at = i * s.cols + j;
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        if (VEC && i < s.rows && j + 3 < s.cols) {
            const Run r = *reinterpret_cast<const Run *>(gp + at);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = u.muon ? update_value(u, gp, mp, at + e) : to_f32(r.v[e]);
        } else if (i < s.rows) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (j + e < s.cols) v[e] = update_value(u, gp, mp, at + e);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = ldexpf(v[e], inv_e) * inv;
        const Four f = split4(v);
        block_put4(blk, line, c, f);
    }
    lds_done();
    if (!s.tall) {
        block_transpose(blk, blk + 4096, lane);
        lds_done();
    }
    block_store(s.tall ? blk : blk + 4096, to, lane);
}

// ---- products ----
enum Product { kGram = 0, kPoly, kApply, kLast };

struct Gemm {
    const char *a, *b;           // factors with rows of kp elements; tile (ti, tj): rows of a, rows of b
    int64_t a_bytes, b_bytes;    // from matrix to matrix
    int64_t kp;
    int tiles_m, tiles_n;        // kGram, kPoly: tiles_m (tiles_m + 1) / 2 lower tiles
    int mats, splits;
    float *part;                 // splits > 1: a tile's sums for each split
    char *o;                     // the product as a factor (kApply: transposed)
    int64_t o_bytes;
    int o_groups;                // its K steps a row
    int a_groups;                // kGram: of a row of X^T
    const char *gram;            // kPoly: A, for b A
    float pa, pb, pc;
    Mats out;                    // kLast
    Update u;
    Shape s;
};

// Tile shapes of a product: BM x BN elements by WM x WN waves, K steps of 32 (rows of 128 bytes) through
// STAGES LDS buffers.  One workgroup fills a CU either way (128 KiB of LDS).
struct SmallTile {  // 8 waves of 64 x 32, two a SIMD: three steps of loads in flight
    static constexpr int BM = 128, WM = 2, WN = 4, STAGES = 4;
};
struct LargeTile {  // 8 waves of 128 x 64, two a SIMD: half the operand bytes per product
    static constexpr int BM = 256, WM = 2, WN = 4, STAGES = 2;
};
template <typename C> struct Tiling : C {
    static constexpr int WAVES = C::WM * C::WN;
    static constexpr int MT = C::BM / C::WM / 32, NT = C::BM / C::WN / 32;  // 32 x 32 blocks of a wave
    static constexpr int TB = C::BM * kRowBytes;                            // one operand's tile of a step
    static constexpr int LDS = 2 * C::STAGES * TB;
    static constexpr int NL = TB / (WAVES * kWave * 16);                    // loads of a lane per operand and step
    static constexpr int BLOCKS = (C::BM / 32) * (C::BM / 32);
    static constexpr int WPE = WAVES / 4;
};

__device__ __forceinline__ void lower_tile(int t, int &ti, int &tj) {
    ti = int((sqrtf(8.f * float(t) + 1.f) - 1.f) * 0.5f);
    while (ti * (ti + 1) / 2 > t) --ti;
    while ((ti + 1) * (ti + 2) / 2 <= t) ++ti;
    tj = t - ti * (ti + 1) / 2;
}

// What a 32 x 32 block of sums becomes, by one wave: register r of lane (col, half) is row acc_row(r, half),
// column col.  buf: LDS address of 8 KiB of the wave's own, on 1 KiB.  (i0, j0): the block's place in the
// product, multiples of 32, so that the block of a factor is a run of 4 KiB, 128 bytes a row.
constexpr int kBufBytes = 8192;
template <typename T, int P>
__device__ __forceinline__ void leave(const Gemm &g, int mat, const floatx16 &acc, int i0, int j0, bool mirror,
                                      uint32_t buf, int lane) {
    const int col = lane & 31, half = lane >> 5;
    if constexpr (P == kLast) {
        typedef __attribute__((address_space(3))) float lds_float;
        lds_float *f = (lds_float *)(uintptr_t)buf;
#pragma unroll
        for (int r = 0; r < 16; ++r) f[acc_row(r, half) * 33 + col] = acc[r] * (1.f / (kScale * kScale));
        lds_done();
        // Along the output's rows: X's row i0 + line, or for a tall matrix X's column j0 + line.
        const int64_t row0 = g.s.tall ? j0 : i0;
        const int64_t at = (g.s.tall ? i0 : j0) + col;
        T *to = g.out.at<T>(mat) + (row0 + half) * g.s.cols + at;
        const int step = g.s.tall ? 1 : 33, across = g.s.tall ? 33 : 1;
        if (at < g.s.cols) {
#pragma unroll
            for (int q = 0; q < 16; ++q, to += 2 * g.s.cols) {
                const int line = 2 * q + half;
                const float v = f[line * step + col * across];
                if (row0 + line < g.s.rows) *to = from_f32<T>(g.u.muon ? fmaf(-g.u.lr, v, g.u.keep * to_f32(*to)) : v);
            }
        }
        lds_done();
    } else {
        // The registers hold four elements of row j0 + col of the transpose at a time: that goes to LDS and out, and the
        // block as it is (symmetric products) is its transpose.
        const int64_t at = factor_at(j0, i0, g.o_groups) + mat * g.o_bytes;
        char *t = g.o + at;
        const char *A0 = P == kPoly ? g.gram + at + col * kRowBytes + 8 * half : nullptr;
        // a I on the diagonal of the rows that exist.
        const int diag = P == kPoly && i0 == j0 && i0 + col < g.s.r ? col - 4 * half : -1;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            f32x4 v = {acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
            v = v * (1.f / kScale);
            if constexpr (P == kPoly) {  // A is symmetric: its row j0 + col
                const f32x4 A = join4(*reinterpret_cast<const u16x4 *>(A0 + 16 * q), *reinterpret_cast<const u16x4 *>(A0 + 16 * q + 64));
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[e] = fmaf(g.pb, A[e], g.pc * v[e]);
                    if (8 * q + e == diag) v[e] += g.pa * kScale;
                }
            }
            block_put4(buf, col, 8 * q + 4 * half, split4(v));
        }
        lds_done();
        if (P == kApply || mirror) block_store(buf, t, lane);
        if constexpr (P != kApply) {
            block_transpose(buf, buf + 4096, lane);
            lds_done();
            block_store(buf + 4096, g.o + mat * g.o_bytes + factor_at(i0, j0, g.o_groups), lane);
        }
        lds_done();  // the next block's writes follow these reads
    }
}

// Work item: matrix, tile, split.  XCD x (workgroup b runs on XCD b % 8) takes contiguous items, which share
// operand rows in its L2.
__device__ __forceinline__ int64_t xcd_item(int64_t n) {
    const int64_t q = (n + 7) / 8;
    return (blockIdx.x % 8) * q + blockIdx.x / 8;
}

// A workgroup: one tile of a b^T over its split of K.  A step's operands are read into registers in two
// halves of 16 of the contraction, the second while the first is multiplied, and the next step's
// first half, after the barrier that publishes it, while the second is.
template <typename T, int P, typename TC>
__global__ __launch_bounds__(Tiling<TC>::WAVES *kWave) __attribute__((amdgpu_waves_per_eu(Tiling<TC>::WPE, Tiling<TC>::WPE)))
void product_kernel(Gemm g) {
    using C = Tiling<TC>;
    constexpr int MT = C::MT, NT = C::NT, TB = C::TB, NL = C::NL;
    __shared__ __attribute__((aligned(1024))) char smem[C::LDS];
    const uint32_t L = lds_addr(smem);
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int wm = wave / C::WN, wn = wave % C::WN, col = lane & 31, half = lane >> 5;
    constexpr bool SYM = P == kGram || P == kPoly;
    const int tiles = SYM ? g.tiles_m * (g.tiles_m + 1) / 2 : g.tiles_m * g.tiles_n;
    const int64_t item = xcd_item(int64_t(g.mats) * tiles * g.splits);
    if (item >= int64_t(g.mats) * tiles * g.splits) return;
    const int t = int(item % tiles), split_i = int(item / tiles % g.splits), mat = int(item / tiles / g.splits);
    int ti, tj;
    if (SYM) lower_tile(t, ti, tj);
    else ti = t % g.tiles_m, tj = t / g.tiles_m;

    constexpr int BLOCK = kPad * kRowBytes;
    const int steps_all = int(g.kp / kGroup);
    const int per = (steps_all + g.splits - 1) / g.splits;
    const int k0 = min(steps_all, split_i * per), k1 = min(steps_all, k0 + per);
    // A step's tile of an operand: BM rows of 128 bytes, or for kGram 32 rows of X^T in each of BM / 32 groups of
    // columns, 4 KiB a group.
    const int64_t panel = int64_t(P == kGram ? g.a_groups : steps_all) * BLOCK;  // 128 rows
    const int64_t tile_bytes = P == kGram ? C::BM / kGroup * int64_t(BLOCK) : C::BM / kPad * panel;
    const char *ga = g.a + mat * g.a_bytes + ti * tile_bytes;
    const char *gb = g.b + mat * g.b_bytes + tj * tile_bytes;
    auto step_at = [&](int k) __attribute__((always_inline)) {
        return P == kGram ? int64_t(k / 4) * panel + (k % 4) * (32 * kRowBytes) : int64_t(k) * BLOCK;
    };
    int64_t src[NL];  // this lane's 16-byte chunks of a step
#pragma unroll
    for (int i = 0; i < NL; ++i) {
        const int p = (wave * NL + i) * kWave + lane, row = p / 8;
        src[i] = (P == kGram ? int64_t(row / 32) * BLOCK + (row % 32) * kRowBytes : (row / kPad) * panel + (row % kPad) * kRowBytes) +
                 16 * ((p % 8) ^ Tile<64>::swz(row));
    }
    auto buffer = [&](int k) __attribute__((always_inline)) { return L + uint32_t((k - k0) % C::STAGES) * 2 * TB; };
    auto issue = [&](int k) __attribute__((always_inline)) {
        const uint32_t to = buffer(k);
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const uint32_t dst = to + uint32_t((wave * NL + i) * kWave * 16);
            const char *pa = ga + src[i] + step_at(k), *pb = gb + src[i] + step_at(k);
            asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(pa),
                         "s"(__builtin_amdgcn_readfirstlane(dst)) : "memory", "m0");
            asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(pb),
                         "s"(__builtin_amdgcn_readfirstlane(dst + TB)) : "memory", "m0");
        }
    };
    // Waits until step k's loads are in, given that later ones up to step `last` are under way.
    auto await = [&](int k, int last) __attribute__((always_inline)) {
        static_assert(2 * NL * 2 <= 63, "vmcnt");
        const int later = last - k;
        if (later <= 0) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        else if (later == 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * NL) : "memory");
        else asm volatile("s_waitcnt vmcnt(%0)" ::"n"(4 * NL) : "memory");
    };
    floatx16 acc[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[m][n] = zero16();
    const uint32_t ra = uint32_t(Tile<64>::off(32 * MT * wm + col, half)), rb = uint32_t(Tile<64>::off(32 * NT * wn + col, half)) + TB;
    struct Half {
        f16x8 ah[MT], al[MT], bh[NT], bl[NT];
    };
    const uint32_t cb0 = col_base<64>(0, 0, 0, lane), cb1 = col_base<64>(0, 0, 1, lane);
    auto read = [&](Half &x, int k, int s) __attribute__((always_inline)) {  // chunks 2 s + half of hi, 4 on of lo
        const uint32_t base = buffer(k);
        if constexpr (P == kGram) {  // columns of 16 rows: the same order of the contraction in both operands
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const uint32_t p = base + TB + uint32_t((NT * wn + n) * 32 * kRowBytes);
                x.bh[n] = read_col<64, f16x8>(p + cb0, p + cb1, s, 0);
                x.bl[n] = read_col<64, f16x8>(p + cb0, p + cb1, s, 1);
            }
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const uint32_t p = base + uint32_t((MT * wm + m) * 32 * kRowBytes);
                x.ah[m] = read_col<64, f16x8>(p + cb0, p + cb1, s, 0);
                x.al[m] = read_col<64, f16x8>(p + cb0, p + cb1, s, 1);
            }
            return;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const uint32_t p = base + rb + uint32_t(32 * n * kRowBytes);
            x.bh[n] = lds_b128<f16x8>(p ^ uint32_t(s << 5));
            x.bl[n] = lds_b128<f16x8>(p ^ uint32_t((s + 2) << 5));
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const uint32_t p = base + ra + uint32_t(32 * m * kRowBytes);
            x.ah[m] = lds_b128<f16x8>(p ^ uint32_t(s << 5));
            x.al[m] = lds_b128<f16x8>(p ^ uint32_t((s + 2) << 5));
        }
    };
    auto cross = [&](const Half &x) __attribute__((always_inline)) {  // lo hi
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[m][n] = F16Fmt::mfma(x.al[m], x.bh[n], acc[m][n]);
    };
    auto rest = [&](const Half &x) __attribute__((always_inline)) {  // hi lo, hi hi
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[m][n] = F16Fmt::mfma(x.ah[m], x.bl[n], acc[m][n]);
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[m][n] = F16Fmt::mfma(x.ah[m], x.bh[n], acc[m][n]);
    };
    // Keeps LDS reads and products in the order they are written in.
    auto keep_order = [&]() __attribute__((always_inline)) {
        asm volatile("" ::: "memory");
        read_fence();
    };
    if (k0 < k1) {
        int last = min(k1 - 1, k0 + C::STAGES - 2);  // the last step whose loads are under way
        for (int k = k0; k <= last; ++k) issue(k);
        await(k0, last);
        lds_barrier();
        if (last + 1 < k1) issue(++last);
        Half x, y;
        read(x, k0, 0);
        for (int k = k0; k < k1; ++k) {
            cross(x);
            keep_order();
            read(y, k, 1);
            keep_order();
            rest(x);
            keep_order();
            cross(y);
            keep_order();
            if (k + 1 < k1) {
                // Every wave has step k in registers: its buffer takes the next loads.
                await(k + 1, last);
                lds_barrier();
                if (last + 1 < k1) issue(++last);
                read(x, k + 1, 0);
            }
            keep_order();
            rest(y);
        }
    }
    if (g.splits > 1) {
        // This split's sums, in register order: the joining wave reads them back the same way.
        float *to = g.part + ((int64_t(mat) * tiles + t) * g.splits + split_i) * C::BM * C::BM + wave * (MT * NT * 1024);
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    *reinterpret_cast<floatx4 *>(to + (((m * NT + n) * 4 + q) * kWave + lane) * 4) =
                        floatx4{acc[m][n][4 * q], acc[m][n][4 * q + 1], acc[m][n][4 * q + 2], acc[m][n][4 * q + 3]};
        return;
    }
    lds_barrier();  // every wave is done with the tiles
    const uint32_t buf = L + uint32_t(wave * kBufBytes);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n)
            leave<T, P>(g, mat, acc[m][n], ti * C::BM + 32 * (MT * wm + m), tj * C::BM + 32 * (NT * wn + n),
                        SYM && ti != tj, buf, lane);
}

// Joins the splits' sums in order: one wave per 32 x 32 block of a tile.
template <typename T, int P, typename TC>
__global__ __launch_bounds__(256) void join_product_kernel(Gemm g) {
    using C = Tiling<TC>;
    constexpr bool SYM = P == kGram || P == kPoly;
    __shared__ __attribute__((aligned(1024))) char buf[4 * kBufBytes];
    const int lane = threadIdx.x & (kWave - 1);
    const int tiles = SYM ? g.tiles_m * (g.tiles_m + 1) / 2 : g.tiles_m * g.tiles_n;
    const int64_t w = int64_t(blockIdx.x) * 4 + threadIdx.x / kWave;
    const int t = int(w / C::BLOCKS % tiles), mat = int(w / C::BLOCKS / tiles), blk = int(w % C::BLOCKS);
    if (mat >= g.mats) return;
    int ti, tj;
    if (SYM) lower_tile(t, ti, tj);
    else ti = t % g.tiles_m, tj = t / g.tiles_m;
    const int wave = blk / (C::MT * C::NT), m = blk / C::NT % C::MT, n = blk % C::NT;
    floatx16 acc = zero16();
    const float *from = g.part + (int64_t(mat) * tiles + t) * g.splits * C::BM * C::BM + blk * 1024;
#pragma unroll 4
    for (int s = 0; s < g.splits; ++s)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const floatx4 x = *reinterpret_cast<const floatx4 *>(from + int64_t(s) * C::BM * C::BM + (q * kWave + lane) * 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[4 * q + e] += x[e];
        }
    leave<T, P>(g, mat, acc, ti * C::BM + 32 * (C::MT * (wave / C::WN) + m),
                tj * C::BM + 32 * (C::NT * (wave % C::WN) + n), SYM && ti != tj, lds_addr(buf) + uint32_t(threadIdx.x / kWave * kBufBytes), lane);
}

// ---- sizes and launches ----
struct Layout {
    Shape s;
    int64_t x_bytes, a_bytes;  // one factor X^T, one factor A
    int64_t off_norm, off_xt[2], off_a, off_b, off_part, bytes;
};

// How a product runs: the tile shape and the splits of K with the least estimated time, one workgroup a CU at a
// time on 256 CUs.  A step of a small tile takes 0.62 us, of a large one 2.5; a workgroup's start and end 12 or 13; joining
// costs a launch and the splits' sums there and back.
struct Choice {
    bool large;
    int splits;
};
Choice choose(bool sym, int64_t mats, int64_t m, int64_t n, int64_t kp) {
    Choice best{false, 1};
    double least = 1e30;
    for (int large = 0; large < 2; ++large) {
        const int64_t bm = large ? LargeTile::BM : SmallTile::BM;
        if (m % bm != 0 || n % bm != 0) continue;
        const int64_t tiles = mats * (sym ? (m / bm) * (m / bm + 1) / 2 : (m / bm) * (n / bm)), steps = kp / kGroup;
        for (int64_t s = 1; s <= 32 && s * 4 <= steps; ++s) {
            const double rounds = double((tiles * s + 255) / 256);
            double us = rounds * (double((steps + s - 1) / s) * (large ? 2.5 : 0.62) + (large ? 13 : 12));
            if (s > 1) us += 4 + double(tiles * s) * double(bm * bm) * 8 / 6e6;
            if (us < least) least = us, best = {large != 0, int(s)};
            if (tiles * s > 512) break;
        }
    }
    return best;
}

Layout layout(int64_t mats, int64_t rows, int64_t cols) {
    Layout l{};
    l.s.rows = rows;
    l.s.cols = cols;
    l.s.tall = rows > cols;
    l.s.r = std::min(rows, cols);
    l.s.c = std::max(rows, cols);
    // Sides from 1024 on to the large tile.
    auto pad = [](int64_t x) {
        const int64_t to = x >= 1024 ? LargeTile::BM : kPad;
        return (x + to - 1) / to * to;
    };
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
    l.off_xt[0] = take(mats * l.x_bytes);
    l.off_xt[1] = take(mats * l.x_bytes);
    l.off_a = take(mats * l.a_bytes);
    l.off_b = take(mats * l.a_bytes);
    auto part = [&](bool sym, int64_t n, int64_t kp) {
        const Choice ch = choose(sym, mats, l.s.rp, n, kp);
        const int64_t bm = ch.large ? LargeTile::BM : SmallTile::BM, tm = l.s.rp / bm;
        return ch.splits > 1 ? mats * (sym ? tm * (tm + 1) / 2 : tm * (n / bm)) * ch.splits * bm * bm * int64_t(4) : 0;
    };
    l.off_part = take(std::max({part(true, l.s.rp, l.s.cp), part(true, l.s.rp, l.s.rp), part(false, l.s.cp, l.s.rp)}));
    l.bytes = at;
    return l;
}

template <typename T, int P, typename TC> hipError_t run_product(const Gemm &g, int64_t tiles, hipStream_t st) {
    using C = Tiling<TC>;
    const int64_t groups = (tiles * g.splits + 7) / 8 * 8, joins = (tiles * C::BLOCKS + 3) / 4;
    if (!grid_fits(groups, C::WAVES * kWave) || !grid_fits(joins, 256)) return hipErrorInvalidValue;
    hipLaunchKernelGGL((product_kernel<T, P, TC>), dim3(unsigned(groups)), dim3(C::WAVES * kWave), 0, st, g);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || g.splits == 1) return e;
    hipLaunchKernelGGL((join_product_kernel<T, P, TC>), dim3(unsigned(joins)), dim3(256), 0, st, g);
    return hipGetLastError();
}

// a [m rows] b [n rows]^T.
template <typename T, int P> hipError_t product(Gemm g, int64_t m, int64_t n, hipStream_t st) {
    constexpr bool SYM = P == kGram || P == kPoly;
    const Choice ch = choose(SYM, g.mats, m, n, g.kp);
    const int64_t bm = ch.large ? LargeTile::BM : SmallTile::BM;
    g.splits = ch.splits;
    g.tiles_m = int(m / bm);
    g.tiles_n = int(n / bm);
    const int64_t tiles = int64_t(g.mats) * (SYM ? int64_t(g.tiles_m) * (g.tiles_m + 1) / 2 : int64_t(g.tiles_m) * g.tiles_n);
    return ch.large ? run_product<T, P, LargeTile>(g, tiles, st) : run_product<T, P, SmallTile>(g, tiles, st);
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
    const int blocks = int(std::max<int64_t>(1, std::min<int64_t>(kNormBlocks, n / 4096)));
    constexpr int V = 16 / int(sizeof(T));
    uintptr_t at = reinterpret_cast<uintptr_t>(x.g.base);
    if (!x.g.base)
        for (int i = 0; i < x.mats; ++i) at |= reinterpret_cast<uintptr_t>(x.g.p[i]);
    if (n % V == 0 && at % 16 == 0)
        hipLaunchKernelGGL((norm_kernel<T, V>), dim3(unsigned(blocks), unsigned(x.mats)), dim3(256), 0, st, x.g, x.m, x.u, n, norm);
    else
        hipLaunchKernelGGL((norm_kernel<T, 1>), dim3(unsigned(blocks), unsigned(x.mats)), dim3(256), 0, st, x.g, x.m, x.u, n, norm);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int64_t gr = l.s.tall ? l.s.cp : l.s.rp, gc = l.s.tall ? l.s.rp : l.s.cp;  // G's padded shape
    const dim3 grid(unsigned(gc / 128), unsigned(gr / 32), unsigned(x.mats));
    auto split_g = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, x.g, x.m, x.u, l.s, x.eps, norm, blocks,
                           ws + l.off_xt[0], l.x_bytes);
    };
    if (l.s.cols % 4 == 0 && at % 16 == 0) split_g(split_kernel<T, true>);
    else split_g(split_kernel<T, false>);
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
        g.a = g.b = xt;
        g.a_bytes = g.b_bytes = l.x_bytes;
        g.a_groups = int(l.s.rp / kGroup);
        g.kp = l.s.cp;
        g.o = ws + l.off_a;
        g.o_bytes = l.a_bytes;
        g.o_groups = int(l.s.rp / kGroup);
        if ((e = product<T, kGram>(g, l.s.rp, l.s.rp, st)) != hipSuccess) return e;
        g.a = g.b = g.gram = ws + l.off_a;
        g.a_bytes = g.b_bytes = l.a_bytes;
        g.kp = l.s.rp;
        g.o = ws + l.off_b;
        if ((e = product<T, kPoly>(g, l.s.rp, l.s.rp, st)) != hipSuccess) return e;
        g.a = ws + l.off_b;
        g.b = xt;
        g.b_bytes = l.x_bytes;
        g.o = ws + l.off_xt[(i + 1) % 2];
        g.o_bytes = l.x_bytes;
        g.o_groups = int(l.s.rp / kGroup);
        e = i + 1 == x.steps ? product<T, kLast>(g, l.s.rp, l.s.cp, st) : product<T, kApply>(g, l.s.rp, l.s.cp, st);
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

// Bytes for `count` matrices in batches of kMaxMats: the last, smaller batch may split its products more.
int64_t batches_bytes(int64_t count, int64_t rows, int64_t cols) {
    int64_t need = layout(std::min<int64_t>(count, kMaxMats), rows, cols).bytes;
    if (count > kMaxMats && count % kMaxMats != 0) need = std::max(need, layout(count % kMaxMats, rows, cols).bytes);
    return need;
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

// Refuses parameters or moments that share memory with any other tensor of the call.
int check_separate(const char *fn, int count, void *const *param, const void *const *grad, void *const *moment, int64_t n,
                   int64_t es) {
    struct Range {
        uintptr_t lo, hi;
        bool written;
    };
    try {
        std::vector<Range> all;
        all.reserve(3 * size_t(count));
        for (int i = 0; i < count; ++i) {
            const auto add = [&](const void *p, int64_t bytes, bool written) {
                const uintptr_t at = reinterpret_cast<uintptr_t>(p);
                all.push_back({at, at + uintptr_t(bytes), written});
            };
            add(param[i], n * es, true);
            add(grad[i], n * es, false);
            add(moment[i], n * 4, true);
        }
        std::sort(all.begin(), all.end(), [](const Range &a, const Range &b) { return a.lo < b.lo; });
        uintptr_t any = 0, written = 0;  // how far the ranges so far reach
        for (const Range &r : all) {
            if (r.lo < written || (r.written && r.lo < any))
                return fail(hipErrorInvalidValue, "%s: a parameter or moment shares memory with another tensor", fn);
            any = std::max(any, r.hi);
            if (r.written) written = std::max(written, r.hi);
        }
    } catch (const std::exception &) {
        return fail(hipErrorOutOfMemory, "%s: out of host memory", fn);
    }
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
    return count == 0 ? 0 : batches_bytes(count, rows, cols);
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
    if (int rc = check_separate(fn, count, param, grad, moment, rows * cols, dtype == CTATTN_F32 ? 4 : 2)) return rc;
    if (int rc = check_workspace(fn, workspace, workspace_bytes, batches_bytes(count, rows, cols))) return rc;
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
