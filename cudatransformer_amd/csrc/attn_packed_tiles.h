// Tile machinery of the packed-sequence attention kernels: the formats (bf16, fp16 on the 32x32x16
// MFMA, fp32 on the 32x32x2 one) behind one interface, and strided global -> LDS tile loads.
//
// A tile is row-major with RB bytes per row, its 16-byte chunks XOR-swizzled by the row as in
// attn_bf16_tiles.h (Tile<RB / 2>).  Row operands: step s of a lane (row, half) is the chunk
// 2 s + half of its row, 8 elements of 16 bits (one MFMA, contraction of 16) or 4 of 32 bits (four
// MFMAs with a contraction of 2 each).  Both operands of a product read the same chunks, so the
// order of the contraction does not matter.  Column operands: the contraction runs over tile rows
// in the order in which an accumulator holds them (register 8 kk + e, lane half: row acc_row(8 kk
// + e, half)), so that P and dS go from accumulators into the next product as they stand.
#pragma once

#include "attn_bf16_tiles.h"

#include <type_traits>

namespace ctattn {
namespace packedtile {

using namespace bf16tile;

// 8 accumulator registers as the B operand of a contraction over 16 rows.
typedef float f32x8 __attribute__((ext_vector_type(8)));

template <typename H> struct Fmt16 : H {
    static constexpr int ES = 2;
    static constexpr bool RANGE = std::is_same_v<H, F16Fmt>;  // narrower in exponent than fp32
    using vec = typename H::vec;  // a 16-byte chunk
    using pvec = vec;             // 8 values as a B operand
    using store = uint16_t;
    __device__ static __forceinline__ floatx16 mma(vec a, vec b, floatx16 c) { return H::mfma(a, b, c); }
    __device__ static __forceinline__ void put(pvec &p, int e, float x) { p[e] = (typename H::elem)x; }
    // What a lane adds to a tile's address for column operands (cb0, cb1).
    template <int RB> __device__ static __forceinline__ uint32_t col0(int lane) { return col_base<RB / 2>(0, 0, 0, lane); }
    template <int RB> __device__ static __forceinline__ uint32_t col1(int lane) { return col_base<RB / 2>(0, 0, 1, lane); }
    struct cols {
        vec v;
    };
    template <int RB> __device__ static __forceinline__ cols read_cols(uint32_t c0, uint32_t c1, int kk, int dt) {
        return {read_col<RB / 2, vec>(c0, c1, kk, dt)};
    }
    __device__ static __forceinline__ floatx16 col_mma(const cols &a, pvec p, floatx16 c) { return H::mfma(a.v, p, c); }
};
using PBf16 = Fmt16<Bf16Fmt>;
using PF16 = Fmt16<F16Fmt>;

struct PF32 {
    static constexpr int ES = 4;
    static constexpr bool RANGE = false;
    using vec = floatx4;
    using pvec = f32x8;
    using store = float;
    __device__ static __forceinline__ floatx16 mma(vec a, vec b, floatx16 c) {
#pragma unroll
        for (int e = 0; e < 4; ++e) c = mfma32x32x2(a[e], b[e], c);
        return c;
    }
    __device__ static __forceinline__ void put(pvec &p, int e, float x) { p[e] = x; }
    __device__ static float widen(float x) { return x; }
    // Lane (col, half): element col of the d tile in rows acc_row(r, half).  The row's swizzle is
    // that of acc_row(r, 0) with its lowest bit flipped by half (rows 4 apart).
    template <int RB> __device__ static __forceinline__ uint32_t col0(int lane) {
        const int col = lane & 31, half = lane >> 5;
        return uint32_t(4 * half * RB + ((((col >> 2) ^ half) << 4) | ((col & 3) << 2)));
    }
    template <int RB> __device__ static __forceinline__ uint32_t col1(int) { return 0; }
    struct cols {
        float v[8];
    };
    template <int RB> __device__ static __forceinline__ cols read_cols(uint32_t c0, uint32_t, int kk, int dt) {
        cols x;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int row = acc_row(8 * kk + e, 0);
            const uint32_t flip = uint32_t((Tile<RB / 2>::swz(row) ^ (8 * dt)) << 4);
            x.v[e] = *(__attribute__((address_space(3))) const float *)(uintptr_t)((c0 ^ flip) + uint32_t(row * RB));
        }
        return x;
    }
    __device__ static __forceinline__ floatx16 col_mma(const cols &a, pvec p, floatx16 c) {
#pragma unroll
        for (int e = 0; e < 8; ++e) c = mfma32x32x2(a.v[e], p[e], c);
        return c;
    }
};

// Stores 4 fp32 values as 4 consecutive elements.
template <typename F> __device__ __forceinline__ void store4(typename F::store *p, const float (&x)[4]) {
    if constexpr (F::ES == 2) {
        u16x4 y;
#pragma unroll
        for (int t = 0; t < 4; ++t) y[t] = F::bits(x[t]);
        *reinterpret_cast<u16x4 *>(p) = y;
    } else {
        *reinterpret_cast<floatx4 *>(p) = floatx4{x[0], x[1], x[2], x[3]};
    }
}

// One 16-byte chunk per lane, global -> LDS, at LDS address dst + 16 lane (dst wave-uniform).  Invisible to
// the compiler, as load_tile_dma: the kernel awaits it (wait_loads) before the barrier.
__device__ __forceinline__ void load_chunk_dma(const void *g, uint32_t dst) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(g),
                 "s"(__builtin_amdgcn_readfirstlane(dst))
                 : "memory", "m0");
}

// ROWS rows of a [tokens, heads, d] tensor's head into a swizzled tile: `block` is the first row,
// `stride` the bytes from row to row, `width` the bytes of a row's d elements (a multiple of 16).  Rows
// at or past `rows` re-read the last one (their results are masked), chunks past `width` are zeros.
template <int RB, int ROWS, int NW, bool PAD>
__device__ __forceinline__ void load_rows(uint32_t tile, const char *block, int64_t stride, int width, int rows,
                                          int wave, int lane) {
    using L = Tile<RB / 2>;
    constexpr int TOTAL = ROWS * L::CH;
    constexpr int NL = (TOTAL + NW * kWave - 1) / (NW * kWave);
    static_assert(TOTAL % kWave == 0, "tile size");
#pragma unroll
    for (int i = 0; i < NL; ++i) {
        const int P = (wave * NL + i) * kWave + lane;
        if (TOTAL % (NW * kWave) == 0 || (wave * NL + i) * kWave < TOTAL) {
            const int r = P / L::CH;
            const int c = 16 * ((P % L::CH) ^ L::swz(r));
            const char *g = block + min(r, rows - 1) * stride + c;
            if (PAD && c >= width) g = reinterpret_cast<const char *>(tile_zeros);
            load_chunk_dma(g, tile + uint32_t((wave * NL + i) * kWave * 16));
        }
    }
}

}  // namespace packedtile
}  // namespace ctattn
