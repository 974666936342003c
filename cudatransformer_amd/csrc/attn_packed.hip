// Attention on packed sequences with shared key heads on MFMA: bf16 and fp16 (32x32x16), fp32
// (32x32x2), fp32 accumulation, head dims that are whole 16-byte chunks up to 128.
//
// Forward: O = softmax(Q K^T / sqrt(d)) V within each sequence, L = log of the row's sum.  A
// workgroup of 4 waves owns 128 rows of (token, head of the group) of one key head, wave w rows
// 32 w .., and walks the sequence's keys in blocks of 64 through LDS (direct global -> LDS loads,
// two buffers); or 32 rows, of whose keys each wave walks a quarter.  Scores are computed
// transposed, S^T = K Q^T, so that a lane holds one row: the running maximum and sum of the
// softmax need one exchange with lane ^ 32, and the accumulator registers are, as they stand, the B
// operand of O^T += V^T P^T.  The maximum is raised only when a block exceeds it by 2^8 (fp16: 2^15; P stays
// below that, exact to scale in fp32 sums).  P is rounded to 16 bits for the second product (the
// MFMA's operand type); the sum adds the unrounded values.
//
// Backward: P = exp(S - L), dV = P^T dO, dS = P (dO V^T - delta), dQ = dS K, dK = dS^T Q, in two
// kernels without atomics: one walks keys for a block of rows (dQ), one walks rows for a block of
// keys (dK, dV; the rows of all heads of the group, so that the sum over the heads that share a key
// head is one more stretch of the same contraction).  S and dP are computed in both: the
// alternative, dQ by atomics, is bound by their rate and not reproducible.  dS is rounded to 16
// bits as an operand, as P is.
//
// Measured (causal; two cards where they differ): bf16 d 128, 16.4k tokens in 5 sequences, 32/8 heads: forward 738 to
// 827 us (1017 to 907 TFLOP/s), dQ 1017 to 1138, dK / dV 1406 to 1576, matrix cores 49 to 55 % busy beside the
// exponentials.  bf16 d 64, 14.7k tokens in 26, 16/4 heads: 77 to 82, 105 to 113, 161 to 176 us, 26 to 30 % busy, vector
// work for half as many products.  fp32 d 64, 4.1k tokens in 13, 6/6 heads: 36, 50, 67 us, waves waiting half of the
// time on a grid of one or two workgroups a CU.  fp16's scales of dS: 3.4 % of forward and backward (the bf16 cases in
// fp16 without / with them 317 / 328 us and 3401 / 3514).
#include "attn_launch.h"
#include "attn_packed.h"
#include "attn_packed_tiles.h"

#include <math.h>

#include <type_traits>

namespace ctattn {
namespace {

using namespace packedtile;

constexpr float kLowest = -3.402823466e38f;  // the running maximum before any score (finite: m - m is 0, not NaN)
// m, the running maximum, is raised when a block exceeds it by 2^8, to the row's maximum.  fp16 (F::RANGE): to 2^7 below
// it, when a block exceeds it by 2^15, so that P fills the format: its smallest step, 2^-24, is 2^-31 of the row's largest
// P then, where 2^-24 of it would be lost for every one of a long row's keys.
template <typename F> struct Rise {
    static constexpr float UNDER = F::RANGE ? 7.f : 0.f;
    static constexpr float BY = F::RANGE ? 15.f : 8.f;
    static constexpr float PSUM = F::RANGE ? 32768.f : 256.f;  // a lane's share of a block's P below which no P exceeds 2^BY
};

// Byte strides and pointers of one [tokens, heads, d] tensor.
struct View {
    char *p;
    int64_t row, head;
    __device__ char *at(int64_t n, int h) const { return p + n * row + h * head; }
};

struct FwdArgs {
    View q, k, v, o;
    float *lse;
    const PackedItem *items;
    int hkv, group, causal, width;  // width: bytes of d elements
    float c;                        // log2(e) / sqrt(d)
};

// How a workgroup's 4 waves share its work: RS slices of 32 rows x KS slices of 32 KT keys of every block.
// KS > 1: the waves of a row slice hold sums over different keys and join them at the end; for grids that
// would leave CUs idle, or wait for the one workgroup with the longest sequence.
template <int RS_, int KS_, int KT_> struct Waves {
    static constexpr int RS = RS_, KS = KS_, KT = KT_;
    static_assert(RS * KS == 4, "4 waves");
    static constexpr PackedTile ROWS = RS == 4 ? kRows128 : RS == 2 ? kRows64 : kRows32;
};
template <typename F, int D, typename W> struct FwdCfg : W {
    static constexpr int NW = 4;
    static constexpr int BM = 32 * W::RS;
    static constexpr int BN = 32 * W::KT * W::KS;
    static constexpr int DT = D / 32;
    static constexpr int RB = D * F::ES;
    static constexpr int STEPS = RB / 32;
    static constexpr int KB = BN * RB;
    // Two buffers, or with shared keys one where that lets a second workgroup onto the CU.
    static constexpr int NBUF = W::KS > 1 && 4 * KB > 80 * 1024 ? 1 : 2;
    static constexpr int LDS = NBUF * 2 * KB;  // buffer b: K at 2 b KB, V behind it
    static constexpr int WPE = RB > 256 || LDS > 80 * 1024 ? 1 : 2;
};

template <typename F, int D, bool PAD, typename W>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(FwdCfg<F, D, W>::WPE, 2))) void packed_fwd_kernel(
    FwdArgs a) {
    using C = FwdCfg<F, D, W>;
    using V = typename F::vec;
    using S = typename F::store;
    __shared__ __attribute__((aligned(1024))) char smem[C::LDS];
    const uint32_t L = lds_addr(smem);
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int col = lane & 31, half = lane >> 5;

    const int kvh = blockIdx.x % a.hkv;
    const PackedItem it = a.items[blockIdx.x / a.hkv];
    const int rows = it.len * a.group;
    const int rs = wave % C::RS, ks = wave / C::RS;
    const int r0 = it.tile * C::BM, r0w = r0 + 32 * rs;
    const int row = r0w + col;
    const int token = row / a.group, head = kvh * a.group + row % a.group;
    const int first_token = r0w / a.group;  // of this wave
    const int last_token = min((r0w + 31) / a.group, it.len - 1);
    const int koff = 32 * C::KT * ks;       // of this wave's keys in a block

    V qb[C::STEPS];
    {
        const char *p = a.q.at(it.start + token, head);
#pragma unroll
        for (int s = 0; s < C::STEPS; ++s) {
            floatx4 x = {0.f, 0.f, 0.f, 0.f};
            if (row < rows && (!PAD || 32 * s + 16 * half < a.width))
                x = *reinterpret_cast<const floatx4 *>(p + 32 * s + 16 * half);
            qb[s] = __builtin_bit_cast(V, x);
        }
    }
    floatx16 oacc[C::DT];
#pragma unroll
    for (int dt = 0; dt < C::DT; ++dt) oacc[dt] = zero16();
    float m_run = kLowest, l_run = 0.f;

    const uint32_t rk = uint32_t(Tile<C::RB / 2>::off(col, half));
    const uint32_t cv0 = F::template col0<C::RB>(lane), cv1 = F::template col1<C::RB>(lane);

    const char *kb0 = a.k.at(it.start, kvh), *vb0 = a.v.at(it.start, kvh);
    const int kend = a.causal ? min(it.len, (min(r0 + C::BM, rows) - 1) / a.group + 1) : it.len;
    const int nkb = (kend + C::BN - 1) / C::BN;
    auto issue = [&](int kb) __attribute__((always_inline)) {
        const uint32_t t = L + uint32_t((kb % C::NBUF) * 2 * C::KB);
        const int j0 = kb * C::BN;
        load_rows<C::RB, C::BN, C::NW, PAD>(t, kb0 + j0 * a.k.row, a.k.row, a.width, it.len - j0, wave, lane);
        load_rows<C::RB, C::BN, C::NW, PAD>(t + C::KB, vb0 + j0 * a.v.row, a.v.row, a.width, it.len - j0, wave, lane);
    };
    // This wave's keys of a block.  MASK: they cross the wave's diagonal or the sequence's end.
    auto block = [&](auto mask, int kb) __attribute__((always_inline)) {
        constexpr bool MASK = decltype(mask)::value;
        const int j0 = kb * C::BN + koff;
        const uint32_t kt0 = L + uint32_t((kb % C::NBUF) * 2 * C::KB) + uint32_t(koff * C::RB);
        bool active[C::KT];
        floatx16 sacc[C::KT];
#pragma unroll
        for (int kt = 0; kt < C::KT; ++kt) {
            const int t0 = j0 + 32 * kt;
            active[kt] = !MASK || (t0 < it.len && (!a.causal || t0 <= last_token));
            sacc[kt] = zero16();
            if (!active[kt]) continue;
            const uint32_t ka = kt0 + rk + uint32_t(32 * kt * C::RB);
            V x[2];
            x[0] = lds_b128<V>(ka);
#pragma unroll
            for (int s = 0; s < C::STEPS; ++s) {
                if (s + 1 < C::STEPS) x[(s + 1) & 1] = lds_b128<V>(ka ^ uint32_t((s + 1) << 5));
                read_fence();
                sacc[kt] = F::mma(x[s & 1], qb[s], sacc[kt]);
            }
            if (MASK) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int key = t0 + acc_row(r, half);
                    if (key >= it.len || (a.causal && key > token)) sacc[kt][r] = -INFINITY;
                }
            }
        }
        typename F::pvec pb[C::KT][2];
        float psum;
        auto expo = [&]() __attribute__((always_inline)) {
            psum = 0.f;
#pragma unroll
            for (int kt = 0; kt < C::KT; ++kt) {
                if (!active[kt]) continue;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float p = fast_exp2(fmaf(sacc[kt][r], a.c, -m_run));
                    psum += p;
                    F::put(pb[kt][r / 8], r % 8, p);
                }
            }
        };
        expo();
        if (__any(!(psum <= Rise<F>::PSUM))) {
            float top = -INFINITY;
#pragma unroll
            for (int kt = 0; kt < C::KT; ++kt) {
                if (!active[kt]) continue;
#pragma unroll
                for (int r = 0; r < 16; ++r) top = fmaxf(top, sacc[kt][r]);
            }
            top = max_xor32(top) * a.c;
            if (__any(top > m_run + Rise<F>::BY)) {
                // A row that sees none of the wave's keys yet keeps m at the lowest: P = 2^(-inf) = 0.
                const float m_new = fmaxf(m_run, top - Rise<F>::UNDER);
                const float resc = fast_exp2(m_run - m_new);
                m_run = m_new;
                l_run *= resc;
#pragma unroll
                for (int dt = 0; dt < C::DT; ++dt) oacc[dt] *= resc;
            }
            expo();
        }
        l_run += psum;
        const uint32_t v0 = kt0 + uint32_t(C::KB) + cv0, v1 = kt0 + uint32_t(C::KB) + cv1;
#pragma unroll
        for (int kt = 0; kt < C::KT; ++kt) {
            if (!active[kt]) continue;
            constexpr int NS = 2 * C::DT;
            typename F::cols x[2];
            x[0] = F::template read_cols<C::RB>(v0 + 32 * kt * C::RB, v1 + 32 * kt * C::RB, 0, 0);
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                if (i + 1 < NS)
                    x[(i + 1) & 1] = F::template read_cols<C::RB>(v0 + 32 * kt * C::RB, v1 + 32 * kt * C::RB,
                                                                  (i + 1) / C::DT, (i + 1) % C::DT);
                read_fence();
                oacc[i % C::DT] = F::col_mma(x[i & 1], pb[kt][i / C::DT], oacc[i % C::DT]);
            }
        }
    };

    auto step = [&](int kb) __attribute__((always_inline)) {
        if (C::NBUF == 1 && kb > 0) {
            lds_barrier();  // every wave is done with the last block
            issue(kb);
        }
        // This wave's loads of the block have landed; after the barrier every wave's have, and
        // (two buffers) every wave is done reading the other one.
        wait_loads();
        lds_barrier();
        if (C::NBUF == 2 && kb + 1 < nkb) issue(kb + 1);
    };
    // This wave's blocks, in loops without branches inside (one loop over both variants makes the
    // compiler copy the accumulators): [0, jp) whole, [jp, jw) across the diagonal or the end,
    // [jw, nkb) none of its pairs.
    const int kwhole = a.causal ? min(it.len, first_token + 1) : it.len;  // keys that every row of the wave sees
    const int ksome = a.causal ? last_token + 1 : it.len;                 // and any of them
    const int jw = r0w < rows && ksome > koff ? (ksome - koff + C::BN - 1) / C::BN : 0;
    const int jp = min(jw, kwhole >= koff + 32 * C::KT ? (kwhole - koff - 32 * C::KT) / C::BN + 1 : 0);
    issue(0);
    int kb = 0;
    for (; kb < jp; ++kb) {
        step(kb);
        block(std::false_type{}, kb);
    }
    for (; kb < jw; ++kb) {
        step(kb);
        block(std::true_type{}, kb);
    }
    for (; kb < nkb; ++kb) step(kb);

    if constexpr (C::KS > 1) {
        // The key slices of a row slice join: m = max, O and l weighted by 2^(their m - m).  A slice that
        // saw no key has the lowest m, weight 0; the first saw key 0.
        constexpr int NR = C::DT * 16 + 2;
        static_assert((C::KS - 1) * C::RS * NR * kWave * 4 <= C::LDS, "join buffer");
        float *jb = reinterpret_cast<float *>(smem);
        lds_barrier();  // every wave is done with the tiles
        if (ks > 0) {
            float *to = jb + ((ks - 1) * C::RS + rs) * NR * kWave + lane;
#pragma unroll
            for (int dt = 0; dt < C::DT; ++dt)
#pragma unroll
                for (int r = 0; r < 16; ++r) to[(dt * 16 + r) * kWave] = oacc[dt][r];
            to[(NR - 2) * kWave] = m_run;
            to[(NR - 1) * kWave] = l_run;
        }
        lds_barrier();
        if (ks > 0) return;
        const float *from = jb + rs * NR * kWave + lane;
        float m = m_run, w[C::KS - 1];
#pragma unroll
        for (int i = 0; i < C::KS - 1; ++i) m = fmaxf(m, from[i * C::RS * NR * kWave + (NR - 2) * kWave]);
        const float w0 = fast_exp2(m_run - m);
        l_run *= w0;
#pragma unroll
        for (int i = 0; i < C::KS - 1; ++i) {
            w[i] = fast_exp2(from[i * C::RS * NR * kWave + (NR - 2) * kWave] - m);
            l_run += from[i * C::RS * NR * kWave + (NR - 1) * kWave] * w[i];
        }
#pragma unroll
        for (int dt = 0; dt < C::DT; ++dt)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                float x = oacc[dt][r] * w0;
#pragma unroll
                for (int i = 0; i < C::KS - 1; ++i) x += from[i * C::RS * NR * kWave + (dt * 16 + r) * kWave] * w[i];
                oacc[dt][r] = x;
            }
        m_run = m;
    }
    const float l_tot = l_run + __shfl_xor(l_run, 32, kWave);
    const float inv_l = 1.f / l_tot;
    if (row < rows) {
        S *orow = reinterpret_cast<S *>(a.o.at(it.start + token, head));
#pragma unroll
        for (int dt = 0; dt < C::DT; ++dt) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                if (PAD && (32 * dt + 8 * g + 4 * half) * F::ES >= a.width) continue;
                const float x[4] = {oacc[dt][4 * g] * inv_l, oacc[dt][4 * g + 1] * inv_l, oacc[dt][4 * g + 2] * inv_l,
                                    oacc[dt][4 * g + 3] * inv_l};
                store4<F>(orow + 32 * dt + 8 * g + 4 * half, x);
            }
        }
        if (a.lse != nullptr && half == 0)
            a.lse[int64_t(it.start + token) * (a.hkv * a.group) + head] = (m_run + __log2f(l_tot)) * kLn2;
    }
}

// ---- backward ----

// fp16 (F::RANGE): P enters dV's product as 2^kPExp P, and dS as es dS with es a power of two of the lane's own row or
// key, from kDsStart down.  Finite inputs keep |es dS| below 2^(10 + 39 + 50) at the start, inside fp32.
constexpr int kPExp = 10;
constexpr float kDsStart = 1125899906842624.f;  // 2^50
constexpr float kDsLimit = 32768.f;  // a lane's sum of |dS| es over 16 rows or keys below which none passes fp16's range

// The lane's 16 values es dS: where their sum passes the limit, and for every lane of the wave that holds a value from
// kDsLimit / 16 on, a smaller es, so that the largest of the row or key (lane and lane ^ 32) lies in [2^7, 2^8).  Returns
// the power of two by which es changes, and with it the values and the sums.
__device__ __forceinline__ float fit_range(float (&w)[16]) {
    float sum = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) sum += fabsf(w[r]);
    if (!__any(!(sum <= kDsLimit))) return 1.f;
    float top = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(w[r]));
    top = max_xor32(top);
    float f = 1.f;
    // 2^(7 - exponent) from the exponent bits; an infinity or NaN stays what it is.
    if (top >= kDsLimit / 16 && top < INFINITY) f = __uint_as_float(uint32_t(127 + 7 + 127 - int(__float_as_uint(top) >> 23)) << 23);
#pragma unroll
    for (int r = 0; r < 16; ++r) w[r] *= f;
    return f;
}

struct BwdArgs {
    View q, k, v, o, dout, dq, dk, dv;
    const float *lse;
    // -delta = -rowsum(dO O) and -L log2(e) (fp16: + kPExp) of every (token, head), rows (token, head of the group) behind
    // each other for each key head, as the dK / dV kernel walks them.  The dQ kernel, which has dO's rows in
    // registers, runs first and writes them.
    float *ndelta, *nl2;
    const PackedItem *items;
    int64_t tokens;
    int hkv, group, causal, width;
    // ceil(65536 / group): x / group = x magic >> 16 while x (group - 1) < 65536, as magic group exceeds 65536 by less than
    // group (KvCfg asserts it of every tile and group).
    uint32_t magic;
    float c, inv_sqrt_d;
};

// KS slices of 32 keys x RS slices of 32 rows, one wave each; the row slices' sums join at the end.
template <int KS_, int RS_, int NBUF_> struct KvWaves {
    static constexpr int KS = KS_, RS = RS_, NBUF = NBUF_;
    static constexpr PackedTile KEYS = KS == 4 ? kKeys128 : KS == 2 ? kKeys64 : kKeys32;
};
template <typename F, int D, typename W> struct KvCfg : W {
    static constexpr int RB = D * F::ES;
    static constexpr int NW = W::KS * W::RS;
    static constexpr int BN = 32 * W::KS;
    static constexpr int BM = 32 * W::RS;
    static constexpr int DT = D / 32;
    static constexpr int STEPS = RB / 32;
    static constexpr int QB = BM * RB;             // Q (or dO) tile
    static constexpr int KB = BN * RB;
    // One key slice: its K and V rows in registers instead of LDS, where they fit beside dK and dV.
    static constexpr bool KREG = W::KS == 1 && !(F::ES == 2 && D == 128);
    static constexpr int K_OFF = W::NBUF * 2 * QB; // buffer b: Q at 2 b QB, dO behind it
    static constexpr int V_OFF = K_OFF + (KREG ? 0 : KB);
    static constexpr int S_OFF = V_OFF + (KREG ? 0 : KB);  // buffer b: nl2[BM], ndelta[BM]
    static constexpr int LDS = S_OFF + W::NBUF * 2 * BM * 4;
    static_assert(LDS <= 160 * 1024, "LDS");
    static_assert((BM + kMfmaMaxGroup - 2) * (kMfmaMaxGroup - 1) < 65536, "rows of a tile by BwdArgs::magic");
    static constexpr int WPE = NW >= 8 || LDS <= 80 * 1024 ? 2 : 1;
    static_assert(W::KS * W::RS / 2 * DT * 2 * 16 * kWave * 4 <= LDS, "reduction buffer");
};

template <typename F, int D, bool PAD, typename W>
__global__ __launch_bounds__((64 * KvCfg<F, D, W>::NW)) __attribute__((amdgpu_waves_per_eu(KvCfg<F, D, W>::WPE, 2))) void
packed_dkdv_kernel(BwdArgs a) {
    using C = KvCfg<F, D, W>;
    using V = typename F::vec;
    using S = typename F::store;
    __shared__ __attribute__((aligned(1024))) char smem[C::LDS];
    const uint32_t L = lds_addr(smem);
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int col = lane & 31, half = lane >> 5;
    const int ks = wave % C::KS, rs = wave / C::KS;

    const int kvh = blockIdx.x % a.hkv;
    const PackedItem it = a.items[blockIdx.x / a.hkv];
    const int rows = it.len * a.group;
    const int k0 = it.tile * C::BN;
    const int kw0 = k0 + 32 * ks;
    const int key = kw0 + col;
    const int64_t sbase = (int64_t(kvh) * a.tokens + it.start) * a.group;

    V kreg[C::KREG ? C::STEPS : 1], vreg[C::KREG ? C::STEPS : 1];
    if constexpr (C::KREG) {
        const char *pk = a.k.at(it.start + key, kvh), *pv = a.v.at(it.start + key, kvh);
#pragma unroll
        for (int s = 0; s < C::STEPS; ++s) {
            floatx4 x = {0.f, 0.f, 0.f, 0.f}, y = {0.f, 0.f, 0.f, 0.f};
            if (key < it.len && (!PAD || 32 * s + 16 * half < a.width)) {
                x = *reinterpret_cast<const floatx4 *>(pk + 32 * s + 16 * half);
                y = *reinterpret_cast<const floatx4 *>(pv + 32 * s + 16 * half);
            }
            kreg[s] = __builtin_bit_cast(V, x);
            vreg[s] = __builtin_bit_cast(V, y);
        }
    } else {
        load_rows<C::RB, C::BN, C::NW, PAD>(L + C::K_OFF, a.k.at(it.start + k0, kvh), a.k.row, a.width, it.len - k0, wave, lane);
        load_rows<C::RB, C::BN, C::NW, PAD>(L + C::V_OFF, a.v.at(it.start + k0, kvh), a.v.row, a.width, it.len - k0, wave, lane);
    }
    floatx16 dk[C::DT], dv[C::DT];
#pragma unroll
    for (int dt = 0; dt < C::DT; ++dt) dk[dt] = zero16(), dv[dt] = zero16();
    float es = kDsStart;  // of the lane's key (fp16)

    const uint32_t rq = uint32_t(Tile<C::RB / 2>::off(32 * rs + col, half));
    const uint32_t ak = L + C::K_OFF + uint32_t(Tile<C::RB / 2>::off(32 * ks + col, half));
    const uint32_t cq0 = F::template col0<C::RB>(lane) + 32 * rs * C::RB, cq1 = F::template col1<C::RB>(lane) + 32 * rs * C::RB;

    const int nqb = (rows + C::BM - 1) / C::BM;
    const int qb_first = a.causal ? int(int64_t(k0) * a.group / C::BM) : 0;
    auto issue = [&](int qb, int buf) __attribute__((always_inline)) {
        using T = Tile<C::RB / 2>;
        constexpr int TOTAL = C::BM * T::CH, NL = (TOTAL + C::NW * kWave - 1) / (C::NW * kWave);
        const int r0 = qb * C::BM;
        const int t0 = r0 / a.group, rem = r0 - t0 * a.group;  // uniform
        const uint32_t qt = L + uint32_t(buf * 2 * C::QB);
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            if ((wave * NL + i) * kWave >= TOTAL) continue;
            const int P = (wave * NL + i) * kWave + lane;
            const int r = P / T::CH;
            const int c = 16 * ((P % T::CH) ^ T::swz(r));
            const int x = rem + min(r, rows - 1 - r0);  // row x - rem of the tile: token t0 + x / group
            const int t = int(uint32_t(x) * a.magic >> 16);
            const int64_t n = it.start + t0 + t;
            const int h = kvh * a.group + x - t * a.group;
            const char *gq = a.q.at(n, h) + c, *gd = a.dout.at(n, h) + c;
            if (PAD && c >= a.width) gq = gd = reinterpret_cast<const char *>(tile_zeros);
            const uint32_t dst = qt + uint32_t((wave * NL + i) * kWave * 16);
            load_chunk_dma(gq, dst);
            load_chunk_dma(gd, dst + C::QB);
        }
        // nl2 and ndelta of the block's rows: 64 a load, the last waves' turn.
        constexpr int SL = (C::BM + kWave - 1) / kWave;
        static_assert(2 * SL <= C::NW && C::BM % kWave == 0, "row statistics");
        if (wave >= C::NW - 2 * SL) {
            const int i = wave - (C::NW - 2 * SL), part = i % SL;
            load_dword_dma((i < SL ? a.nl2 : a.ndelta) + sbase + min(r0 + part * kWave + lane, rows - 1),
                           L + C::S_OFF + uint32_t((buf * 2 + i / SL) * C::BM * 4 + part * kWave * 4));
        }
    };
    // One 32-row x 32-key tile: S, dP - delta (its accumulator starts from -delta), P, dS.
    auto block = [&](auto mask, int r0w, int buf) __attribute__((always_inline)) {
        constexpr bool MASK = decltype(mask)::value;
        const uint32_t qt = L + uint32_t(buf * 2 * C::QB);
        const uint32_t anl = L + C::S_OFF + uint32_t(buf * 2 * C::BM * 4 + 4 * (32 * rs + 4 * half));
        floatx16 s = zero16(), dp;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const floatx4 x = lds_f4(anl + C::BM * 4 + 32 * g);
#pragma unroll
            for (int t = 0; t < 4; ++t) dp[4 * g + t] = x[t];
        }
        {
            V q[2], k[2], g[2], v[2];
            const uint32_t aq = qt + rq;
            q[0] = lds_b128<V>(aq);
            g[0] = lds_b128<V>(aq + C::QB);
            if (!C::KREG) {
                k[0] = lds_b128<V>(ak);
                v[0] = lds_b128<V>(ak + C::KB);
            }
#pragma unroll
            for (int st = 0; st < C::STEPS; ++st) {
                const int cur = st & 1, nxt = cur ^ 1;
                if (st + 1 < C::STEPS) {
                    const uint32_t xq = aq ^ uint32_t((st + 1) << 5), xk = ak ^ uint32_t((st + 1) << 5);
                    q[nxt] = lds_b128<V>(xq);
                    g[nxt] = lds_b128<V>(xq + C::QB);
                    if (!C::KREG) {
                        k[nxt] = lds_b128<V>(xk);
                        v[nxt] = lds_b128<V>(xk + C::KB);
                    }
                }
                read_fence();
                s = F::mma(q[cur], C::KREG ? kreg[C::KREG ? st : 0] : k[cur], s);
                dp = F::mma(g[cur], C::KREG ? vreg[C::KREG ? st : 0] : v[cur], dp);
            }
        }
        typename F::pvec pb[2], db[2];
        [[maybe_unused]] float w[16];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const floatx4 n4 = lds_f4(anl + 32 * g);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const int r = 4 * g + t;
                float p = fast_exp2(fmaf(s[r], a.c, n4[t]));
                float ds = p * dp[r];
                if (MASK) {
                    // key > row / group is key * group > row.  dS by itself: 0 times an infinite dP is not 0.
                    const int row = r0w + acc_row(r, half);
                    const bool hidden = row >= rows || key >= it.len || (a.causal && key * a.group > row);
                    p = hidden ? 0.f : p;
                    ds = hidden ? 0.f : ds;
                }
                F::put(pb[r / 8], r % 8, p);
                if constexpr (F::RANGE) w[r] = ds * es;
                else F::put(db[r / 8], r % 8, ds);
            }
        }
        if constexpr (F::RANGE) {
            const float f = fit_range(w);
            if (__any(f != 1.f)) {
                es *= f;
#pragma unroll
                for (int dt = 0; dt < C::DT; ++dt) dk[dt] *= f;
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) F::put(db[r / 8], r % 8, w[r]);
        }
        constexpr int NS = 2 * C::DT;
        typename F::cols go[2], gq[2];
        const uint32_t c0 = qt + cq0, c1 = qt + cq1;
        go[0] = F::template read_cols<C::RB>(c0 + C::QB, c1 + C::QB, 0, 0);
        gq[0] = F::template read_cols<C::RB>(c0, c1, 0, 0);
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const int cur = i & 1, nxt = cur ^ 1;
            if (i + 1 < NS) {
                go[nxt] = F::template read_cols<C::RB>(c0 + C::QB, c1 + C::QB, (i + 1) / C::DT, (i + 1) % C::DT);
                gq[nxt] = F::template read_cols<C::RB>(c0, c1, (i + 1) / C::DT, (i + 1) % C::DT);
            }
            read_fence();
            dv[i % C::DT] = F::col_mma(go[cur], pb[i / C::DT], dv[i % C::DT]);
            dk[i % C::DT] = F::col_mma(gq[cur], db[i / C::DT], dk[i % C::DT]);
        }
    };

    // Rows from the last to the first that sees the keys: the workgroups of a sequence and key head begin with the
    // same blocks, which they find in L2 (bf16 d 128, 16.4k tokens, 32/8 heads: 1574 us from the diagonal down, 1515
    // from the end up).
    auto step = [&](int qb) __attribute__((always_inline)) {
        const int buf = C::NBUF == 2 ? (nqb - 1 - qb) & 1 : 0;
        if (C::NBUF == 1) {
            lds_barrier();  // every wave is done with the last block
            issue(qb, 0);
        }
        wait_loads();
        lds_barrier();
        if (C::NBUF == 2 && qb > qb_first) issue(qb - 1, buf ^ 1);
        return buf;
    };
    // This wave's blocks, in loops without branches inside (one loop over both variants makes the
    // compiler copy the accumulators): [qb_first, qa) none of its pairs, [qa, qp) across the diagonal,
    // [qp, qe) whole, [qe, qn) across the last row, [qn, nqb) none of its rows.
    int qa = nqb, qp = nqb, qe = nqb, qn = nqb;
    if (kw0 < it.len) {
        auto first_block = [&](int r) { return max(qb_first, (r - 32 * rs + C::BM - 1) / C::BM); };  // rows from r on
        qn = max(qb_first, (rows - 32 * rs + C::BM - 1) / C::BM);          // r0w < rows before it
        qe = max(qb_first, rows < 32 * rs + 32 ? 0 : (rows - 32 * rs - 32) / C::BM + 1);
        // Causal: r0w + 31 >= kw0 * group for a pair, r0w >= (kw0 + 31) * group for whole tiles.
        qa = a.causal ? first_block(max(0, kw0 * a.group - 31)) : qb_first;
        qp = kw0 + 32 > it.len ? qn : a.causal ? first_block((kw0 + 31) * a.group) : qb_first;
        qn = min(qn, nqb);
        qa = min(qa, qn);
        qp = min(max(qp, qa), qn);
        qe = min(max(qe, qp), qn);
    }
    if (C::NBUF == 2) issue(nqb - 1, 0);  // the tile's first key is in the sequence: qb_first < nqb
    int qb = nqb - 1;
    for (; qb >= qn; --qb) step(qb);
    for (; qb >= qe; --qb) {
        const int buf = step(qb);
        block(std::true_type{}, qb * C::BM + 32 * rs, buf);
    }
    for (; qb >= qp; --qb) {
        const int buf = step(qb);
        block(std::false_type{}, qb * C::BM + 32 * rs, buf);
    }
    for (; qb >= qa; --qb) {
        const int buf = step(qb);
        block(std::true_type{}, qb * C::BM + 32 * rs, buf);
    }
    for (; qb >= qb_first; --qb) step(qb);

    if constexpr (F::RANGE) {
        const float back = 1.f / (es * float(1 << kPExp));
#pragma unroll
        for (int dt = 0; dt < C::DT; ++dt) dk[dt] *= back, dv[dt] *= 1.f / float(1 << kPExp);
    }
    // The row slices' sums join through LDS, the upper half of them added to the lower.
    float *red = reinterpret_cast<float *>(smem);
#pragma unroll
    for (int h = C::RS / 2; h >= 1; h /= 2) {
        lds_barrier();
        float *at = red + ((rs % h) * C::KS + ks) * C::DT * 32 * kWave + lane;
        if (rs >= h && rs < 2 * h) {
#pragma unroll
            for (int dt = 0; dt < C::DT; ++dt)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    at[(dt * 32 + r) * kWave] = dk[dt][r];
                    at[(dt * 32 + 16 + r) * kWave] = dv[dt][r];
                }
        }
        lds_barrier();
        if (rs < h) {
#pragma unroll
            for (int dt = 0; dt < C::DT; ++dt)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    dk[dt][r] += at[(dt * 32 + r) * kWave];
                    dv[dt][r] += at[(dt * 32 + 16 + r) * kWave];
                }
        }
    }
    if (rs == 0 && key < it.len) {
        S *dkr = reinterpret_cast<S *>(a.dk.at(it.start + key, kvh));
        S *dvr = reinterpret_cast<S *>(a.dv.at(it.start + key, kvh));
#pragma unroll
        for (int dt = 0; dt < C::DT; ++dt) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                if (PAD && (32 * dt + 8 * g + 4 * half) * F::ES >= a.width) continue;
                float xk[4], xv[4];
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    xk[t] = dk[dt][4 * g + t] * a.inv_sqrt_d;
                    xv[t] = dv[dt][4 * g + t];
                }
                store4<F>(dkr + 32 * dt + 8 * g + 4 * half, xk);
                store4<F>(dvr + 32 * dt + 8 * g + 4 * half, xv);
            }
        }
    }
}

template <typename F, int D, typename W> struct QCfg : W {
    static constexpr int NW = 4;
    static constexpr int BM = 32 * W::RS;
    static constexpr int BN = 32 * W::KS;
    static_assert(W::KT == 1, "32 keys of a wave");
    static constexpr int RB = D * F::ES;
    static constexpr int DT = D / 32;
    static constexpr int STEPS = RB / 32;
    static constexpr int KB = BN * RB;
    static constexpr int NBUF = W::KS > 1 && 4 * KB > 80 * 1024 ? 1 : 2;  // as in the forward
    static constexpr int LDS = NBUF * 2 * KB;
    static constexpr int WPE = RB > 256 || LDS > 80 * 1024 ? 1 : 2;
};

template <typename F, int D, bool PAD, typename W>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(QCfg<F, D, W>::WPE, 2))) void packed_dq_kernel(
    BwdArgs a) {
    using C = QCfg<F, D, W>;
    using V = typename F::vec;
    using S = typename F::store;
    __shared__ __attribute__((aligned(1024))) char smem[C::LDS];
    const uint32_t L = lds_addr(smem);
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int col = lane & 31, half = lane >> 5;

    const int kvh = blockIdx.x % a.hkv;
    const PackedItem it = a.items[blockIdx.x / a.hkv];
    const int rows = it.len * a.group;
    const int rs = wave % C::RS, ks = wave / C::RS, koff = 32 * ks;
    const int r0 = it.tile * C::BM;
    const int r0w = r0 + 32 * rs;
    const int row = r0w + col;
    const int token = row / a.group, head = kvh * a.group + row % a.group;
    const int first_token = r0w / a.group;
    const int last_token = min((r0w + 31) / a.group, it.len - 1);

    V qb[C::STEPS], gb[C::STEPS];
    float nd = 0.f;
    {
        const char *pq = a.q.at(it.start + token, head), *pg = a.dout.at(it.start + token, head);
        const char *po = a.o.at(it.start + token, head);
#pragma unroll
        for (int s = 0; s < C::STEPS; ++s) {
            floatx4 x = {0.f, 0.f, 0.f, 0.f}, y = {0.f, 0.f, 0.f, 0.f}, z = {0.f, 0.f, 0.f, 0.f};
            if (row < rows && (!PAD || 32 * s + 16 * half < a.width)) {
                x = *reinterpret_cast<const floatx4 *>(pq + 32 * s + 16 * half);
                y = *reinterpret_cast<const floatx4 *>(pg + 32 * s + 16 * half);
                z = *reinterpret_cast<const floatx4 *>(po + 32 * s + 16 * half);
            }
            qb[s] = __builtin_bit_cast(V, x);
            gb[s] = __builtin_bit_cast(V, y);
            const V ov = __builtin_bit_cast(V, z);
#pragma unroll
            for (int e = 0; e < 16 / F::ES; ++e) nd -= float(gb[s][e]) * float(ov[e]);
        }
    }
    nd += __shfl_xor(nd, 32, kWave);  // the row's other half
    const float nl = row < rows ? -a.lse[int64_t(it.start + token) * (a.hkv * a.group) + head] * kLog2e : 0.f;
    floatx16 dq[C::DT];
#pragma unroll
    for (int dt = 0; dt < C::DT; ++dt) dq[dt] = zero16();
    // fp16: dS's scale of the lane's row, which P's exponent takes along.
    float es = F::RANGE ? kDsStart : 1.f;
    float nls = F::RANGE ? nl + log2f(kDsStart) : nl;

    const uint32_t rk = uint32_t(Tile<C::RB / 2>::off(col, half));
    const uint32_t ck0 = F::template col0<C::RB>(lane), ck1 = F::template col1<C::RB>(lane);
    const char *kb0 = a.k.at(it.start, kvh), *vb0 = a.v.at(it.start, kvh);
    const int kend = a.causal ? min(it.len, (min(r0 + C::BM, rows) - 1) / a.group + 1) : it.len;
    const int nkb = (kend + C::BN - 1) / C::BN;
    auto issue = [&](int kb) __attribute__((always_inline)) {
        const uint32_t t = L + uint32_t((kb % C::NBUF) * 2 * C::KB);
        const int j0 = kb * C::BN;
        load_rows<C::RB, C::BN, C::NW, PAD>(t, kb0 + j0 * a.k.row, a.k.row, a.width, it.len - j0, wave, lane);
        load_rows<C::RB, C::BN, C::NW, PAD>(t + C::KB, vb0 + j0 * a.v.row, a.v.row, a.width, it.len - j0, wave, lane);
    };
    // ALONE: the block holds every key that the wave's rows see, so that delta = sum_j P dP is there before dS needs it.
    // rowsum(dO O) is off by O's rounding, which for rows of few keys (O as large as V, dS small or 0) is as much as the
    // other roundings of dQ and dK: 26 documents of 1 to 3011 tokens, bf16, dQ off by 2.6e-3 of its norm with it
    // everywhere, by 2.4e-3 this way.
    auto block = [&](auto mask, auto alone, int kb) __attribute__((always_inline)) {
        constexpr bool MASK = decltype(mask)::value, ALONE = decltype(alone)::value;
        const uint32_t kt = L + uint32_t((kb % C::NBUF) * 2 * C::KB) + uint32_t(koff * C::RB);
        floatx16 s = zero16(), dp;
#pragma unroll
        for (int r = 0; r < 16; ++r) dp[r] = ALONE ? 0.f : nd;
        V k[2], v[2];
        const uint32_t ak = kt + rk;
        k[0] = lds_b128<V>(ak);
        v[0] = lds_b128<V>(ak + C::KB);
#pragma unroll
        for (int st = 0; st < C::STEPS; ++st) {
            const int cur = st & 1, nxt = cur ^ 1;
            if (st + 1 < C::STEPS) {
                const uint32_t x = ak ^ uint32_t((st + 1) << 5);
                k[nxt] = lds_b128<V>(x);
                v[nxt] = lds_b128<V>(x + C::KB);
            }
            read_fence();
            s = F::mma(k[cur], qb[st], s);
            dp = F::mma(v[cur], gb[st], dp);
        }
        typename F::pvec db[2];
        [[maybe_unused]] float w[16];
        if constexpr (ALONE) {
            float delta = 0.f;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int key = kb * C::BN + koff + acc_row(r, half);
                const bool hidden = key >= it.len || (a.causal && key > token);
                s[r] = hidden ? 0.f : fast_exp2(fmaf(s[r], a.c, nl));
                dp[r] = hidden ? 0.f : dp[r];
                delta = fmaf(s[r], dp[r], delta);
            }
            delta += __shfl_xor(delta, 32, kWave);
            nd = row < rows ? -delta : 0.f;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float ds = s[r] * (dp[r] - delta);
                if constexpr (F::RANGE) w[r] = ds * es;
                else F::put(db[r / 8], r % 8, ds);
            }
        } else {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                float ds = fast_exp2(fmaf(s[r], a.c, nls)) * dp[r];
                if (MASK) {
                    const int key = kb * C::BN + koff + acc_row(r, half);
                    ds = (key >= it.len || (a.causal && key > token)) ? 0.f : ds;
                }
                if constexpr (F::RANGE) w[r] = ds;
                else F::put(db[r / 8], r % 8, ds);
            }
        }
        if constexpr (F::RANGE) {
            const float f = fit_range(w);
            if (__any(f != 1.f)) {
                es *= f;
                nls = nl + log2f(es);
#pragma unroll
                for (int dt = 0; dt < C::DT; ++dt) dq[dt] *= f;
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) F::put(db[r / 8], r % 8, w[r]);
        }
        constexpr int NS = 2 * C::DT;
        typename F::cols x[2];
        x[0] = F::template read_cols<C::RB>(kt + ck0, kt + ck1, 0, 0);
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            if (i + 1 < NS)
                x[(i + 1) & 1] = F::template read_cols<C::RB>(kt + ck0, kt + ck1, (i + 1) / C::DT, (i + 1) % C::DT);
            read_fence();
            dq[i % C::DT] = F::col_mma(x[i & 1], db[i / C::DT], dq[i % C::DT]);
        }
    };
    auto step = [&](int kb) __attribute__((always_inline)) {
        if (C::NBUF == 1 && kb > 0) {
            lds_barrier();
            issue(kb);
        }
        wait_loads();
        lds_barrier();
        if (C::NBUF == 2 && kb + 1 < nkb) issue(kb + 1);
    };
    // As in the forward; rows past the last one have P = exp2(0 + 0) dP = 0, so they need no mask.
    const int kwhole = a.causal ? min(it.len, first_token + 1) : it.len;
    const int ksome = a.causal ? last_token + 1 : it.len;
    const int jw = r0w < rows && ksome > koff ? (ksome - koff + C::BN - 1) / C::BN : 0;
    const int jp = min(jw, kwhole >= koff + 32 ? (kwhole - koff - 32) / C::BN + 1 : 0);
    issue(0);
    int kb = 0;
    if (jw == 1 && ksome <= 32) {
        step(0);
        block(std::true_type{}, std::true_type{}, 0);
        kb = 1;
    }
    for (; kb < jp; ++kb) {
        step(kb);
        block(std::false_type{}, std::false_type{}, kb);
    }
    for (; kb < jw; ++kb) {
        step(kb);
        block(std::true_type{}, std::false_type{}, kb);
    }
    for (; kb < nkb; ++kb) step(kb);
    if (row < rows && ks == 0 && half == 0) {
        const int64_t at = (int64_t(kvh) * a.tokens + it.start) * a.group + row;
        a.ndelta[at] = nd;
        a.nl2[at] = F::RANGE ? nl + float(kPExp) : nl;
    }
    if constexpr (F::RANGE) {
#pragma unroll
        for (int dt = 0; dt < C::DT; ++dt) dq[dt] *= 1.f / es;
    }
    if constexpr (C::KS > 1) {
        // The key slices' sums join through LDS, the upper half of them added to the lower.
        static_assert(C::KS / 2 * C::RS * C::DT * 16 * kWave * 4 <= C::LDS, "join buffer");
        float *jb = reinterpret_cast<float *>(smem);
#pragma unroll
        for (int h = C::KS / 2; h >= 1; h /= 2) {
            lds_barrier();
            float *at = jb + ((ks % h) * C::RS + rs) * C::DT * 16 * kWave + lane;
            if (ks >= h && ks < 2 * h) {
#pragma unroll
                for (int dt = 0; dt < C::DT; ++dt)
#pragma unroll
                    for (int r = 0; r < 16; ++r) at[(dt * 16 + r) * kWave] = dq[dt][r];
            }
            lds_barrier();
            if (ks < h) {
#pragma unroll
                for (int dt = 0; dt < C::DT; ++dt)
#pragma unroll
                    for (int r = 0; r < 16; ++r) dq[dt][r] += at[(dt * 16 + r) * kWave];
            }
        }
        if (ks > 0) return;
    }
    if (row < rows) {
        S *p = reinterpret_cast<S *>(a.dq.at(it.start + token, head));
#pragma unroll
        for (int dt = 0; dt < C::DT; ++dt) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                if (PAD && (32 * dt + 8 * g + 4 * half) * F::ES >= a.width) continue;
                const float x[4] = {dq[dt][4 * g] * a.inv_sqrt_d, dq[dt][4 * g + 1] * a.inv_sqrt_d,
                                    dq[dt][4 * g + 2] * a.inv_sqrt_d, dq[dt][4 * g + 3] * a.inv_sqrt_d};
                store4<F>(p + 32 * dt + 8 * g + 4 * half, x);
            }
        }
    }
}

// ---- launches ----

// Whether the grid is short of work for its longest workgroup: that one walks `longest` blocks, and the
// batch's pairs make fewer than a quarter of as many blocks of `pairs_of_block` for each of the `slots` workgroups that
// the chip holds at once.  Then smaller tiles, whose waves share the walk, win; else larger ones, which load less for a
// pair.  Measured, us, causal, larger / smaller tiles, with the ratio:
//   forward  bf16 d 64: 26 documents of 14.7k tokens, 16/4 heads (1.1) 78 / 155; 8 x 512 16/4 (2) 14 / 25; 4096 4/2 (8)
//            55 / 28.  d 128: 8192 8/2 (2) 200 / 254; 2048 8/2 (8) 44 / 29.  fp32 d 64: 13 documents of 4k tokens, 6/6 (9)
//            76 / 36; 16 x 512 12/12 (1.3) 83 / 108.  fp32 d 128: 4 x 1024 8/2 (4) 153 / 104
//   dK, dV   (whole backward) bf16 d 64: the 26 documents (4.5) 328 / 275; 8 x 512 16/4 (8) 68 / 49; 4096 4/2 (16) 211 /
//            148; 32 x 512 16/4 (2) 143 / 149; 4 x 2048 16/16 (1) 199 / 232.  d 128: 2048 8/2 (16) 255 / 226;
//            8192 8/2 (4) 1045 / 1292.  fp32 d 64: the 13 documents (4.7) 244 / 175; 16 x 512 12/12 (0.7) 295 / 315
//   dQ       (whole backward) bf16 d 64: 4096 4/2 (8) 210 / 169; 4096 16/4 (2) 365 / 370.  fp32 d 64: the 13 documents (9)
//            244 / 189
bool short_of_work(const PackedCall &c, int64_t longest, int64_t pairs_of_block, int64_t slots, int64_t ratio = 4) {
    const double pairs = double(c.causal ? c.host->pairs_causal : c.host->pairs) * double(c.hq);
    return double(longest) * double(pairs_of_block) * double(slots) >= double(ratio) * pairs;
}

View view(const void *p, const PackedStride &s, int es) {
    return {static_cast<char *>(const_cast<void *>(p)), s.row * es, s.head * es};
}

template <typename F, int D, bool PAD, typename W>
hipError_t fwd_as(const PackedCall &c, FwdArgs a, hipStream_t stream) {
    const int64_t blocks = c.item_count(W::ROWS) * c.hkv;
    if (!grid_fits(blocks, 256)) return hipErrorInvalidValue;
    a.items = c.items(W::ROWS);
    hipLaunchKernelGGL((packed_fwd_kernel<F, D, PAD, W>), dim3(unsigned(blocks)), dim3(256), 0, stream, a);
    return hipGetLastError();
}

template <typename F, int D, bool PAD>
hipError_t run_fwd(const PackedCall &c, const void *q, const void *k, const void *v, void *o, float *lse,
                   hipStream_t stream) {
    FwdArgs a{view(q, c.sq, F::ES), view(k, c.sk, F::ES), view(v, c.sv, F::ES), view(o, c.so, F::ES), lse,
              nullptr, int(c.hkv), int(c.group()), int(c.causal), int(c.d) * F::ES, kLog2e / sqrtf(float(c.d))};
    const bool few = short_of_work(c, (c.host->max_len + 63) / 64, 128 * 64, 2 * device_cus(stream));
    if constexpr (D * F::ES > 256) return few ? fwd_as<F, D, PAD, Waves<2, 2, 1>>(c, a, stream) : fwd_as<F, D, PAD, Waves<4, 1, 2>>(c, a, stream);
    else return few ? fwd_as<F, D, PAD, Waves<1, 4, 1>>(c, a, stream) : fwd_as<F, D, PAD, Waves<4, 1, 2>>(c, a, stream);
}

template <typename F, int D, bool PAD, typename W> hipError_t dkdv_as(const PackedCall &c, BwdArgs a, hipStream_t stream) {
    const int64_t blocks = c.item_count(W::KEYS) * c.hkv;
    constexpr int threads = 64 * KvCfg<F, D, W>::NW;
    if (!grid_fits(blocks, threads)) return hipErrorInvalidValue;
    a.items = c.items(W::KEYS);
    hipLaunchKernelGGL((packed_dkdv_kernel<F, D, PAD, W>), dim3(unsigned(blocks)), dim3(threads), 0, stream, a);
    return hipGetLastError();
}
template <typename F, int D, bool PAD, typename W> hipError_t dq_as(const PackedCall &c, BwdArgs a, hipStream_t stream) {
    const int64_t blocks = c.item_count(W::ROWS) * c.hkv;
    if (!grid_fits(blocks, 256)) return hipErrorInvalidValue;
    a.items = c.items(W::ROWS);
    hipLaunchKernelGGL((packed_dq_kernel<F, D, PAD, W>), dim3(unsigned(blocks)), dim3(256), 0, stream, a);
    return hipGetLastError();
}

template <typename F, int D, bool PAD>
hipError_t run_bwd(const PackedCall &c, const void *q, const void *k, const void *v, const void *o, const void *dout,
                   const float *lse, float *ws, void *dq, void *dk, void *dv, hipStream_t stream) {
    const int64_t rows = c.tokens() * c.hq;
    BwdArgs a{view(q, c.sq, F::ES), view(k, c.sk, F::ES), view(v, c.sv, F::ES), view(o, c.so, F::ES),
              view(dout, c.sdo, F::ES), view(dq, c.sdq, F::ES), view(dk, c.sdk, F::ES), view(dv, c.sdv, F::ES),
              lse, ws, ws + rows, nullptr, c.tokens(), int(c.hkv), int(c.group()), int(c.causal), int(c.d) * F::ES,
              uint32_t((65536 + c.group() - 1) / c.group()), kLog2e / sqrtf(float(c.d)), 1.f / sqrtf(float(c.d))};
    constexpr int RB = D * F::ES;
    const int64_t cus = device_cus(stream);
    hipError_t e;
    const bool few_q = short_of_work(c, (c.host->max_len + 63) / 64, 128 * 64, 2 * cus);
    if constexpr (RB > 256) e = few_q ? dq_as<F, D, PAD, Waves<2, 2, 1>>(c, a, stream) : dq_as<F, D, PAD, Waves<4, 1, 1>>(c, a, stream);
    else e = few_q ? dq_as<F, D, PAD, Waves<1, 4, 1>>(c, a, stream) : dq_as<F, D, PAD, Waves<4, 1, 1>>(c, a, stream);
    if (e != hipSuccess) return e;
    // A workgroup of 128 keys walks its first key's rows in blocks of 64; up to 80 KiB of LDS two share a CU.
    const int64_t walk = (c.host->max_len * c.group() + 63) / 64, slots = RB <= 128 ? 2 * cus : cus;
    if constexpr (RB > 256) return dkdv_as<F, D, PAD, KvWaves<2, 2, 1>>(c, a, stream);
    else if constexpr (F::ES == 4) return short_of_work(c, walk, 128 * 64, slots) ? dkdv_as<F, D, PAD, KvWaves<1, 4, 1>>(c, a, stream) : dkdv_as<F, D, PAD, KvWaves<4, 2, 2>>(c, a, stream);
    else if constexpr (RB <= 128) return short_of_work(c, walk, 128 * 64, slots) ? dkdv_as<F, D, PAD, KvWaves<1, 4, 2>>(c, a, stream) : dkdv_as<F, D, PAD, KvWaves<4, 2, 2>>(c, a, stream);
    else return short_of_work(c, walk, 128 * 64, slots, 8) ? dkdv_as<F, D, PAD, KvWaves<1, 8, 1>>(c, a, stream) : dkdv_as<F, D, PAD, KvWaves<4, 2, 2>>(c, a, stream);
}

// The tile width: the next of 32, 64, 128 elements at or above d, rows of another length padded with zeros.
template <typename F, typename Fn> hipError_t by_width(const PackedCall &c, Fn fn) {
    if (c.d <= 32) return c.d == 32 ? fn.template operator()<F, 32, false>() : fn.template operator()<F, 32, true>();
    if (c.d <= 64) return c.d == 64 ? fn.template operator()<F, 64, false>() : fn.template operator()<F, 64, true>();
    return c.d == 128 ? fn.template operator()<F, 128, false>() : fn.template operator()<F, 128, true>();
}

struct FwdCall {
    const PackedCall &c;
    const void *q, *k, *v;
    void *o;
    float *lse;
    hipStream_t stream;
    template <typename F, int D, bool PAD> hipError_t operator()() const {
        return run_fwd<F, D, PAD>(c, q, k, v, o, lse, stream);
    }
};
struct BwdCall {
    const PackedCall &c;
    const void *q, *k, *v, *o, *dout;
    const float *lse;
    float *ws;
    void *dq, *dk, *dv;
    hipStream_t stream;
    template <typename F, int D, bool PAD> hipError_t operator()() const {
        return run_bwd<F, D, PAD>(c, q, k, v, o, dout, lse, ws, dq, dk, dv, stream);
    }
};

}  // namespace

bool packed_mfma_supported(int dtype, int64_t d, int64_t group) {
    if (dtype != 0 && dtype != 1 && dtype != 2) return false;
    return d >= 1 && d <= 128 && d % (dtype == 0 ? 4 : 8) == 0 && group <= kMfmaMaxGroup;
}

int64_t packed_bwd_scratch_bytes(const PackedCall &c) { return c.tokens() * c.hq * 2 * int64_t(sizeof(float)); }

hipError_t launch_packed_fwd(const PackedCall &c, const void *q, const void *k, const void *v, void *o, float *lse,
                             hipStream_t stream) {
    const FwdCall f{c, q, k, v, o, lse, stream};
    return c.dtype == 0 ? by_width<PF32>(c, f) : c.dtype == 1 ? by_width<PBf16>(c, f) : by_width<PF16>(c, f);
}

hipError_t launch_packed_bwd(const PackedCall &c, const void *q, const void *k, const void *v, const void *o,
                             const void *dout, const float *lse, void *scratch, void *dq, void *dk, void *dv,
                             hipStream_t stream) {
    const BwdCall f{c, q, k, v, o, dout, lse, static_cast<float *>(scratch), dq, dk, dv, stream};
    return c.dtype == 0 ? by_width<PF32>(c, f) : c.dtype == 1 ? by_width<PBf16>(c, f) : by_width<PF16>(c, f);
}

}  // namespace ctattn
