// Attention on packed sequences with shared key heads on MFMA: bf16 and fp16 (32x32x16), fp32
// (32x32x2), fp32 accumulation, head dims that are whole 16-byte chunks up to 128.
//
// Forward: O = softmax(Q K^T / sqrt(d)) V within each sequence, L = log of the row's sum.  A
// workgroup of 4 waves owns 128 rows of (token, head of the group) of one key head, wave w rows
// 32 w .., and walks the sequence's keys in blocks of 64 through LDS (direct global -> LDS loads,
// two buffers).  Scores are computed transposed, S^T = K Q^T, so that a lane holds one row: the
// running maximum and sum of the softmax need one exchange with lane ^ 32, and the accumulator
// registers are, as they stand, the B operand of O^T += V^T P^T.  The maximum is raised only when
// a block exceeds it by 2^8 (P stays below 2^8, exact to scale in fp32 sums).  P is rounded to 16
// bits for the second product (the MFMA's operand type); the sum adds the unrounded values.
//
// Backward: P = exp(S - L), dV = P^T dO, dS = P (dO V^T - delta), dQ = dS K, dK = dS^T Q, in two
// kernels without atomics: one walks rows for a block of keys (dK, dV; the rows of all heads of
// the group, so that the sum over the heads that share a key head is one more stretch of the
// same contraction), one walks keys for a block of rows (dQ).  S and dP are computed in both: the
// alternative, dQ by atomics, is bound by their rate and not reproducible.
#include "attn_launch.h"
#include "attn_packed.h"
#include "attn_packed_tiles.h"

#include <math.h>

#include <type_traits>

namespace ctattn {
namespace {

using namespace packedtile;

constexpr float kRaise = 8.0f;       // raise the running maximum when a block exceeds it by 2^8
constexpr float kPsumLimit = 256.f;  // a lane's share of a block's P below which no P exceeds 2^8

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

template <typename F, int D> struct FwdCfg {
    static constexpr int NW = 4;
    static constexpr int BM = 32 * NW;
    static constexpr int BN = 64;
    static constexpr int KT = BN / 32;
    static constexpr int DT = D / 32;
    static constexpr int RB = D * F::ES;
    static constexpr int STEPS = RB / 32;
    static constexpr int KB = BN * RB;
    static constexpr int LDS = 4 * KB;  // buffer b: K at 2 b KB, V behind it
    static constexpr int WPE = LDS > 80 * 1024 ? 1 : 2;
};

template <typename F, int D, bool PAD>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(FwdCfg<F, D>::WPE, 2))) void packed_fwd_kernel(
    FwdArgs a) {
    using C = FwdCfg<F, D>;
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
    const int r0 = it.tile * C::BM;
    const int row = r0 + 32 * wave + col;
    const int token = row / a.group, head = kvh * a.group + row % a.group;
    const int first_token = (r0 + 32 * wave) / a.group;  // of this wave
    const int last_token = min((r0 + 32 * wave + 31) / a.group, it.len - 1);
    const bool wave_rows = r0 + 32 * wave < rows;

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
    float m_run = -INFINITY, l_run = 0.f;

    const uint32_t rk = uint32_t(Tile<C::RB / 2>::off(col, half));
    const uint32_t cv0 = F::template col0<C::RB>(lane), cv1 = F::template col1<C::RB>(lane);

    const char *kb0 = a.k.at(it.start, kvh), *vb0 = a.v.at(it.start, kvh);
    const int kend = a.causal ? min(it.len, (min(r0 + C::BM, rows) - 1) / a.group + 1) : it.len;
    const int nkb = (kend + C::BN - 1) / C::BN;
    auto issue = [&](int kb) __attribute__((always_inline)) {
        const uint32_t t = L + uint32_t((kb & 1) * 2 * C::KB);
        const int j0 = kb * C::BN;
        load_rows<C::RB, C::BN, C::NW, PAD>(t, kb0 + j0 * a.k.row, a.k.row, a.width, it.len - j0, wave, lane);
        load_rows<C::RB, C::BN, C::NW, PAD>(t + C::KB, vb0 + j0 * a.v.row, a.v.row, a.width, it.len - j0, wave, lane);
    };
    // One 64-key block.  MASK: it crosses the wave's diagonal or the sequence's end.
    auto block = [&](auto mask, int kb) __attribute__((always_inline)) {
        constexpr bool MASK = decltype(mask)::value;
        const int j0 = kb * C::BN;
        const uint32_t kt0 = L + uint32_t((kb & 1) * 2 * C::KB);
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
        if (__any(!(psum <= kPsumLimit))) {
            float top = -INFINITY;
#pragma unroll
            for (int kt = 0; kt < C::KT; ++kt) {
                if (!active[kt]) continue;
#pragma unroll
                for (int r = 0; r < 16; ++r) top = fmaxf(top, sacc[kt][r]);
            }
            top = max_xor32(top) * a.c;
            if (__any(top > m_run + kRaise)) {
                // Key 0 is in every row's mask and in its first block, so m is finite from there on.
                const float m_new = fmaxf(m_run, top);
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
        // This wave's loads of the block have landed; after the barrier every wave's have, and
        // every wave is done reading the other buffer.
        wait_loads();
        lds_barrier();
        if (kb + 1 < nkb) issue(kb + 1);
    };
    // This wave's blocks, in loops without branches inside (one loop over both variants makes the
    // compiler copy the accumulators): [0, jp) whole, [jp, jw) across the diagonal or the end,
    // [jw, nkb) none of its pairs.
    const int jw = !wave_rows ? 0 : a.causal ? last_token / C::BN + 1 : nkb;
    const int jp = min(jw, min(it.len, a.causal ? first_token + 1 : it.len) / C::BN);
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

// -delta = -rowsum(dO O) and -L log2(e) of every (token, head), laid out as the kernels walk them: rows
// (token, head of the group) behind each other for each key head.  16 lanes a row.
template <typename F>
__global__ __launch_bounds__(256) void packed_rowstats_kernel(View o, View dout, const float *__restrict__ lse,
                                                             float *__restrict__ ndelta, float *__restrict__ nl2,
                                                             int64_t rows, int64_t tokens, int hkv, int group,
                                                             int width) {
    using V = typename F::store;
    constexpr int EC = 16 / F::ES;
    typedef V vecv __attribute__((ext_vector_type(EC)));
    const int hq = hkv * group;
    const int64_t stride = int64_t(gridDim.x) * blockDim.x;
    for (int64_t t = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; t / 16 < rows; t += stride) {
        const int64_t row = t / 16, n = row / hq;
        const int h = int(row % hq);
        float s = 0.f;
        for (int c = 16 * int(t % 16); c < width; c += 256) {
            const vecv x = *reinterpret_cast<const vecv *>(o.at(n, h) + c);
            const vecv y = *reinterpret_cast<const vecv *>(dout.at(n, h) + c);
#pragma unroll
            for (int e = 0; e < EC; ++e) s += F::widen(x[e]) * F::widen(y[e]);
        }
        s = group_sum<16>(s);
        if (t % 16 == 0) {
            const int64_t at = (int64_t(h / group) * tokens + n) * group + h % group;
            ndelta[at] = -s;
            nl2[at] = -lse[row] * kLog2e;
        }
    }
}

struct BwdArgs {
    View q, k, v, dout, dq, dk, dv;
    const float *ndelta, *nl2;
    const PackedItem *items;
    int64_t tokens;
    int hkv, group, causal, width;
    uint32_t magic;  // ceil(65536 / group): x / group = x magic >> 16 for x < 64 + group, group <= 128
    float c, inv_sqrt_d;
};

template <typename F, int D> struct KvCfg {
    static constexpr int RB = D * F::ES;
    static constexpr bool WIDE = RB > 256;         // fp32 at D = 128: half the keys, one Q buffer
    static constexpr int KS = WIDE ? 2 : 4;        // key slices of 32
    static constexpr int NW = 2 * KS;              // x 2 row slices
    static constexpr int BN = 32 * KS;
    static constexpr int BM = 64;
    static constexpr int NBUF = WIDE ? 1 : 2;
    static constexpr int DT = D / 32;
    static constexpr int STEPS = RB / 32;
    static constexpr int QB = BM * RB;             // Q (or dO) tile
    static constexpr int KB = BN * RB;
    static constexpr int K_OFF = NBUF * 2 * QB;    // buffer b: Q at 2 b QB, dO behind it
    static constexpr int V_OFF = K_OFF + KB;
    static constexpr int S_OFF = V_OFF + KB;       // buffer b: nl2[BM], ndelta[BM]
    static constexpr int LDS = S_OFF + NBUF * 2 * BM * 4;
    static constexpr int WPE = WIDE ? 1 : 2;
    static constexpr PackedTile KIND = WIDE ? kKeys64 : kKeys128;
    static_assert(KS * DT * 2 * 16 * kWave * 4 <= LDS, "reduction buffer");
};

template <typename F, int D, bool PAD>
__global__ __launch_bounds__((64 * KvCfg<F, D>::NW)) __attribute__((amdgpu_waves_per_eu(KvCfg<F, D>::WPE, 2))) void
packed_dkdv_kernel(BwdArgs a) {
    using C = KvCfg<F, D>;
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

    load_rows<C::RB, C::BN, C::NW, PAD>(L + C::K_OFF, a.k.at(it.start + k0, kvh), a.k.row, a.width, it.len - k0, wave,
                                        lane);
    load_rows<C::RB, C::BN, C::NW, PAD>(L + C::V_OFF, a.v.at(it.start + k0, kvh), a.v.row, a.width, it.len - k0, wave,
                                        lane);
    floatx16 dk[C::DT], dv[C::DT];
#pragma unroll
    for (int dt = 0; dt < C::DT; ++dt) dk[dt] = zero16(), dv[dt] = zero16();

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
        if (wave >= C::NW - 2) {
            const bool is_nl = wave == C::NW - 2;
            load_dword_dma((is_nl ? a.nl2 : a.ndelta) + sbase + min(r0 + lane, rows - 1),
                           L + C::S_OFF + uint32_t(buf * 2 * C::BM * 4 + (is_nl ? 0 : C::BM * 4)));
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
            k[0] = lds_b128<V>(ak);
            g[0] = lds_b128<V>(aq + C::QB);
            v[0] = lds_b128<V>(ak + C::KB);
#pragma unroll
            for (int st = 0; st < C::STEPS; ++st) {
                const int cur = st & 1, nxt = cur ^ 1;
                if (st + 1 < C::STEPS) {
                    const uint32_t xq = aq ^ uint32_t((st + 1) << 5), xk = ak ^ uint32_t((st + 1) << 5);
                    q[nxt] = lds_b128<V>(xq);
                    k[nxt] = lds_b128<V>(xk);
                    g[nxt] = lds_b128<V>(xq + C::QB);
                    v[nxt] = lds_b128<V>(xk + C::KB);
                }
                read_fence();
                s = F::mma(q[cur], k[cur], s);
                dp = F::mma(g[cur], v[cur], dp);
            }
        }
        typename F::pvec pb[2], db[2];
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
                F::put(db[r / 8], r % 8, ds);
            }
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

    auto step = [&](int qb) __attribute__((always_inline)) {
        const int buf = C::NBUF == 2 ? (qb - qb_first) & 1 : 0;
        if (C::NBUF == 1) {
            lds_barrier();  // every wave is done with the last block
            issue(qb, 0);
        }
        wait_loads();
        lds_barrier();
        if (C::NBUF == 2 && qb + 1 < nqb) issue(qb + 1, buf ^ 1);
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
    if (C::NBUF == 2) issue(qb_first, 0);  // the tile's first key is in the sequence: qb_first < nqb
    int qb = qb_first;
    for (; qb < qa; ++qb) step(qb);
    for (; qb < qp; ++qb) {
        const int buf = step(qb);
        block(std::true_type{}, qb * C::BM + 32 * rs, buf);
    }
    for (; qb < qe; ++qb) {
        const int buf = step(qb);
        block(std::false_type{}, qb * C::BM + 32 * rs, buf);
    }
    for (; qb < qn; ++qb) {
        const int buf = step(qb);
        block(std::true_type{}, qb * C::BM + 32 * rs, buf);
    }
    for (; qb < nqb; ++qb) step(qb);

    // The second row slice's sums join the first's through LDS.
    float *red = reinterpret_cast<float *>(smem);
    __syncthreads();
    if (rs == 1) {
#pragma unroll
        for (int dt = 0; dt < C::DT; ++dt)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                red[(((ks * C::DT + dt) * 2 + 0) * 16 + r) * kWave + lane] = dk[dt][r];
                red[(((ks * C::DT + dt) * 2 + 1) * 16 + r) * kWave + lane] = dv[dt][r];
            }
    }
    __syncthreads();
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
                    const int r = 4 * g + t;
                    xk[t] = (dk[dt][r] + red[(((ks * C::DT + dt) * 2 + 0) * 16 + r) * kWave + lane]) * a.inv_sqrt_d;
                    xv[t] = dv[dt][r] + red[(((ks * C::DT + dt) * 2 + 1) * 16 + r) * kWave + lane];
                }
                store4<F>(dkr + 32 * dt + 8 * g + 4 * half, xk);
                store4<F>(dvr + 32 * dt + 8 * g + 4 * half, xv);
            }
        }
    }
}

template <typename F, int D> struct QCfg {
    static constexpr int NW = 4;
    static constexpr int BM = 32 * NW;
    static constexpr int BN = 32;
    static constexpr int RB = D * F::ES;
    static constexpr int DT = D / 32;
    static constexpr int STEPS = RB / 32;
    static constexpr int KB = BN * RB;
    static constexpr int LDS = 4 * KB;
    static constexpr int WPE = RB > 256 ? 1 : 2;
};

template <typename F, int D, bool PAD>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(QCfg<F, D>::WPE, 2))) void packed_dq_kernel(
    BwdArgs a) {
    using C = QCfg<F, D>;
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
    const int r0 = it.tile * C::BM;
    const int r0w = r0 + 32 * wave;
    const int row = r0w + col;
    const int token = row / a.group, head = kvh * a.group + row % a.group;
    const int first_token = r0w / a.group;
    const int last_token = min((r0w + 31) / a.group, it.len - 1);

    V qb[C::STEPS], gb[C::STEPS];
    {
        const char *pq = a.q.at(it.start + token, head), *pg = a.dout.at(it.start + token, head);
#pragma unroll
        for (int s = 0; s < C::STEPS; ++s) {
            floatx4 x = {0.f, 0.f, 0.f, 0.f}, y = {0.f, 0.f, 0.f, 0.f};
            if (row < rows && (!PAD || 32 * s + 16 * half < a.width)) {
                x = *reinterpret_cast<const floatx4 *>(pq + 32 * s + 16 * half);
                y = *reinterpret_cast<const floatx4 *>(pg + 32 * s + 16 * half);
            }
            qb[s] = __builtin_bit_cast(V, x);
            gb[s] = __builtin_bit_cast(V, y);
        }
    }
    const int64_t sbase = (int64_t(kvh) * a.tokens + it.start) * a.group;
    const float nl = row < rows ? a.nl2[sbase + row] : 0.f;
    const float nd = row < rows ? a.ndelta[sbase + row] : 0.f;
    floatx16 dq[C::DT];
#pragma unroll
    for (int dt = 0; dt < C::DT; ++dt) dq[dt] = zero16();

    const uint32_t rk = uint32_t(Tile<C::RB / 2>::off(col, half));
    const uint32_t ck0 = F::template col0<C::RB>(lane), ck1 = F::template col1<C::RB>(lane);
    const char *kb0 = a.k.at(it.start, kvh), *vb0 = a.v.at(it.start, kvh);
    const int kend = a.causal ? min(it.len, (min(r0 + C::BM, rows) - 1) / a.group + 1) : it.len;
    const int nkb = (kend + C::BN - 1) / C::BN;
    auto issue = [&](int kb) __attribute__((always_inline)) {
        const uint32_t t = L + uint32_t((kb & 1) * 2 * C::KB);
        const int j0 = kb * C::BN;
        load_rows<C::RB, C::BN, C::NW, PAD>(t, kb0 + j0 * a.k.row, a.k.row, a.width, it.len - j0, wave, lane);
        load_rows<C::RB, C::BN, C::NW, PAD>(t + C::KB, vb0 + j0 * a.v.row, a.v.row, a.width, it.len - j0, wave, lane);
    };
    auto block = [&](auto mask, int kb) __attribute__((always_inline)) {
        constexpr bool MASK = decltype(mask)::value;
        const uint32_t kt = L + uint32_t((kb & 1) * 2 * C::KB);
        floatx16 s = zero16(), dp;
#pragma unroll
        for (int r = 0; r < 16; ++r) dp[r] = nd;
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
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            float ds = fast_exp2(fmaf(s[r], a.c, nl)) * dp[r];
            if (MASK) {
                const int key = kb * C::BN + acc_row(r, half);
                ds = (key >= it.len || (a.causal && key > token)) ? 0.f : ds;
            }
            F::put(db[r / 8], r % 8, ds);
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
        wait_loads();
        lds_barrier();
        if (kb + 1 < nkb) issue(kb + 1);
    };
    // As in the forward; rows past the last one have P = exp2(0 + 0) dP = 0, so they need no mask.
    const int jw = r0w >= rows ? 0 : a.causal ? last_token / C::BN + 1 : nkb;
    const int jp = min(jw, min(it.len, a.causal ? first_token + 1 : it.len) / C::BN);
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

View view(const void *p, const PackedStride &s, int es) {
    return {static_cast<char *>(const_cast<void *>(p)), s.row * es, s.head * es};
}

template <typename F, int D, bool PAD>
hipError_t run_fwd(const PackedCall &c, const void *q, const void *k, const void *v, void *o, float *lse,
                   hipStream_t stream) {
    const int64_t blocks = c.item_count(kRows128) * c.hkv;
    if (!grid_fits(blocks, 256)) return hipErrorInvalidValue;
    FwdArgs a{view(q, c.sq, F::ES), view(k, c.sk, F::ES), view(v, c.sv, F::ES), view(o, c.so, F::ES), lse,
              c.items(kRows128), int(c.hkv), int(c.group()), int(c.causal), int(c.d) * F::ES,
              kLog2e / sqrtf(float(c.d))};
    hipLaunchKernelGGL((packed_fwd_kernel<F, D, PAD>), dim3(unsigned(blocks)), dim3(256), 0, stream, a);
    return hipGetLastError();
}

template <typename F, int D, bool PAD>
hipError_t run_bwd(const PackedCall &c, const void *q, const void *k, const void *v, const void *o, const void *dout,
                   const float *lse, float *ws, void *dq, void *dk, void *dv, hipStream_t stream) {
    using KC = KvCfg<F, D>;
    const int64_t rows = c.tokens() * c.hq;
    const int64_t kv_blocks = c.item_count(KC::KIND) * c.hkv, q_blocks = c.item_count(kRows128) * c.hkv;
    if (!grid_fits(kv_blocks, 64 * KC::NW) || !grid_fits(q_blocks, 256)) return hipErrorInvalidValue;
    BwdArgs a{view(q, c.sq, F::ES), view(k, c.sk, F::ES), view(v, c.sv, F::ES), view(dout, c.sdo, F::ES),
              view(dq, c.sdq, F::ES), view(dk, c.sdk, F::ES), view(dv, c.sdv, F::ES), ws, ws + rows,
              c.items(KC::KIND), c.tokens(), int(c.hkv), int(c.group()), int(c.causal), int(c.d) * F::ES,
              uint32_t((65536 + c.group() - 1) / c.group()), kLog2e / sqrtf(float(c.d)), 1.f / sqrtf(float(c.d))};
    hipLaunchKernelGGL((packed_rowstats_kernel<F>), dim3(stride_grid((rows * 16 + 255) / 256, 256)), dim3(256), 0,
                       stream, view(o, c.so, F::ES), a.dout, lse, ws, ws + rows, rows, c.tokens(), int(c.hkv),
                       int(c.group()), a.width);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((packed_dkdv_kernel<F, D, PAD>), dim3(unsigned(kv_blocks)), dim3(64 * KC::NW), 0, stream, a);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    a.items = c.items(kRows128);
    hipLaunchKernelGGL((packed_dq_kernel<F, D, PAD>), dim3(unsigned(q_blocks)), dim3(256), 0, stream, a);
    return hipGetLastError();
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
    return d >= 1 && d <= 128 && d % (dtype == 0 ? 4 : 8) == 0 && group <= 128;
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
