// Attention of requests that share a prompt, keys and values in a paged cache, on MFMA: bf16 and fp16
// (32x32x16), fp32 (32x32x2), fp32 accumulation, head dims that are whole 16-byte chunks up to 128.
//
// O = softmax(q K^T / sqrt(d)) V over the prompt's keys and the request's own.  A softmax over two sets of
// keys is the two softmaxes joined by weights exp(m_s - max m), so the sets are worked on apart.  The rows
// (request, token, head of the group) of a whole group of requests and one key head are one matrix beside the
// prompt: a workgroup takes 128 (or 32) of them and a stretch of the prompt's keys, which it reads once for all of
// them.  A request's own keys are walked beside its own rows alone.  Both split long stretches of keys over
// workgroups; every workgroup leaves O (not yet divided), m and l in fp32 in the workspace, and a second launch joins
// them.
//
// The walk itself is that of the packed attention forward: 4 waves, S^T = K Q^T so that a lane holds one row,
// P in the accumulators' own order as operand of O^T += V^T P^T, the maximum raised only when a block exceeds it
// by 2^8 (fp16 2^15), two LDS buffers filled by direct global -> LDS loads.  Loads find their rows through the page
// table: where a load instruction's rows lie in one page (pages of at least 64 rows / (16-byte chunks a row)), the page
// is looked up once a wave a block ahead, and the load takes it as a scalar base with fixed lane offsets; smaller pages and the
// last block look up every lane's row.  P is rounded to 16 bits for the second product (the MFMA's operand type); l
// adds the unrounded values.
#include "attn_launch.h"
#include "attn_packed_tiles.h"
#include "attn_shared.h"

#include <algorithm>

#include <math.h>

#include <type_traits>

namespace ctattn {
namespace {

using namespace packedtile;

constexpr float kLowest = -3.402823466e38f;  // the running maximum before any score (finite: m - m is 0, not NaN)

// When the running maximum rises, and to where: as in attn_packed.hip, fp16 holds it 2^7 below the row's so
// that P fills the format.
template <typename F> struct Rise {
    static constexpr float UNDER = F::RANGE ? 7.f : 0.f;
    static constexpr float BY = F::RANGE ? 15.f : 8.f;
    static constexpr float PSUM = F::RANGE ? 32768.f : 256.f;
};

// Byte strides and pointers.
struct View {
    char *p;
    int64_t row, head;
    __device__ char *at(int64_t n, int h) const { return p + n * row + h * head; }
};
struct CacheView {
    const char *p;
    int64_t page, token, head;
};

struct Args {
    SharedLayout lay;
    View q, o;
    CacheView k, v;
    float *po;   // [splits][rows][hq][dp], O before the division
    float *ml;   // [splits][rows][hq][2], m (in powers of two) and l
    float *lse;
    int dp;      // d in whole tiles of 32
    int width;   // bytes of d elements
    int fill;
    int one_page;  // a load instruction's rows lie in one page, both caches at equal token strides
    int ptiles, psplits, otiles, osplits;
    float c;     // log2(e) / sqrt(d)
};

// How a workgroup's 4 waves share its work: RS slices of 32 rows x KS slices of 32 KT keys of every block.
template <int RS_, int KS_, int KT_> struct Waves {
    static constexpr int RS = RS_, KS = KS_, KT = KT_;
    static_assert(RS * KS == 4, "4 waves");
};
template <typename F, int D, typename W> struct Cfg : W {
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
    using L = Tile<RB / 2>;
    static constexpr int RPL = kWave / L::CH;        // rows of one load instruction
    static constexpr int NL = BN / (NW * RPL);       // load instructions of a wave a tile
    static_assert(kWave % L::CH == 0 && BN % (NW * RPL) == 0, "tile loads");
};

// What a workgroup works on: rows (token, head of the group) r0 .. of `tokens` tokens from row `first` on, keys
// k0 .. k1 - 1 of a page table; token t sees keys below min(len, off + t + 1).
struct Item {
    int first, tokens, r0;
    int len, off, k0, k1;
    const int32_t *pages;
    int split;
};

__device__ __forceinline__ void stretch(Item &it, int part, int parts, int block) {
    const int each = ((it.len + parts - 1) / parts + block - 1) / block * block;
    const int64_t k0 = int64_t(part) * each;
    it.k0 = k0 < it.len ? int(k0) : it.len;
    it.k1 = it.len - it.k0 > each ? it.k0 + each : it.len;
}

// Tiles of a list of row ranges [row(i), row(i + 1)) have places of their own without a scan: range i's begin at
// floor(row(i) G / BM) + i, and up to the next range's there are at least as many as it has tiles.
template <typename Row> __device__ __forceinline__ int range_of(int n, int slot, int group, int bm, Row row) {
    int lo = 0;
    for (int hi = n - 1; lo < hi;) {
        const int mid = (lo + hi + 1) / 2;
        if (row(mid) * group / bm + mid <= slot) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}
template <int BM, int BN> __device__ __forceinline__ bool prefix_item(const Args &a, int slot, int part, Item &it) {
    const SharedLayout &y = a.lay;
    const auto row = [&](int g) { return y.group_row(g); };
    const int g = range_of(y.groups, slot, y.group, BM, row);
    it.first = row(g);
    it.tokens = row(g + 1) - it.first;
    it.r0 = (slot - (it.first * y.group / BM + g)) * BM;
    it.len = y.prefix_len(g);
    it.off = it.len;
    it.pages = y.prefix_table + g * y.prefix_row;
    it.split = part;
    stretch(it, part, a.psplits, BN);
    return it.r0 >= 0 && it.r0 < it.tokens * y.group;
}
template <int BM, int BN> __device__ __forceinline__ bool own_item(const Args &a, int slot, int part, Item &it) {
    const SharedLayout &y = a.lay;
    const auto row = [&](int i) { return y.first_row(i); };
    const int i = range_of(y.requests, slot, y.group, BM, row);
    it.first = row(i);
    it.tokens = row(i + 1) - it.first;
    it.r0 = (slot - (it.first * y.group / BM + i)) * BM;
    it.len = y.own_len(i);
    it.off = it.len - it.tokens;
    it.pages = y.table + i * y.table_row;
    it.split = a.psplits + part;
    stretch(it, part, a.osplits, BN);
    return it.r0 >= 0 && it.r0 < it.tokens * y.group;
}

__device__ __forceinline__ void load_chunk_saddr(uint32_t off, uint64_t base, uint32_t dst) {
    const uint32_t lo = __builtin_amdgcn_readfirstlane(uint32_t(base));
    const uint32_t hi = __builtin_amdgcn_readfirstlane(uint32_t(base >> 32));
    const uint64_t b = uint64_t(hi) << 32 | lo;
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(b),
                 "s"(__builtin_amdgcn_readfirstlane(dst))
                 : "memory", "m0");
}

template <typename F, int D, bool PAD, typename W>
__device__ __forceinline__ void walk(const Args &a, const Item &it, const int kvh, char *smem) {
    using C = Cfg<F, D, W>;
    using T = typename C::L;
    using V = typename F::vec;
    const uint32_t L = lds_addr(smem);
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int col = lane & 31, half = lane >> 5;
    const int group = a.lay.group;
    const int rows = it.tokens * group;
    const int rs = wave % C::RS, ks = wave / C::RS;
    const int r0w = it.r0 + 32 * rs;
    const int row = r0w + col;
    const int token = row / group, head = kvh * group + row % group;
    const int koff = 32 * C::KT * ks;
    // Keys from k0 on that a token sees.
    const auto seen = [&](int t) { return max(min(it.k1, it.off >= it.len ? it.len : it.off + t + 1) - it.k0, 0); };
    const int row_end = seen(token);
    const int whole = seen(r0w / group);  // every row of the wave
    const int some = seen(min((r0w + 31) / group, it.tokens - 1));  // any of them
    const int kend = seen((min(it.r0 + C::BM, rows) - 1) / group);  // any of the workgroup
    const int nkb = (kend + C::BN - 1) / C::BN;

    V qb[C::STEPS];
    {
        const char *p = a.q.at(it.first + token, head);
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

    const uint32_t rk = uint32_t(T::off(col, half));
    const uint32_t cv0 = F::template col0<C::RB>(lane), cv1 = F::template col1<C::RB>(lane);

    // Loads.  Instruction i of a wave fills rows RPL (wave NL + i) .. of the tile; a lane its chunk of one of them.
    const int lr = lane / T::CH;
    const int shift = a.lay.shift, in_page = (1 << shift) - 1;
    const char *kbase = a.k.p + kvh * a.k.head, *vbase = a.v.p + kvh * a.v.head;
    const auto chunk = [&](int i) { return 16 * ((lane % T::CH) ^ T::swz(C::RPL * (wave * C::NL + i) + lr)); };
    int page[C::NL];
    const auto look_up = [&](int kb) __attribute__((always_inline)) {
        // Past the end the last key's page: no place of the table is read that its length does not cover.
        if (!a.one_page) return;
#pragma unroll
        for (int i = 0; i < C::NL; ++i) {
            const int key = min(it.k0 + kb * C::BN + C::RPL * (wave * C::NL + i), it.k0 + kend - 1);
            page[i] = a.lay.page_at(it.pages, key);
        }
    };
    const auto issue = [&](int kb) __attribute__((always_inline)) {
        const uint32_t t = L + uint32_t((kb % C::NBUF) * 2 * C::KB);
        const int j0 = kb * C::BN;
        if (a.one_page && j0 + C::BN <= kend) {
#pragma unroll
            for (int i = 0; i < C::NL; ++i) {
                const int first = C::RPL * (wave * C::NL + i);
                const int64_t in = (it.k0 + j0 + first) & in_page;
                const uint32_t dst = t + uint32_t(first * C::RB);
                const uint32_t off = uint32_t(lr * int(a.k.token) + chunk(i));
                if (!PAD || chunk(i) < a.width) {
                    load_chunk_saddr(off, uint64_t(kbase) + uint64_t(int64_t(page[i]) * a.k.page + in * a.k.token), dst);
                    load_chunk_saddr(off, uint64_t(vbase) + uint64_t(int64_t(page[i]) * a.v.page + in * a.v.token), dst + C::KB);
                }
            }
        } else {
            // Rows past the last key re-read it (their results are masked).
#pragma unroll
            for (int i = 0; i < C::NL; ++i) {
                const int first = C::RPL * (wave * C::NL + i);
                const int key = it.k0 + min(j0 + first + lr, kend - 1);
                const int64_t pg = a.lay.page_at(it.pages, key), in = key & in_page;
                const uint32_t dst = t + uint32_t(first * C::RB);
                if (!PAD || chunk(i) < a.width) {
                    load_chunk_dma(kbase + pg * a.k.page + in * a.k.token + chunk(i), dst);
                    load_chunk_dma(vbase + pg * a.v.page + in * a.v.token + chunk(i), dst + C::KB);
                }
            }
        }
    };
    // This wave's keys of a block.  MASK: some rows of the wave do not see some of them.
    auto block = [&](auto mask, int kb) __attribute__((always_inline)) {
        constexpr bool MASK = decltype(mask)::value;
        const int j0 = kb * C::BN + koff;
        const uint32_t kt0 = L + uint32_t((kb % C::NBUF) * 2 * C::KB) + uint32_t(koff * C::RB);
        bool active[C::KT];
        floatx16 sacc[C::KT];
#pragma unroll
        for (int kt = 0; kt < C::KT; ++kt) {
            const int t0 = j0 + 32 * kt;
            active[kt] = !MASK || t0 < some;
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
                for (int r = 0; r < 16; ++r)
                    if (t0 + acc_row(r, half) >= row_end) sacc[kt][r] = -INFINITY;
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
            if (kb + 1 < nkb) look_up(kb + 1);
        }
        // This wave's loads of the block have landed; after the barrier every wave's have, and
        // (two buffers) every wave is done reading the other one.
        wait_loads();
        lds_barrier();
        if (C::NBUF == 2 && kb + 1 < nkb) {
            issue(kb + 1);
            if (kb + 2 < nkb) look_up(kb + 2);
        }
    };
    if (PAD) {
        // Chunks past the head dim are zeros that no load overwrites.
        for (uint32_t x = threadIdx.x * 16; x < uint32_t(C::LDS); x += 256 * 16)
            *reinterpret_cast<floatx4 *>(smem + x) = floatx4{0.f, 0.f, 0.f, 0.f};
        lds_barrier();
    }
    if (nkb > 0) {
        look_up(0);
        issue(0);
        if (nkb > 1) look_up(1);
    }
    // This wave's blocks, in loops without branches inside: [0, jp) whole, [jp, jw) masked, [jw, nkb) none of its pairs.
    const int jw = r0w < rows && some > koff ? (some - koff + C::BN - 1) / C::BN : 0;
    const int jp = min(jw, whole >= koff + 32 * C::KT ? (whole - koff - 32 * C::KT) / C::BN + 1 : 0);
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
        // saw no key has the lowest m and l = 0.
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
    if (row >= rows) return;
    const int64_t at = (int64_t(it.split) * a.lay.rows + it.first + token) * (a.lay.hkv * group) + head;
    if (half == 0) *reinterpret_cast<float2 *>(a.ml + 2 * at) = float2{m_run, l_tot};
    if (row_end == 0) return;  // l = 0: nothing to join
    float *po = a.po + at * a.dp;
#pragma unroll
    for (int dt = 0; dt < C::DT; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            if (!PAD || (32 * dt + 8 * g + 4 * half) * F::ES < a.width)
                *reinterpret_cast<floatx4 *>(po + 32 * dt + 8 * g + 4 * half) =
                    floatx4{oacc[dt][4 * g], oacc[dt][4 * g + 1], oacc[dt][4 * g + 2], oacc[dt][4 * g + 3]};
}

template <typename F, int D, typename WP, typename WO> struct Both {
    static constexpr int LDS = Cfg<F, D, WP>::LDS > Cfg<F, D, WO>::LDS ? Cfg<F, D, WP>::LDS : Cfg<F, D, WO>::LDS;
    static constexpr int WPE = Cfg<F, D, WP>::RB > 256 || LDS > 80 * 1024 ? 1 : 2;
};

// Workgroups of the prompts' keys first, then those of the requests' own.
template <typename F, int D, bool PAD, typename WP, typename WO>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(Both<F, D, WP, WO>::WPE, 2))) void shared_kernel(
    Args a) {
    __shared__ __attribute__((aligned(1024))) char smem[Both<F, D, WP, WO>::LDS];
    const int hkv = a.lay.hkv;
    const int kvh = blockIdx.x % hkv;
    int slot = blockIdx.x / hkv;
    Item it;
    if (slot < a.ptiles * a.psplits) {
        if (!prefix_item<Cfg<F, D, WP>::BM, Cfg<F, D, WP>::BN>(a, slot % a.ptiles, slot / a.ptiles, it)) return;
        walk<F, D, PAD, WP>(a, it, kvh, smem);
    } else {
        slot -= a.ptiles * a.psplits;
        if (!own_item<Cfg<F, D, WO>::BM, Cfg<F, D, WO>::BN>(a, slot % a.otiles, slot / a.otiles, it)) return;
        walk<F, D, PAD, WO>(a, it, kvh, smem);
    }
}

// O = sum of 2^(m_s - m) O_s / sum of 2^(m_s - m) l_s over the splits s that saw a key.  A thread joins 4 elements of a row's
// head.
template <typename F> __global__ __launch_bounds__(256) void shared_join_kernel(Args a, int d) {
    using S = typename F::store;
    const SharedLayout &y = a.lay;
    const int per = (d + 3) / 4, hq = y.hkv * y.group;
    const int64_t t = int64_t(blockIdx.x) * 256 + threadIdx.x;
    const int64_t rh = t / per;
    const int c = int(t % per) * 4;
    if (rh >= int64_t(y.rows) * hq) return;
    const int n = int(rh / hq), h = int(rh % hq);
    const bool there = n >= y.first_row(0) && n < y.first_row(y.requests);
    if (!there && !a.fill) return;
    const bool prompt = there && a.psplits > 0 && n >= y.group_row(0) && n < y.group_row(y.groups);
    const int s0 = prompt ? 0 : a.psplits, s1 = there ? a.psplits + a.osplits : s0;
    const int64_t step = int64_t(y.rows) * hq;
    float m = kLowest;
    for (int s = s0; s < s1; ++s) {
        const float2 x = *reinterpret_cast<const float2 *>(a.ml + 2 * (s * step + rh));
        if (!(x.y == 0.f)) m = fmaxf(m, x.x);
    }
    float l = 0.f;
    floatx4 o = {0.f, 0.f, 0.f, 0.f};
    for (int s = s0; s < s1; ++s) {
        const float2 x = *reinterpret_cast<const float2 *>(a.ml + 2 * (s * step + rh));
        if (x.y == 0.f) continue;
        const float w = fast_exp2(x.x - m);
        l += w * x.y;
        o += w * *reinterpret_cast<const floatx4 *>(a.po + (s * step + rh) * a.dp + c);
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const float r[4] = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
    store4<F>(reinterpret_cast<S *>(a.o.at(n, h)) + c, r);
    if (a.lse != nullptr && c == 0) a.lse[rh] = l == 0.f ? -INFINITY : (m + __log2f(l)) * kLn2;
}

using Rows128 = Waves<4, 1, 2>;
using Rows32 = Waves<1, 4, 1>;

// Tiles and splits, from the call's shapes alone.
struct Plan {
    bool tall_prefix, tall_own;
    int ptiles, psplits, otiles, osplits;
};
Plan plan_of(const SharedCall &c) {
    Plan p{};
    const int64_t work_rows = c.rows * c.group();
    const auto tiles = [&](int64_t ranges, bool tall) { return int(work_rows / (tall ? 128 : 32) + ranges); };
    const auto splits = [&](int64_t tiles, int64_t keys, int64_t least) {
        const int64_t want = 512 / std::max<int64_t>(1, tiles * c.hkv);
        return int(std::max<int64_t>(1, std::min(want, keys / least)));
    };
    p.tall_own = work_rows > 32 * c.requests;
    p.tall_prefix = p.tall_own || (c.groups > 0 && work_rows > 32 * c.groups);
    p.otiles = c.requests > 0 ? tiles(c.requests, p.tall_own) : 0;
    p.osplits = splits(p.otiles, c.max_own(), 128);
    if (c.max_prefix() > 0) {
        p.ptiles = tiles(c.groups, p.tall_prefix);
        p.psplits = splits(p.ptiles, c.max_prefix(), 256);
    }
    return p;
}
int64_t up(int64_t x) { return (x + 255) / 256 * 256; }
int64_t dp_of(int64_t d) { return d <= 32 ? 32 : d <= 64 ? 64 : 128; }

template <typename F, int D, bool PAD> hipError_t launch_d(const Args &a, const Plan &p, hipStream_t stream) {
    const int64_t blocks = (int64_t(p.ptiles) * p.psplits + int64_t(p.otiles) * p.osplits) * a.lay.hkv;
    if (!grid_fits(blocks, 256)) return hipErrorInvalidValue;
    if (blocks > 0) {
        const dim3 grid(static_cast<unsigned>(blocks)), block(256);
        if (p.tall_own) shared_kernel<F, D, PAD, Rows128, Rows128><<<grid, block, 0, stream>>>(a);
        else if (p.tall_prefix) shared_kernel<F, D, PAD, Rows128, Rows32><<<grid, block, 0, stream>>>(a);
        else shared_kernel<F, D, PAD, Rows32, Rows32><<<grid, block, 0, stream>>>(a);
    }
    return hipGetLastError();
}

template <typename F> hipError_t launch_f(const SharedCall &c, void *workspace, hipStream_t stream) {
    const Plan p = plan_of(c);
    Args a{};
    const int64_t e = F::ES;
    a.lay = layout_of(c);
    a.q = {const_cast<char *>(static_cast<const char *>(c.q)), c.sq.row * e, c.sq.head * e};
    a.o = {static_cast<char *>(c.o), c.so.row * e, c.so.head * e};
    a.k = {static_cast<const char *>(c.k), c.sk.page * e, c.sk.token * e, c.sk.head * e};
    a.v = {static_cast<const char *>(c.v), c.sv.page * e, c.sv.token * e, c.sv.head * e};
    a.dp = int(dp_of(c.d));
    a.width = int(c.d * e);
    a.fill = c.fill ? 1 : 0;
    a.lse = static_cast<float *>(c.lse);
    const int64_t row_heads = (p.psplits + p.osplits) * c.rows * c.hq;
    a.po = static_cast<float *>(workspace);
    a.ml = a.po + up(row_heads * a.dp * 4) / 4;
    a.ptiles = p.ptiles;
    a.psplits = p.psplits;
    a.otiles = p.otiles;
    a.osplits = p.osplits;
    a.c = kLog2e / sqrtf(float(c.d));
    // Rows of a load instruction: 64 lanes of 16 bytes; lane offsets are 32 bits from the first of them.
    const int64_t rows_per_load = kWave * 16 / (a.dp * e);
    a.one_page = c.page_size >= rows_per_load && a.k.token == a.v.token && a.k.token >= 0 && a.k.token < (int64_t(1) << 26);
    hipError_t rc;
    if (a.dp == 32) rc = a.width == 32 * e ? launch_d<F, 32, false>(a, p, stream) : launch_d<F, 32, true>(a, p, stream);
    else if (a.dp == 64) rc = a.width == 64 * e ? launch_d<F, 64, false>(a, p, stream) : launch_d<F, 64, true>(a, p, stream);
    else rc = a.width == 128 * e ? launch_d<F, 128, false>(a, p, stream) : launch_d<F, 128, true>(a, p, stream);
    if (rc != hipSuccess) return rc;
    const int64_t threads = c.rows * c.hq * ((c.d + 3) / 4);
    const int64_t blocks = (threads + 255) / 256;
    if (!grid_fits(blocks, 256)) return hipErrorInvalidValue;
    shared_join_kernel<F><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(a, int(c.d));
    return hipGetLastError();
}

}  // namespace

bool shared_mfma_supported(int dtype, int64_t d, int64_t group) {
    const int64_t e = dtype == 0 ? 4 : 2;
    return dtype <= 2 && d <= 128 && (d * e) % 16 == 0 && group <= 128;
}

int64_t shared_workspace_bytes(const SharedCall &c) {
    const Plan p = plan_of(c);
    const int64_t row_heads = (p.psplits + p.osplits) * c.rows * c.hq;
    return up(row_heads * dp_of(c.d) * 4) + up(row_heads * 8);
}

hipError_t launch_shared(const SharedCall &c, void *workspace, hipStream_t stream) {
    switch (c.dtype) {
    case 0: return launch_f<PF32>(c, workspace, stream);
    case 1: return launch_f<PBf16>(c, workspace, stream);
    default: return launch_f<PF16>(c, workspace, stream);
    }
}

}  // namespace ctattn
