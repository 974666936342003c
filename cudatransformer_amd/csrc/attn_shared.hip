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
// The walk itself is that of the packed attention forward: S^T = K Q^T so that a lane holds one row, P in the
// accumulators' own order as operand of O^T += V^T P^T, the maximum raised only when a block exceeds it by 2^8 (fp16
// 2^15), tiles filled by direct global -> LDS loads.  128-row tiles are a workgroup's, whose 4 waves walk the same keys
// through two buffers; where rows are fewer a wave walks its own stretch of keys for 32 rows by itself, with no barrier, K of
// the next 32 keys on its way while it adds V of these.  (Four waves of a workgroup that walked a quarter each and joined
// in LDS: 226 us and 72 for the requests' own keys of the two cases below, waves apart 220 and 71.)  Loads find their
// rows through the page table: where a load instruction's rows lie in one page (pages of at least 64 rows / (16-byte chunks a
// row)), the page is a scalar load a block ahead, and the load takes it as scalar base with fixed lane offsets;
// smaller pages and a stretch's last block look up every lane's row.  P is rounded to 16 bits for the second product (the
// MFMA's operand type); l adds the unrounded values.
//
// Measured, bf16, 32/8 heads of 128, one token a request: 256 requests of 1 to 2048 own tokens on a prompt of 32768 keys
// 305 us (3.95 TB/s, 463 TFLOP/s, of a floor of 235 by bytes), their own keys alone 220 (4.9 TB/s, HBM), the prompt alone 175
// (786 TFLOP/s, 35 % of the matrix cores' cycles with the launch's ends in them); 8 prompts of up to 2000 keys, 16 requests of 1 to 1024
// each 80 us (4.07 TB/s, floor 64).  Deeper tile or operand prefetch changed neither (3 buffers of 64 keys, 4 and 5 of 32, 1 to 4 operands
// ahead: 175 to 205 us for the prompt).
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
    int one_page;  // a load instruction's rows lie in one page, and lane offsets in 32 bits
    int ptiles, psplits, otiles, osplits;
    int pper, oper;  // tiles of each group or request where all have as many, or 0
    int omost;       // keys of a request's own that a workgroup takes, or 0: equal stretches
    float c;         // log2(e) / sqrt(d)
};

// Rows of a tile: 128, of which each of a workgroup's 4 waves takes 32 and all walk the same keys (tall), or 32 of a wave by
// itself (flat).
template <typename F, int D> struct Base {
    static constexpr int NW = 4;
    static constexpr int DT = D / 32;
    static constexpr int RB = D * F::ES;
    static constexpr int STEPS = RB / 32;
    using L = Tile<RB / 2>;
    static constexpr int RPL = kWave / L::CH;  // rows of one load instruction
    static_assert(kWave % L::CH == 0, "tile loads");
};
template <typename F, int D> struct Tall : Base<F, D> {
    using B = Base<F, D>;
    static constexpr int BM = 128;
    static constexpr int KT = 2;
    static constexpr int BN = 32 * KT;
    static constexpr int KB = BN * B::RB;
    static constexpr int LDS = 4 * KB;  // two buffers of K with V behind it
    static constexpr int NL = BN / (B::NW * B::RPL);  // load instructions of a wave a tile
};
template <typename F, int D> struct Flat : Base<F, D> {
    using B = Base<F, D>;
    static constexpr int BM = 32;
    static constexpr int BN = 32;
    static constexpr int KB = 32 * B::RB;
    static constexpr int LDS = B::NW * 2 * KB;  // a wave's K with V behind it
    static constexpr int NL = 32 / B::RPL;
};

// What a workgroup works on: rows (token, head of the group) r0 .. of `tokens` tokens from row `first` on, keys
// k0 .. k1 - 1 of a page table; token t sees keys below min(len, off + t + 1).
struct Item {
    int first, tokens, r0;
    int len, off, k0, k1;
    const int32_t *pages;
    int split;
};

// Part `part` of its keys, in whole blocks: `most` keys each, or if that is 0 in `parts` equal stretches.
__device__ __forceinline__ void stretch(Item &it, int part, int parts, int most, int block) {
    const int each = most > 0 ? most : ((it.len + parts - 1) / parts + block - 1) / block * block;
    const int64_t k0 = int64_t(part) * each;
    it.k0 = k0 < it.len ? int(k0) : it.len;
    it.k1 = it.len - it.k0 > each ? it.k0 + each : it.len;
}

// Tiles of a list of row ranges [row(i), row(i + 1)).  Equal ranges of one row a request have as many tiles each
// (`per`).  Others have places of their own without a scan: range i's begin at floor(row(i) G / BM) + i, and up to
// the next range's there are at least as many as it has tiles.
template <typename Row> __device__ __forceinline__ int range_of(int n, int slot, int per, int group, int bm, Row row, int &tile) {
    if (per > 0) {
        tile = slot % per;
        return slot / per;
    }
    int lo = 0;
    for (int hi = n - 1; lo < hi;) {
        const int mid = (lo + hi + 1) / 2;
        if (row(mid) * group / bm + mid <= slot) lo = mid;
        else hi = mid - 1;
    }
    tile = slot - (row(lo) * group / bm + lo);
    return lo;
}
template <int BM, int BN> __device__ __forceinline__ bool prefix_item(const Args &a, int slot, int part, Item &it) {
    const SharedLayout &y = a.lay;
    const auto row = [&](int g) { return y.group_row(g); };
    int tile;
    const int g = range_of(y.groups, slot, a.pper, y.group, BM, row, tile);
    it.first = row(g);
    it.tokens = row(g + 1) - it.first;
    it.r0 = tile * BM;
    it.len = y.prefix_len(g);
    it.off = it.len;
    it.pages = y.prefix_table + g * y.prefix_row;
    it.split = part;
    stretch(it, part, a.psplits, 0, BN);
    return tile >= 0 && it.r0 < it.tokens * y.group;
}
template <int BM, int BN> __device__ __forceinline__ bool own_item(const Args &a, int slot, int part, Item &it) {
    const SharedLayout &y = a.lay;
    const auto row = [&](int i) { return y.first_row(i); };
    int tile;
    const int i = range_of(y.requests, slot, a.oper, y.group, BM, row, tile);
    it.first = row(i);
    it.tokens = row(i + 1) - it.first;
    it.r0 = tile * BM;
    it.len = y.own_len(i);
    it.off = it.len - it.tokens;
    it.pages = y.table + i * y.table_row;
    it.split = a.psplits + part;
    stretch(it, part, a.osplits, a.omost, BN);
    return tile >= 0 && it.r0 < it.tokens * y.group;
}

__device__ __forceinline__ void load_chunk_saddr(uint32_t off, uint64_t base, uint32_t dst) {
    const uint32_t lo = __builtin_amdgcn_readfirstlane(uint32_t(base));
    const uint32_t hi = __builtin_amdgcn_readfirstlane(uint32_t(base >> 32));
    const uint64_t b = uint64_t(hi) << 32 | lo;
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(b),
                 "s"(__builtin_amdgcn_readfirstlane(dst))
                 : "memory", "m0");
}

// A wave's 32 rows: query operands, O^T, and the running maximum and sum.
template <typename F, int D> struct WaveState {
    using B = Base<F, D>;
    typename F::vec qb[B::STEPS];
    floatx16 o[B::DT];
    float m = kLowest, l = 0.f;

    template <bool PAD> __device__ __forceinline__ void init(const char *p, bool there, int width, int half) {
#pragma unroll
        for (int s = 0; s < B::STEPS; ++s) {
            floatx4 x = {0.f, 0.f, 0.f, 0.f};
            if (there && (!PAD || 32 * s + 16 * half < width)) x = *reinterpret_cast<const floatx4 *>(p + 32 * s + 16 * half);
            qb[s] = __builtin_bit_cast(typename F::vec, x);
        }
#pragma unroll
        for (int dt = 0; dt < B::DT; ++dt) o[dt] = zero16();
    }
    // S^T of the 32 keys whose tile's row operands begin at ka.
    __device__ __forceinline__ floatx16 scores(uint32_t ka) const {
        using V = typename F::vec;
        floatx16 c = zero16();
        V x[2];
        x[0] = lds_b128<V>(ka);
#pragma unroll
        for (int s = 0; s < B::STEPS; ++s) {
            if (s + 1 < B::STEPS) x[(s + 1) & 1] = lds_b128<V>(ka ^ uint32_t((s + 1) << 5));
            read_fence();
            c = F::mma(x[s & 1], qb[s], c);
        }
        return c;
    }
    // P of KT tiles' scores, with the maximum raised where they pass it by far.
    template <int KT>
    __device__ __forceinline__ void softmax(const floatx16 (&c)[KT], const bool (&active)[KT], typename F::pvec (&pb)[KT][2], float scale) {
        float psum;
        auto expo = [&]() __attribute__((always_inline)) {
            psum = 0.f;
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
                if (!active[kt]) continue;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float p = fast_exp2(fmaf(c[kt][r], scale, -m));
                    psum += p;
                    F::put(pb[kt][r / 8], r % 8, p);
                }
            }
        };
        expo();
        if (__any(!(psum <= Rise<F>::PSUM))) {
            float top = -INFINITY;
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
                if (!active[kt]) continue;
#pragma unroll
                for (int r = 0; r < 16; ++r) top = fmaxf(top, c[kt][r]);
            }
            top = max_xor32(top) * scale;
            if (__any(top > m + Rise<F>::BY)) {
                const float m_new = fmaxf(m, top - Rise<F>::UNDER);
                const float resc = fast_exp2(m - m_new);
                m = m_new;
                l *= resc;
#pragma unroll
                for (int dt = 0; dt < B::DT; ++dt) o[dt] *= resc;
            }
            expo();
        }
        l += psum;
    }
    // O^T += V^T P^T of 32 keys whose column operands begin at v0, v1.
    __device__ __forceinline__ void add(uint32_t v0, uint32_t v1, const typename F::pvec (&pb)[2]) {
        constexpr int NS = 2 * B::DT;
        typename F::cols x[2];
        x[0] = F::template read_cols<B::RB>(v0, v1, 0, 0);
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            if (i + 1 < NS) x[(i + 1) & 1] = F::template read_cols<B::RB>(v0, v1, (i + 1) / B::DT, (i + 1) % B::DT);
            read_fence();
            o[i % B::DT] = F::col_mma(x[i & 1], pb[i / B::DT], o[i % B::DT]);
        }
    }
    // The row's part of the item's split: m and l, and O where a key was seen.
    template <bool PAD>
    __device__ __forceinline__ void leave(const Args &a, const Item &it, int token, int head, int half, bool saw) const {
        const float sum = l + __shfl_xor(l, 32, kWave);
        const int64_t at = (int64_t(it.split) * a.lay.rows + it.first + token) * (a.lay.hkv * a.lay.group) + head;
        if (half == 0) *reinterpret_cast<float2 *>(a.ml + 2 * at) = float2{m, sum};
        if (!saw) return;
        float *po = a.po + at * a.dp;
#pragma unroll
        for (int dt = 0; dt < B::DT; ++dt)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                if (!PAD || (32 * dt + 8 * g + 4 * half) * F::ES < a.width)
                    *reinterpret_cast<floatx4 *>(po + 32 * dt + 8 * g + 4 * half) =
                        floatx4{o[dt][4 * g], o[dt][4 * g + 1], o[dt][4 * g + 2], o[dt][4 * g + 3]};
    }
};

// Loads of NL instructions of RPL rows each, rows base(i) .. of a stretch of keys from k0 on; PAD: chunks past `width`
// bytes are left as they are (zeros).
template <typename B, int NL, bool PAD> struct PagedLoads {
    const Args &a;
    const Item &it;
    const char *k, *v;
    int row0, lane;  // the first instruction's first row in a block
    int page[NL];    // of the next block's rows, or the block's own lanes' pages at the end

    __device__ __forceinline__ PagedLoads(const Args &a_, const Item &it_, int kvh, int row0_, int lane_)
        : a(a_), it(it_), k(a_.k.p + kvh * a_.k.head), v(a_.v.p + kvh * a_.v.head), row0(row0_), lane(lane_) {}
    __device__ __forceinline__ int chunk(int i) const {
        return 16 * ((lane % B::L::CH) ^ B::L::swz(row0 + B::RPL * i + lane / B::L::CH));
    }
    __device__ __forceinline__ bool fast(int j0, int block, int end) const { return a.one_page && j0 + block <= end; }
    // The pages of the rows of a block at j0 (keys from k0 on, `end` of them); past the end the last key's: no place of
    // the table is read that its length does not cover.  Through the constant address space: scalar loads.
    __device__ __forceinline__ void look_up(int j0, int end) {
        if (!a.one_page) return;
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int key = __builtin_amdgcn_readfirstlane(it.k0 + min(j0 + row0 + B::RPL * i, end - 1));
            const auto *t = (const __attribute__((address_space(4))) int32_t *)(it.pages + (key >> a.lay.shift));
            const int p = *t;
            page[i] = uint32_t(p) < uint32_t(a.lay.pages) ? p : 0;
        }
    }
    // Every lane's row of the block at j0; rows past the last key are that key's (their results are masked).
    __device__ __forceinline__ int last_key(int j0, int end, int i) const {
        return it.k0 + min(j0 + row0 + B::RPL * i + lane / B::L::CH, end - 1);
    }
    __device__ __forceinline__ void look_up_lanes(int j0, int end) {
#pragma unroll
        for (int i = 0; i < NL; ++i) page[i] = a.lay.page_at(it.pages, last_key(j0, end, i));
    }
    __device__ __forceinline__ void load(const char *cache, const CacheView &c, uint32_t tile, int j0, int end, bool whole) const {
        const int in_page = (1 << a.lay.shift) - 1;
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const uint32_t dst = tile + uint32_t(B::RPL * i * B::RB);
            if (whole) {
                const int64_t in = (it.k0 + j0 + row0 + B::RPL * i) & in_page;
                if (!PAD || chunk(i) < a.width)
                    load_chunk_saddr(uint32_t((lane / B::L::CH) * int(c.token) + chunk(i)),
                                     uint64_t(cache) + uint64_t(int64_t(page[i]) * c.page + in * c.token), dst);
            } else {
                const int64_t in = last_key(j0, end, i) & in_page;
                if (!PAD || chunk(i) < a.width) load_chunk_dma(cache + int64_t(page[i]) * c.page + in * c.token + chunk(i), dst);
            }
        }
    }
};

template <bool PAD, int BYTES> __device__ __forceinline__ void clear_padding(char *smem) {
    // Chunks past the head dim are zeros that no load overwrites.
    if (!PAD) return;
    for (uint32_t x = threadIdx.x * 16; x < uint32_t(BYTES); x += 256 * 16)
        *reinterpret_cast<floatx4 *>(smem + x) = floatx4{0.f, 0.f, 0.f, 0.f};
    lds_barrier();
}

// 128 rows, whose waves walk the same keys in blocks of 64, two buffers.
template <typename F, int D, bool PAD>
__device__ __forceinline__ void walk_tall(const Args &a, const Item &it, const int kvh, char *smem) {
    using C = Tall<F, D>;
    const uint32_t L = lds_addr(smem);
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int col = lane & 31, half = lane >> 5;
    const int group = a.lay.group, rows = it.tokens * group;
    const int r0w = it.r0 + 32 * wave, row = r0w + col;
    const int token = row / group, head = kvh * group + row % group;
    // Keys from k0 on that a token sees.
    const auto seen = [&](int t) { return max(min(it.k1, it.off >= it.len ? it.len : it.off + t + 1) - it.k0, 0); };
    const int row_end = seen(token);
    const int whole = seen(r0w / group);  // every row of the wave
    const int some = r0w < rows ? seen(min((r0w + 31) / group, it.tokens - 1)) : 0;  // any of them
    const int end = seen((min(it.r0 + C::BM, rows) - 1) / group);  // any of the workgroup
    const int nkb = (end + C::BN - 1) / C::BN;
    WaveState<F, D> w;
    w.template init<PAD>(a.q.at(it.first + token, head), row < rows, a.width, half);
    const uint32_t rk = uint32_t(C::L::off(col, half));
    const uint32_t cv0 = F::template col0<C::RB>(lane), cv1 = F::template col1<C::RB>(lane);
    PagedLoads<Base<F, D>, C::NL, PAD> loads(a, it, kvh, C::RPL * C::NL * wave, lane);

    const auto issue = [&](int kb) __attribute__((always_inline)) {
        const uint32_t t = L + uint32_t((kb & 1) * 2 * C::KB + C::RPL * C::NL * wave * C::RB);
        const int j0 = kb * C::BN;
        const bool fast = loads.fast(j0, C::BN, end);
        if (fast) {
            loads.load(loads.k, a.k, t, j0, end, true);
            loads.load(loads.v, a.v, t + C::KB, j0, end, true);
        } else {
            loads.look_up_lanes(j0, end);
            loads.load(loads.k, a.k, t, j0, end, false);
            loads.load(loads.v, a.v, t + C::KB, j0, end, false);
        }
    };
    // MASK: some rows of the wave do not see some keys of the block.
    const auto block = [&](auto mask, int kb) __attribute__((always_inline)) {
        constexpr bool MASK = decltype(mask)::value;
        const uint32_t kt0 = L + uint32_t((kb & 1) * 2 * C::KB);
        bool active[C::KT];
        floatx16 c[C::KT];
#pragma unroll
        for (int kt = 0; kt < C::KT; ++kt) {
            const int t0 = kb * C::BN + 32 * kt;
            active[kt] = !MASK || t0 < some;
            if (!active[kt]) continue;
            c[kt] = w.scores(kt0 + rk + uint32_t(32 * kt * C::RB));
            if (MASK) {
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (t0 + acc_row(r, half) >= row_end) c[kt][r] = -INFINITY;
            }
        }
        typename F::pvec pb[C::KT][2];
        w.template softmax<C::KT>(c, active, pb, a.c);
        const uint32_t vt = kt0 + uint32_t(C::KB);
#pragma unroll
        for (int kt = 0; kt < C::KT; ++kt)
            if (active[kt]) w.add(vt + cv0 + 32 * kt * C::RB, vt + cv1 + 32 * kt * C::RB, pb[kt]);
    };
    const auto step = [&](int kb) __attribute__((always_inline)) {
        // This wave's loads of the block have landed; after the barrier every wave's have, and every wave is done reading
        // the other buffer.
        wait_loads();
        lds_barrier();
        if (kb + 1 < nkb) {
            issue(kb + 1);
            if (kb + 2 < nkb) loads.look_up((kb + 2) * C::BN, end);
        }
    };
    clear_padding<PAD, C::LDS>(smem);
    if (nkb > 0) {
        loads.look_up(0, end);
        issue(0);
        if (nkb > 1) loads.look_up(C::BN, end);
    }
    // This wave's blocks, in loops without branches inside: [0, jp) whole, [jp, jw) masked, [jw, nkb) none of its pairs.
    const int jw = (some + C::BN - 1) / C::BN;
    const int jp = min(jw, whole / C::BN);
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
    if (row < rows) w.template leave<PAD>(a, it, token, head, half, row_end > 0);
}

template <int N> __device__ __forceinline__ void wait_loads_but() {
    static_assert(N < 64, "vmcnt");
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// 32 rows of a wave by itself, through LDS of its own: no barriers, and the next K is on its way while V is added, the next
// V while scores are computed.
template <typename F, int D, bool PAD>
__device__ __forceinline__ void walk_flat(const Args &a, const Item &it, const int kvh, const uint32_t kt) {
    using C = Flat<F, D>;
    const int lane = threadIdx.x & (kWave - 1);
    const int col = lane & 31, half = lane >> 5;
    const int group = a.lay.group, rows = it.tokens * group;
    const int row = it.r0 + col;
    const int token = row / group, head = kvh * group + row % group;
    const auto seen = [&](int t) { return max(min(it.k1, it.off >= it.len ? it.len : it.off + t + 1) - it.k0, 0); };
    const int row_end = seen(token);
    const int whole = seen(it.r0 / group);
    const int end = seen((min(it.r0 + C::BM, rows) - 1) / group);
    WaveState<F, D> w;
    w.template init<PAD>(a.q.at(it.first + token, head), row < rows, a.width, half);
    const uint32_t vt = kt + uint32_t(C::KB);
    const uint32_t rk = kt + uint32_t(C::L::off(col, half));
    const uint32_t cv0 = vt + F::template col0<C::RB>(lane), cv1 = vt + F::template col1<C::RB>(lane);
    PagedLoads<Base<F, D>, C::NL, PAD> loads(a, it, kvh, 0, lane);

    int j0 = 0;
    bool fast = false;
    const auto load_k = [&](int j) __attribute__((always_inline)) {
        fast = loads.fast(j, C::BN, end);
        if (fast) {
            loads.load(loads.k, a.k, kt, j, end, true);
        } else {
            loads.look_up_lanes(j, end);
            loads.load(loads.k, a.k, kt, j, end, false);
        }
    };
    const auto load_v = [&](int j) __attribute__((always_inline)) {
        if (fast) loads.load(loads.v, a.v, vt, j, end, true);
        else loads.load(loads.v, a.v, vt, j, end, false);
    };
    if (end > 0) {
        loads.look_up(0, end);
        load_k(0);
        load_v(0);
        while (true) {
            const int next = j0 + C::BN;
            const bool more = next < end;
            floatx16 c[1];
            const bool active[1] = {true};
            typename F::pvec pb[1][2];
            wait_loads_but<C::NL>();  // K is there, V may be on its way
            c[0] = w.scores(rk);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // K has been read
            if (more) {
                loads.look_up(next, end);
                load_k(next);
            }
            if (next > whole) {
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (j0 + acc_row(r, half) >= row_end) c[0][r] = -INFINITY;
            }
            w.template softmax<1>(c, active, pb, a.c);
            if (more) wait_loads_but<C::NL>();  // V is there
            else wait_loads_but<0>();
            w.add(cv0, cv1, pb[0]);
            if (!more) break;
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // V has been read
            load_v(next);
            j0 = next;
        }
    }
    if (row < rows) w.template leave<PAD>(a, it, token, head, half, row_end > 0);
}

// Workgroups of the prompts' keys first, then those of the requests' own.
template <typename F, int D, bool TP, bool TO> struct Both {
    static constexpr int TALL = TP || TO ? Tall<F, D>::LDS : 0, FLAT = TP && TO ? 0 : Flat<F, D>::LDS;
    static constexpr int LDS = TALL > FLAT ? TALL : FLAT;
    static constexpr int WPE = Base<F, D>::RB > 256 || LDS > 80 * 1024 ? 1 : 2;
};
template <typename F, int D, bool PAD, bool TP, bool TO>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(Both<F, D, TP, TO>::WPE, 2))) void shared_kernel(Args a) {
    __shared__ __attribute__((aligned(1024))) char smem[Both<F, D, TP, TO>::LDS];
    const int hkv = a.lay.hkv;
    const int pitems = a.ptiles * a.psplits * hkv, oitems = a.otiles * a.osplits * hkv;
    Item it;
    if (TP && int(blockIdx.x) < pitems) {
        const int slot = blockIdx.x / hkv;
        if (prefix_item<Tall<F, D>::BM, Tall<F, D>::BN>(a, slot % a.ptiles, slot / a.ptiles, it))
            walk_tall<F, D, PAD>(a, it, blockIdx.x % hkv, smem);
        return;
    }
    if constexpr (TO) {
        const int x = blockIdx.x - pitems, slot = x / hkv;
        if (own_item<Tall<F, D>::BM, Tall<F, D>::BN>(a, slot % a.otiles, slot / a.otiles, it))
            walk_tall<F, D, PAD>(a, it, x % hkv, smem);
    } else {
        // A wave's item: the key heads of a tile and stretch beside each other, prompts' before own.
        clear_padding<PAD, Flat<F, D>::LDS>(smem);
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
        int x = (int(blockIdx.x) - (TP ? pitems : 0)) * 4 + wave;
        const uint32_t tile = lds_addr(smem) + uint32_t(wave * 2 * Flat<F, D>::KB);
        bool there;
        if (!TP && x < pitems) {
            const int slot = x / hkv;
            there = prefix_item<Flat<F, D>::BM, Flat<F, D>::BN>(a, slot % a.ptiles, slot / a.ptiles, it);
        } else {
            if (!TP) x -= pitems;
            const int slot = x / hkv;
            there = x < oitems && own_item<Flat<F, D>::BM, Flat<F, D>::BN>(a, slot % a.otiles, slot / a.otiles, it);
        }
        if (there) walk_flat<F, D, PAD>(a, it, x % hkv, tile);
    }
}

// O = sum of 2^(m_s - m) O_s / sum of 2^(m_s - m) l_s over the splits s that saw a key.  A thread joins 4 elements of a row's
// head, 8 splits' loads at a time.
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
    const float *ml = a.ml + 2 * rh, *po = a.po + rh * a.dp + c;
    constexpr int N = 8;
    float m = kLowest, l = 0.f;
    floatx4 o = {0.f, 0.f, 0.f, 0.f};
    for (int s = s0; s < s1; s += N) {
        float2 x[N];
        floatx4 p[N];
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = s + i < s1 ? *reinterpret_cast<const float2 *>(ml + 2 * (s + i) * step) : float2{kLowest, 0.f};
#pragma unroll
        for (int i = 0; i < N; ++i)
            p[i] = x[i].y == 0.f ? floatx4{0.f, 0.f, 0.f, 0.f} : *reinterpret_cast<const floatx4 *>(po + (s + i) * step * a.dp);
        float top = m;
#pragma unroll
        for (int i = 0; i < N; ++i) top = x[i].y == 0.f ? top : fmaxf(top, x[i].x);
        const float keep = fast_exp2(m - top);
        l *= keep;
        o *= keep;
        m = top;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float w = x[i].y == 0.f ? 0.f : fast_exp2(x[i].x - top);
            l += w * x[i].y;
            o += w * p[i];
        }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const float r[4] = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
    store4<F>(reinterpret_cast<S *>(a.o.at(n, h)) + c, r);
    if (a.lse != nullptr && c == 0) a.lse[rh] = l == 0.f ? -INFINITY : (m + __log2f(l)) * kLn2;
}

// Tiles and splits, from the call's shapes and whether it says which rows and requests belong together.
struct Plan {
    bool tall_prefix, tall_own;
    int ptiles, psplits, otiles, osplits, pper, oper, omost;
};
int64_t up(int64_t x) { return (x + 255) / 256 * 256; }
int64_t dp_of(int64_t d) { return d <= 32 ? 32 : d <= 64 ? 64 : 128; }
// A request's own keys that one work item takes, where `tiles` tiles of rows and key heads have up to `most` each and all rows'
// O is `bytes`.  Flat: 4096 waves, two for every wave's place, and no more than 512 keys a wave, for lengths differ (256
// requests of 1 to 2048 keys, 8 key heads of 128: 128 / 256 / 512 / 1024 keys 226 / 220 / 220 / 238 us; 128 requests of
// 1 to 1024: 69 / 71 / 70 / 84).  At most 64 stretches, and no more than leave 256 MB of partial O, whatever the table's width:
// with as many rows the chip is full, and every stretch writes and reads them (tables of 32768 tokens, 32/8 heads of 128, bf16,
// on a prompt of 512; bound of 64 / 256 / 1024 MB, and none: 8192 rows of 8 full requests 4.7 / 4.7 / 4.9 and 6.3 ms, of
// short ones 348 / 348 / 415 and 780 us; 1024 rows of one request each of 1 to 4000 tokens 1.55 / 1.54 / 1.87 and 1.87 ms, with
// one of 32768 among short ones 970 / 740 / 970 and 970 us; tables of 131072, 75 rows of each of 24 requests, one of them full:
// 1540 / 570 / 520 and 620 us).
int64_t keys_each(int64_t tiles, int64_t most, bool tall, int64_t bytes) {
    const int64_t x = tiles * most / 4096, lo = tall ? 256 : 64, hi = tall ? 1024 : 512;
    const int64_t parts = std::min(int64_t(64), std::max(int64_t(1), (int64_t(256) << 20) / bytes));
    return (std::max(std::min(std::max(x, lo), hi), (most + parts - 1) / parts) + 63) / 64 * 64;
}
Plan plan_of(const SharedCall &c, bool starts, bool group_starts) {
    Plan p{};
    const int64_t work_rows = c.rows * c.group();
    const auto div = [](int64_t x, int64_t y) { return (x + y - 1) / y; };
    p.tall_own = work_rows > 32 * c.requests;
    p.tall_prefix = p.tall_own || (c.groups > 0 && work_rows > 32 * c.groups);
    if (c.requests > 0) {
        const int64_t bm = p.tall_own ? 128 : 32;
        p.oper = starts ? 0 : int(div(c.group(), bm));
        p.otiles = int(p.oper > 0 ? p.oper * c.requests : work_rows / bm + c.requests);
        p.omost = int(keys_each(p.otiles * c.hkv, c.max_own(), p.tall_own, c.rows * c.hq * dp_of(c.d) * 4));
        p.osplits = int(std::max<int64_t>(1, div(c.max_own(), p.omost)));
    }
    if (c.max_prefix() > 0) {
        const int64_t bm = p.tall_prefix ? 128 : 32;
        p.pper = starts || group_starts ? 0 : int(div(c.requests / c.groups * c.group(), bm));
        p.ptiles = int(p.pper > 0 ? p.pper * c.groups : c.groups == 1 ? div(work_rows, bm) : work_rows / bm + c.groups);
        // Tall: a workgroup a CU where the requests' own keys are as many, so that these stream in beside it, and two
        // where not (32768 keys, 1024 rows of 8 key heads, with 1 to 2048 keys of 256 requests' own: 306 us with 256
        // workgroups, 377 with 512; without: 211 and 175).
        const bool beside = !p.tall_own && c.requests * c.max_own() >= c.groups * c.max_prefix();
        const int64_t items = p.tall_prefix ? (beside ? 256 : 512) : 2048, least = p.tall_prefix ? 128 : 64;
        p.psplits = int(std::max<int64_t>(1, std::min({int64_t(128), items / std::max<int64_t>(1, p.ptiles * c.hkv), div(c.max_prefix(), least)})));
    }
    return p;
}
Plan plan_of(const SharedCall &c) { return plan_of(c, c.starts != nullptr, c.group_starts != nullptr); }
int64_t workspace_of(const SharedCall &c, const Plan &p) {
    const int64_t row_heads = (p.psplits + p.osplits) * c.rows * c.hq;
    return up(row_heads * dp_of(c.d) * 4) + up(row_heads * 8);
}

template <typename F, int D, bool PAD> hipError_t launch_d(const Args &a, const Plan &p, hipStream_t stream) {
    const int64_t prompts = int64_t(p.ptiles) * p.psplits * a.lay.hkv, own = int64_t(p.otiles) * p.osplits * a.lay.hkv;
    if (prompts + own > 0x7FFFFFFF) return hipErrorInvalidValue;
    const int64_t flat = (p.tall_own ? 0 : own) + (p.tall_prefix ? 0 : prompts);  // waves
    const int64_t blocks = (p.tall_prefix ? prompts : 0) + (p.tall_own ? own : 0) + (flat + 3) / 4;
    if (!grid_fits(blocks, 256)) return hipErrorInvalidValue;
    if (blocks > 0) {
        const dim3 grid(static_cast<unsigned>(blocks)), block(256);
        if (p.tall_own) shared_kernel<F, D, PAD, true, true><<<grid, block, 0, stream>>>(a);
        else if (p.tall_prefix) shared_kernel<F, D, PAD, true, false><<<grid, block, 0, stream>>>(a);
        else shared_kernel<F, D, PAD, false, false><<<grid, block, 0, stream>>>(a);
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
    a.pper = p.pper;
    a.oper = p.oper;
    a.omost = p.omost;
    a.c = kLog2e / sqrtf(float(c.d));
    // Rows of a load instruction: 64 lanes of 16 bytes; lane offsets are 32 bits from the first of them.
    const int64_t rows_per_load = kWave * 16 / (a.dp * e);
    a.one_page = c.page_size >= rows_per_load && a.k.token < (int64_t(1) << 26) && a.v.token < (int64_t(1) << 26);
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

int64_t shared_workspace_bytes(const SharedCall &c) { return workspace_of(c, plan_of(c)); }

int64_t shared_workspace_most(const SharedCall &c) {
    // With starts the groups' make no difference; other than one row a request is never without.
    int64_t most = workspace_of(c, plan_of(c, true, false));
    if (c.rows == c.requests) {
        most = std::max(most, workspace_of(c, plan_of(c, false, true)));
        if (c.groups == 0 || c.requests % c.groups == 0) most = std::max(most, workspace_of(c, plan_of(c, false, false)));
    }
    return most;
}

hipError_t launch_shared(const SharedCall &c, void *workspace, hipStream_t stream) {
    switch (c.dtype) {
    case 0: return launch_f<PF32>(c, workspace, stream);
    case 1: return launch_f<PBf16>(c, workspace, stream);
    default: return launch_f<PF16>(c, workspace, stream);
    }
}

}  // namespace ctattn
