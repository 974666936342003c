// Scaled token lookup and its gradient by sorted tokens (entry points in include/ctattn.h).
//
//   out[n] = scale table[ids[n]]                         dtable[v] = scale sum_{n: ids[n] = v} dout[n]
//
// The gradient groups equal ids with a stable radix sort of (id, position) and sums each group in the
// order of its positions in fixed pieces: no atomics on values, so the same inputs give the same bits, and
// sums are held in fp32 (fp64 for fp64) and rounded once, where adds into a 16-bit table would round at
// every one.  Ids outside the table sort behind every row and are dropped.
//
// Steps: (1) the sort, 9 bits of the id a pass, each pass a histogram per block of tokens and a scatter (a
// batch of up to 4096 tokens is sorted by one workgroup in LDS instead); the table's zeros are written by
// further workgroups of the same launches, which would leave most of the chip idle.  (2) Pieces of
// 16 or 32 sorted tokens, one wave per piece and slab of columns, its loads of whole row segments
// in flight together: a row whose tokens lie within the piece is written at once, sums that go on
// across the piece's ends are kept.  (3) Those are joined, in order, by a workgroup for each such row and
// slab, so that a row as frequent as half of the batch is spread over as many waves as any others.
// Bound by HBM: the rows of dout once, the table once.  Measured, bf16: lookup of 16384 rows of 768 9.0 us (5.6 TB/s);
// gradient of 65536 tokens x 2048 into 131072 rows 231 us, of it 101 in the sort's launches (the zeros at 5.7 TB/s
// beside it), 121 sums (3.3 TB/s of random rows), 14 joins; 16384 x 768 into 50257 rows 46 us, 31 of them sort and zeros.
#include "attn_common.h"
#include "attn_launch.h"
#include "capi_util.h"
#include "ctattn.h"

#include <algorithm>
#include <type_traits>

namespace ctattn {
namespace {

constexpr int kBits = 9;            // of the id per pass
constexpr int kBins = 1 << kBits;
constexpr int kSmall = 4096;        // tokens that one workgroup sorts
constexpr int kSmallWaves = 16;
constexpr int kSortThreads = 256;   // a block of the passes over more tokens

template <int W> struct Raw;
template <> struct Raw<2> { using type = uint16_t; };
template <> struct Raw<4> { using type = uint32_t; };
template <> struct Raw<8> { using type = uint2; };
template <> struct Raw<16> { using type = uint4; };

// VEC elements of T as one access.
template <typename T, int VEC> struct Pack {
    using R = typename Raw<int(sizeof(T)) * VEC>::type;
    T v[VEC];
    __device__ static Pack load(const T *p) { return __builtin_bit_cast(Pack, *reinterpret_cast<const R *>(p)); }
    __device__ void store(T *p) const { *reinterpret_cast<R *>(p) = __builtin_bit_cast(R, *this); }
};

template <typename I> __device__ __forceinline__ uint32_t key_of(const I *ids, int64_t n, int64_t vocab) {
    const int64_t id = int64_t(ids[n]);
    return id >= 0 && id < vocab ? uint32_t(id) : uint32_t(vocab);
}

// ---- lookup: a wave per row and slab of 64 VEC columns ----
template <typename T, typename I, int VEC>
__global__ __launch_bounds__(256) void lookup_kernel(const I *__restrict__ ids, const T *__restrict__ table,
                                                    T *__restrict__ out, int64_t rows, int64_t D, int64_t vocab,
                                                    int slabs, acc_t<T> scale) {
    const int lane = threadIdx.x & (kWave - 1);
    const int64_t waves = int64_t(gridDim.x) * (blockDim.x / kWave);
    const int64_t total = rows * slabs;
    for (int64_t w = int64_t(blockIdx.x) * (blockDim.x / kWave) + threadIdx.x / kWave; w < total; w += waves) {
        const int64_t n = w / slabs, c = (int64_t(w % slabs) * kWave + lane) * VEC;
        if (c >= D) continue;
        const int64_t id = int64_t(ids[n]);
        Pack<T, VEC> x;
        if (id >= 0 && id < vocab) {
            x = Pack<T, VEC>::load(table + id * D + c);
#pragma unroll
            for (int e = 0; e < VEC; ++e) x.v[e] = from_acc<T>(to_acc(x.v[e]) * scale);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) x.v[e] = from_acc<T>(acc_t<T>(0));
        }
        x.store(out + n * D + c);
    }
}

// ---- zeros: workgroup b of nb writes its share of `bytes`, whose ends may lie off 16 bytes ----
struct Fill {
    char *p;
    int64_t bytes;
};
__device__ __forceinline__ void fill_share(const Fill &f, int64_t b, int64_t nb) {
    const int64_t head = (16 - int64_t(reinterpret_cast<uintptr_t>(f.p) & 15)) & 15;
    if (f.bytes <= head + 16) {
        if (b == 0)
            for (int64_t i = threadIdx.x; i < f.bytes; i += blockDim.x) f.p[i] = 0;
        return;
    }
    const int64_t n16 = (f.bytes - head) / 16, tail = f.bytes - head - 16 * n16;
    uint4 *q = reinterpret_cast<uint4 *>(f.p + head);
    for (int64_t i = b * blockDim.x + threadIdx.x; i < n16; i += nb * blockDim.x) q[i] = make_uint4(0, 0, 0, 0);
    if (b == 0) {
        if (int64_t(threadIdx.x) < head) f.p[threadIdx.x] = 0;
        if (int64_t(threadIdx.x) < tail) f.p[f.bytes - tail + threadIdx.x] = 0;
    }
}

// Lanes of the wave whose digit equals this lane's, among `live` lanes.
__device__ __forceinline__ uint64_t same_digit(uint32_t digit, uint64_t live) {
    uint64_t m = live;
#pragma unroll
    for (int b = 0; b < kBits; ++b) {
        const bool bit = (digit >> b) & 1;
        const uint64_t set = __ballot(bit);
        m &= bit ? set : ~set;
    }
    return m;
}
__device__ __forceinline__ int below(uint64_t m, int lane) { return __popcll(m & ((uint64_t(1) << lane) - 1)); }

// Exclusive sums over the waves' counts and the digits: cnt[w][bin] becomes the first place of wave w's
// tokens with that digit, given that digits below start at base[bin] (base may be null: from 0).
template <int WAVES>
__device__ __forceinline__ void place_bins(uint32_t (*cnt)[kBins], uint32_t *total, const uint32_t *base) {
    for (int bin = threadIdx.x; bin < kBins; bin += blockDim.x) {
        uint32_t s = 0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const uint32_t x = cnt[w][bin];
            cnt[w][bin] = s;
            s += x;
        }
        total[bin] = s;
    }
    __syncthreads();
    if (base == nullptr && threadIdx.x < kWave) {  // one wave scans the digits, 8 a lane
        uint32_t v[kBins / kWave], s = 0;
#pragma unroll
        for (int i = 0; i < kBins / kWave; ++i) {
            v[i] = s;
            s += total[threadIdx.x * (kBins / kWave) + i];
        }
        uint32_t run = s;
#pragma unroll
        for (int off = 1; off < kWave; off <<= 1) {
            const uint32_t y = __shfl_up(run, off, kWave);
            if (int(threadIdx.x) >= off) run += y;
        }
#pragma unroll
        for (int i = 0; i < kBins / kWave; ++i) total[threadIdx.x * (kBins / kWave) + i] = v[i] + run - s;
    }
    __syncthreads();
    for (int bin = threadIdx.x; bin < kBins; bin += blockDim.x) {
        const uint32_t b = base == nullptr ? total[bin] : base[bin];
#pragma unroll
        for (int w = 0; w < WAVES; ++w) cnt[w][bin] += b;
    }
    __syncthreads();
}

// ---- up to kSmall tokens: workgroup 0 sorts, the others write zeros ----
template <typename I>
__global__ __launch_bounds__(kSmallWaves *kWave) void sort_small_kernel(const I *__restrict__ ids, int n, int64_t vocab,
                                                                       int passes, uint2 *__restrict__ sorted,
                                                                       Fill fill) {
    if (blockIdx.x > 0) {
        fill_share(fill, blockIdx.x - 1, gridDim.x - 1);
        return;
    }
    __shared__ uint2 buf[2][kSmall];
    __shared__ uint32_t cnt[kSmallWaves][kBins];
    __shared__ uint32_t total[kBins];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    for (int i = threadIdx.x; i < n; i += blockDim.x) buf[0][i] = make_uint2(key_of(ids, i, vocab), uint32_t(i));
    const int per = (n + kSmallWaves * kWave - 1) / (kSmallWaves * kWave) * kWave;  // tokens of a wave
    const int lo = wave * per, hi = min(n, lo + per);
    for (int pass = 0; pass < passes; ++pass) {
        const uint2 *from = buf[pass & 1];
        uint2 *to = buf[(pass & 1) ^ 1];
        for (int i = threadIdx.x; i < kSmallWaves * kBins; i += blockDim.x) (&cnt[0][0])[i] = 0;
        __syncthreads();
        for (int i = lo + lane; i < hi; i += kWave) atomicAdd(&cnt[wave][(from[i].x >> (kBits * pass)) & (kBins - 1)], 1u);
        __syncthreads();
        place_bins<kSmallWaves>(cnt, total, nullptr);
        for (int i0 = lo; i0 < hi; i0 += kWave) {  // uniform per wave: every lane votes
            const int i = i0 + lane;
            const uint2 x = from[min(i, n - 1)];
            const uint32_t digit = (x.x >> (kBits * pass)) & (kBins - 1);
            const uint64_t m = same_digit(digit, __ballot(i < hi));
            uint32_t at = 0;
            if (i < hi) at = cnt[wave][digit] + below(m, lane);
            // The wave's lanes have read their counts before the group's last lane moves them on.
            __builtin_amdgcn_wave_barrier();
            if (i < hi) {
                to[at] = x;
                if ((m >> lane) == 1) cnt[wave][digit] = at + 1;
            }
            __builtin_amdgcn_wave_barrier();
        }
        __syncthreads();
    }
    for (int i = threadIdx.x; i < n; i += blockDim.x) sorted[i] = buf[passes & 1][i];
}

// ---- more tokens: a histogram of each block's tokens for the first pass, zeros for the others', which the
// scatter of the pass before counts ----
template <typename I>
__global__ __launch_bounds__(kSortThreads) void hist_kernel(const I *__restrict__ ids, int64_t n, int64_t vocab,
                                                           int passes, int blocks, int per, uint32_t *__restrict__ hist,
                                                           Fill fill) {
    if (int(blockIdx.x) >= blocks) {
        fill_share(fill, blockIdx.x - blocks, gridDim.x - blocks);
        return;
    }
    __shared__ uint32_t h[kBins];
    for (int i = threadIdx.x; i < kBins; i += blockDim.x) h[i] = 0;
    __syncthreads();
    const int64_t lo = int64_t(blockIdx.x) * per, hi = min(n, lo + per);
    for (int64_t i = lo + threadIdx.x; i < hi; i += blockDim.x) atomicAdd(&h[key_of(ids, i, vocab) & (kBins - 1)], 1u);
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += blockDim.x) {
        hist[int64_t(blockIdx.x) * kBins + i] = h[i];
        for (int p = 1; p < passes; ++p) hist[(int64_t(p) * blocks + blockIdx.x) * kBins + i] = 0;
    }
}

// A block's tokens to their places: digits below, the same digit in blocks before, then within the block in order.
template <typename I>
__global__ __launch_bounds__(kSortThreads) void scatter_kernel(const I *__restrict__ ids, const uint2 *__restrict__ from,
                                                              int64_t n, int64_t vocab, int pass, int blocks, int per,
                                                              const uint32_t *__restrict__ hist,
                                                              uint32_t *__restrict__ next, uint2 *__restrict__ to,
                                                              Fill fill) {
    if (int(blockIdx.x) >= blocks) {
        fill_share(fill, blockIdx.x - blocks, gridDim.x - blocks);
        return;
    }
    constexpr int WAVES = kSortThreads / kWave;
    __shared__ uint32_t cnt[WAVES][kBins];
    __shared__ uint32_t base[kBins];
    __shared__ uint32_t total[kBins];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    for (int i = threadIdx.x; i < WAVES * kBins; i += blockDim.x) (&cnt[0][0])[i] = 0;
    for (int bin = threadIdx.x; bin < kBins; bin += blockDim.x) {
        uint32_t before = 0, all = 0;
#pragma unroll 16
        for (int b = 0; b < blocks; ++b) {
            const uint32_t x = hist[int64_t(b) * kBins + bin];
            before += b < int(blockIdx.x) ? x : 0;
            all += x;
        }
        base[bin] = before;
        total[bin] = all;
    }
    __syncthreads();
    if (threadIdx.x < kWave) {  // digits below
        uint32_t v[kBins / kWave], s = 0;
#pragma unroll
        for (int i = 0; i < kBins / kWave; ++i) {
            v[i] = s;
            s += total[threadIdx.x * (kBins / kWave) + i];
        }
        uint32_t run = s;
#pragma unroll
        for (int off = 1; off < kWave; off <<= 1) {
            const uint32_t y = __shfl_up(run, off, kWave);
            if (int(threadIdx.x) >= off) run += y;
        }
#pragma unroll
        for (int i = 0; i < kBins / kWave; ++i) base[threadIdx.x * (kBins / kWave) + i] += v[i] + run - s;
    }
    __syncthreads();
    const int64_t lo0 = int64_t(blockIdx.x) * per, hi0 = min(n, lo0 + per);
    const int64_t lo = lo0 + int64_t(wave) * (per / WAVES), hi = min(hi0, lo + per / WAVES);
    auto item = [&](int64_t i) {
        return pass == 0 ? make_uint2(key_of(ids, i, vocab), uint32_t(i)) : from[i];
    };
    // The first tokens of a lane stay in registers (all of them in blocks of 1024).
    constexpr int KEEP = 1024 / kSortThreads;
    uint2 kept[KEEP];
#pragma unroll
    for (int j = 0; j < KEEP; ++j) kept[j] = item(min(lo + j * kWave + lane, n - 1));
    auto digit_of = [&](uint32_t key) { return (key >> (kBits * pass)) & (kBins - 1); };
#pragma unroll
    for (int j = 0; j < KEEP; ++j)
        if (lo + j * kWave + lane < hi) atomicAdd(&cnt[wave][digit_of(kept[j].x)], 1u);
    for (int64_t i = lo + KEEP * kWave + lane; i < hi; i += kWave) atomicAdd(&cnt[wave][digit_of(item(i).x)], 1u);
    __syncthreads();
    place_bins<WAVES>(cnt, total, base);
    auto place = [&](const uint2 &x, bool live) __attribute__((always_inline)) {
        const uint32_t digit = digit_of(x.x);
        const uint64_t m = same_digit(digit, __ballot(live));
        uint32_t at = 0;
        if (live) at = cnt[wave][digit] + below(m, lane);
        __builtin_amdgcn_wave_barrier();
        if (live) {
            to[at] = x;
            if ((m >> lane) == 1) cnt[wave][digit] = at + 1;
            if (next != nullptr) atomicAdd(next + int64_t(at / uint32_t(per)) * kBins + ((x.x >> (kBits * (pass + 1))) & (kBins - 1)), 1u);
        }
        __builtin_amdgcn_wave_barrier();
    };
#pragma unroll
    for (int j = 0; j < KEEP; ++j)
        if (lo + j * kWave < hi) place(kept[j], lo + j * kWave + lane < hi);
    for (int64_t i0 = lo + KEEP * kWave; i0 < hi; i0 += kWave) place(item(min(i0 + lane, n - 1)), i0 + lane < hi);
}

// ---- sums ----
// Columns of a lane: STRIPS runs of VEC elements, 64 VEC apart.
template <typename T, int VEC, int STRIPS> struct Cols {
    using A = acc_t<T>;
    A a[STRIPS][VEC];
    __device__ void zero() {
#pragma unroll
        for (int s = 0; s < STRIPS; ++s)
#pragma unroll
            for (int e = 0; e < VEC; ++e) a[s][e] = 0;
    }
};

template <typename T, int VEC, int STRIPS>
__device__ __forceinline__ void put_row(T *row, const Cols<T, VEC, STRIPS> &x, int64_t c0, int64_t D, acc_t<T> scale,
                                        bool accumulate) {
#pragma unroll
    for (int s = 0; s < STRIPS; ++s) {
        const int64_t c = c0 + int64_t(s) * kWave * VEC;
        if (c >= D) continue;
        Pack<T, VEC> y;
        if (accumulate) y = Pack<T, VEC>::load(row + c);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const acc_t<T> v = x.a[s][e] * scale;
            y.v[e] = from_acc<T>(accumulate ? to_acc(y.v[e]) + v : v);
        }
        y.store(row + c);
    }
}

// What is said of a chunk's end: no row goes on behind it, the row that goes on began in it, or it went on
// into it as well.
enum : uint32_t { kEnds = 0, kBegins, kThrough };

// One wave per chunk of CH sorted tokens and slab.  edge[chunk] is the sum of the chunk's tokens whose row
// began in an earlier chunk, edge[chunks + chunk] of those whose row goes on into the next one and began
// in this.  (Letting a wave finish a row that ends within the next 48 tokens, to have fewer sums to join, made
// chains of loads of it: 16384 tokens x 768 13 -> 33 us.)
template <typename T, int VEC, int STRIPS, int CH>
__global__ __launch_bounds__(256) void sum_kernel(const uint2 *__restrict__ sorted, const T *__restrict__ dout,
                                                 T *__restrict__ dtable, acc_t<T> *__restrict__ edge,
                                                 uint2 *__restrict__ ends, int64_t n, int64_t chunks, int64_t D,
                                                 int slabs, int64_t vocab, acc_t<T> scale, int accumulate) {
    using A = acc_t<T>;
    static_assert(CH <= kWave, "a lane per token");
    const int lane = threadIdx.x & (kWave - 1);
    const int64_t w = int64_t(blockIdx.x) * (blockDim.x / kWave) + threadIdx.x / kWave;
    const int64_t chunk = w / slabs;
    if (chunk >= chunks) return;
    const int slab = int(w % slabs);
    const int64_t c0 = int64_t(slab) * kWave * VEC * STRIPS + int64_t(lane) * VEC;
    const int64_t lo = chunk * CH;
    const int cnt = int(min(n - lo, int64_t(CH)));
    const uint2 mine = sorted[lo + min(lane, cnt - 1)];
    const uint32_t prev = lo > 0 ? sorted[lo - 1].x : 0xFFFFFFFFu;
    const uint32_t next = lo + cnt < n ? sorted[lo + cnt].x : 0xFFFFFFFFu;
    auto key_at = [&](int i) __attribute__((always_inline)) { return uint32_t(__builtin_amdgcn_readlane(mine.x, i)); };
    int64_t col[STRIPS];  // held inside the row: a guard on each load would make a chain of them
#pragma unroll
    for (int s = 0; s < STRIPS; ++s) col[s] = min(c0 + int64_t(s) * kWave * VEC, D - VEC);
    Cols<T, VEC, STRIPS> sum;
    sum.zero();
    bool begun = key_at(0) != prev;  // the current row began in this chunk
    uint32_t row = 0, state = kEnds;
    constexpr int U = sizeof(T) * VEC * STRIPS >= 16 ? 8 : 16;  // rows in flight
    for (int i0 = 0; i0 < cnt; i0 += U) {
        Pack<T, VEC> x[U][STRIPS];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t pos = uint32_t(__builtin_amdgcn_readlane(mine.y, min(i0 + u, cnt - 1)));
#pragma unroll
            for (int s = 0; s < STRIPS; ++s) x[u][s] = Pack<T, VEC>::load(dout + pos * D + col[s]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u;
            if (i >= cnt) break;
            const uint32_t key = key_at(i);
            if (key >= uint32_t(vocab)) {  // the rest belongs to no row
                i0 = cnt;
                break;
            }
            row = key;
#pragma unroll
            for (int s = 0; s < STRIPS; ++s)
#pragma unroll
                for (int e = 0; e < VEC; ++e) sum.a[s][e] += to_acc(x[u][s].v[e]);
            const bool at_end = i + 1 >= cnt;
            const bool goes_on = (at_end ? next : key_at(min(i + 1, cnt - 1))) == key;
            if (goes_on && !at_end) continue;
            if (!goes_on && begun) {
                put_row<T, VEC, STRIPS>(dtable + int64_t(key) * D, sum, c0, D, scale, accumulate != 0);
            } else {
                A *to = edge + (begun ? chunks + chunk : chunk) * D;
                state = !goes_on ? kEnds : begun ? kBegins : kThrough;
#pragma unroll
                for (int s = 0; s < STRIPS; ++s)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        const int64_t c = c0 + int64_t(s) * kWave * VEC + e;
                        if (c < D) to[c] = sum.a[s][e];
                    }
            }
            sum.zero();
            begun = true;
        }
    }
    if (slab == 0 && lane == 0) ends[chunk] = make_uint2(row, state);
}

// Rows across chunks: the workgroup of the chunk in which the row begins (and of a slab of columns) adds up its
// own edge and those of the following chunks, wave w of 4 the w-th quarter of them, the waves' sums in order.  `ends`
// tells in one load whether the chunk has such a row and how far it goes.  The pieces are loaded 8 at a time, their
// columns held inside the row rather than guarded, so that a frequent row is not a chain of loads (16384 tokens x
// 768: 13 us with guarded loads).
constexpr int kJoinWaves = 4;
constexpr int kJoinCols = 4;  // columns of a lane, 64 apart
template <typename T>
__global__ __launch_bounds__(kJoinWaves *kWave) void join_kernel(const uint2 *__restrict__ ends, T *__restrict__ dtable,
                                                                const acc_t<T> *__restrict__ edge, int64_t chunks,
                                                                int64_t D, int slabs, acc_t<T> scale, int accumulate) {
    using A = acc_t<T>;
    __shared__ A part[kJoinWaves][kJoinCols * kWave];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int64_t chunk = blockIdx.x / slabs;
    const uint2 mine = ends[chunk];
    int64_t last = chunk + 1;  // the row's last chunk: the first from here on that it does not go through
    uint32_t other = ends[min(last + lane, chunks - 1)].y;
    if (mine.y != kBegins) return;
    for (;;) {
        const uint64_t m = __ballot(last + lane >= chunks - 1 || other != kThrough);
        if (m != 0) {
            last += __ffsll((unsigned long long)m) - 1;
            break;
        }
        last += kWave;
        other = ends[min(last + lane, chunks - 1)].y;
    }
    const uint32_t key = mine.x;
    const int64_t parts = last - chunk + 1;  // this chunk's own edge first
    const int64_t per = (parts + kJoinWaves - 1) / kJoinWaves;
    const int64_t c0 = int64_t(blockIdx.x % slabs) * kJoinCols * kWave + lane;
    int64_t col[kJoinCols];
    A s[kJoinCols];
#pragma unroll
    for (int k = 0; k < kJoinCols; ++k) col[k] = min(c0 + k * kWave, D - 1), s[k] = 0;
    const int64_t p_end = min(parts, (wave + 1) * per);
    constexpr int U = 8;
    for (int64_t p = wave * per; p < p_end; p += U) {
        A x[U][kJoinCols];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t q = min(p + u, p_end - 1);
            const A *piece = edge + (q == 0 ? chunks + chunk : chunk + q) * D;
#pragma unroll
            for (int k = 0; k < kJoinCols; ++k) x[u][k] = piece[col[k]];
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int k = 0; k < kJoinCols; ++k) s[k] += p + u < p_end ? x[u][k] : A(0);
    }
#pragma unroll
    for (int k = 0; k < kJoinCols; ++k) part[wave][k * kWave + lane] = s[k];
    __syncthreads();
    static_assert(kJoinWaves == kJoinCols, "wave w writes strip w");
    const int64_t c = c0 + wave * kWave;
    if (c < D) {
        A v = 0;
#pragma unroll
        for (int w = 0; w < kJoinWaves; ++w) v += part[w][wave * kWave + lane];
        T *to = dtable + int64_t(key) * D + c;
        v *= scale;
        *to = from_acc<T>(accumulate ? to_acc(*to) + v : v);
    }
}

// ---- sizes ----
struct GradPlan {
    int passes, blocks, per;  // sort
    int chunk;                // tokens of a piece: 16 or 32
    int64_t chunks;
    int64_t off_a, off_b, off_hist, off_ends, off_edge, bytes;
};
GradPlan grad_plan(int dtype, int64_t n, int64_t D, int64_t vocab) {
    GradPlan g{};
    int bits = 1;
    while ((int64_t(1) << bits) <= vocab) ++bits;  // ids 0 .. vocab, the last for those outside
    g.passes = (bits + kBits - 1) / kBits;
    // A scatter reads every block's histogram, so there are at most 64 of them.  (bf16: 128 blocks are the same up to
    // 65536 tokens, 131072 tokens x 768 into 50257 rows 117 us with 64 and 107 with 128, 262144 x 256 125 and 103.)
    int64_t per = 1024;
    while (per * 64 < n) per *= 2;
    g.per = int(per);
    g.blocks = int((n + per - 1) / per);
    // Pieces of 32 tokens keep fewer sums across their ends; 16 make twice the waves.  bf16, 16 / 32 tokens, us: n D 2^23.6
    // (16384 x 768 into 50257 rows) 44.6 / 46.8, 2^24 (8192 x 2048) 66.3 / 68.6, 2^24.6 57.1 / 58.6, 2^25 (16384 x 2048)
    // 72.3 / 71.7 and (32768 x 1024) 62.5 / 61.4, 2^26 (32768 x 2048 into 131072) 178 / 170, 2^27 239 / 233.
    g.chunk = n * D < (int64_t(1) << 25) ? 16 : 32;
    g.chunks = (n + g.chunk - 1) / g.chunk;
    const int64_t pairs = capi::align_up(n * int64_t(sizeof(uint2)));
    g.off_a = 0;
    g.off_b = pairs;
    g.off_hist = 2 * pairs;
    g.off_ends = g.off_hist + capi::align_up(int64_t(64) * g.passes * kBins * 4);
    g.off_edge = g.off_ends + capi::align_up(g.chunks * int64_t(sizeof(uint2)));
    g.bytes = g.off_edge + 2 * g.chunks * D * (dtype == CTATTN_F64 ? 8 : 4);
    return g;
}

template <typename T, typename I>
hipError_t lookup(const I *ids, const T *table, T *out, int64_t n, int64_t D, int64_t vocab, double scale,
                  hipStream_t st) {
    auto launch = [&](auto kernel, int vec) {
        const int64_t slabs = (D + kWave * vec - 1) / (kWave * vec);
        hipLaunchKernelGGL(kernel, dim3(stride_grid((n * slabs + 3) / 4, 256)), dim3(256), 0, st, ids, table, out, n, D,
                           vocab, int(slabs), acc_t<T>(scale));
        return hipGetLastError();
    };
    constexpr int V = 16 / int(sizeof(T));
    const uintptr_t at = reinterpret_cast<uintptr_t>(table) | reinterpret_cast<uintptr_t>(out);
    if (D % V == 0 && at % 16 == 0) return launch(lookup_kernel<T, I, V>, V);
    return launch(lookup_kernel<T, I, 1>, 1);
}

template <typename T, int CH>
hipError_t sums(const GradPlan &g, const uint2 *sorted, const T *dout, T *dtable, acc_t<T> *edge, uint2 *ends,
                double scale,
                bool accumulate, int64_t n, int64_t D, int64_t vocab, hipStream_t st) {
    using A = acc_t<T>;
    auto pieces = [&](auto kernel, int cols) {
        const int64_t slabs = (D + kWave * cols - 1) / (kWave * cols);
        const int64_t waves = g.chunks * slabs;
        if (!grid_fits((waves + 3) / 4, 256)) return hipErrorInvalidValue;
        hipLaunchKernelGGL(kernel, dim3(unsigned((waves + 3) / 4)), dim3(256), 0, st, sorted, dout, dtable, edge, ends, n,
                           g.chunks, D, int(slabs), vocab, A(scale), int(accumulate));
        return hipGetLastError();
    };
    // 16 bytes a lane, or half of that where a row then fills its last slab better.
    constexpr int V = 16 / int(sizeof(T)), H = sizeof(T) < 8 ? V / 2 : V;
    const uintptr_t at = reinterpret_cast<uintptr_t>(dout) | reinterpret_cast<uintptr_t>(dtable);
    const auto lost = [&](int v) { return (D + kWave * v - 1) / (kWave * v) * (kWave * v) - D; };
    hipError_t e;
    if (D % V != 0 || at % 16 != 0) e = pieces(sum_kernel<T, 1, 4, CH>, 4);
    else if (lost(H) < lost(V)) e = pieces(sum_kernel<T, H, 1, CH>, H);
    else e = pieces(sum_kernel<T, V, 1, CH>, V);
    if (e != hipSuccess) return e;
    const int64_t slabs = (D + kJoinCols * kWave - 1) / (kJoinCols * kWave);
    const int64_t groups = g.chunks * slabs;
    if (!grid_fits(groups, kJoinWaves * kWave)) return hipErrorInvalidValue;
    hipLaunchKernelGGL(join_kernel<T>, dim3(unsigned(groups)), dim3(kJoinWaves * kWave), 0, st, ends, dtable, edge,
                       g.chunks, D, int(slabs), A(scale), int(accumulate));
    return hipGetLastError();
}

template <typename T, typename I>
hipError_t grad(int dtype, const I *ids, const T *dout, T *dtable, double scale, bool accumulate, char *ws, int64_t n,
                int64_t D, int64_t vocab, hipStream_t st) {
    using A = acc_t<T>;
    const GradPlan g = grad_plan(dtype, n, D, vocab);
    uint2 *a = reinterpret_cast<uint2 *>(ws + g.off_a), *b = reinterpret_cast<uint2 *>(ws + g.off_b);
    uint32_t *hist = reinterpret_cast<uint32_t *>(ws + g.off_hist);
    A *edge = reinterpret_cast<A *>(ws + g.off_edge);
    uint2 *ends = reinterpret_cast<uint2 *>(ws + g.off_ends);
    const int64_t table_bytes = accumulate ? 0 : vocab * D * int64_t(sizeof(T));
    char *const table = reinterpret_cast<char *>(dtable);
    // Workgroups that write `bytes` of zeros: enough for every CU, 64 KiB each at least.
    auto fillers = [](int64_t bytes) { return unsigned(std::min<int64_t>((bytes + 65535) / 65536, 2048)); };
    const uint2 *sorted;
    hipError_t e;
    if (n <= kSmall) {
        const Fill f{table, table_bytes};
        hipLaunchKernelGGL(sort_small_kernel<I>, dim3(1 + fillers(table_bytes)), dim3(kSmallWaves * kWave), 0, st, ids,
                           int(n), vocab, g.passes, a, f);
        if ((e = hipGetLastError()) != hipSuccess || n == 0) return e;
        sorted = a;
    } else {
        const int launches = 1 + g.passes;
        int step = 0;
        auto share = [&]() {
            const int64_t lo = table_bytes / launches / 256 * 256 * step;
            const int64_t hi = ++step == launches ? table_bytes : table_bytes / launches / 256 * 256 * step;
            return Fill{table + lo, hi - lo};
        };
        Fill f = share();
        hipLaunchKernelGGL(hist_kernel<I>, dim3(unsigned(g.blocks) + fillers(f.bytes)), dim3(kSortThreads), 0, st, ids,
                           n, vocab, g.passes, g.blocks, g.per, hist, f);
        if ((e = hipGetLastError()) != hipSuccess) return e;
        const uint2 *from = nullptr;
        for (int pass = 0; pass < g.passes; ++pass) {
            uint2 *to = pass % 2 == 0 ? a : b;
            uint32_t *here = hist + int64_t(pass) * g.blocks * kBins;
            f = share();
            hipLaunchKernelGGL(scatter_kernel<I>, dim3(unsigned(g.blocks) + fillers(f.bytes)), dim3(kSortThreads), 0,
                               st, ids, from, n, vocab, pass, g.blocks, g.per, here,
                               pass + 1 < g.passes ? here + int64_t(g.blocks) * kBins : nullptr, to, f);
            if ((e = hipGetLastError()) != hipSuccess) return e;
            from = to;
        }
        sorted = from;
    }
    return g.chunk == 16 ? sums<T, 16>(g, sorted, dout, dtable, edge, ends, scale, accumulate, n, D, vocab, st)
                         : sums<T, 32>(g, sorted, dout, dtable, edge, ends, scale, accumulate, n, D, vocab, st);
}

template <typename Fn> hipError_t typed(int dtype, bool ids64, Fn fn) {
    auto ids = [&](auto *t) { return ids64 ? fn(t, static_cast<int64_t *>(nullptr)) : fn(t, static_cast<int32_t *>(nullptr)); };
    switch (dtype) {
        case CTATTN_F32: return ids(static_cast<float *>(nullptr));
        case CTATTN_BF16: return ids(static_cast<bf16_t *>(nullptr));
        case CTATTN_F16: return ids(static_cast<f16_t *>(nullptr));
        default: return ids(static_cast<double *>(nullptr));
    }
}

int check(const char *fn, int dtype, int id_dtype, int64_t n, int64_t D, int64_t vocab) {
    using capi::fail;
    if (dtype != CTATTN_F32 && dtype != CTATTN_BF16 && dtype != CTATTN_F16 && dtype != CTATTN_F64)
        return fail(hipErrorInvalidValue, "%s: unknown dtype %d (0 = f32, 1 = bf16, 2 = f16, 3 = f64)", fn, dtype);
    if (id_dtype != CTATTN_I32 && id_dtype != CTATTN_I64)
        return fail(hipErrorInvalidValue, "%s: ids must be i32 or i64, got dtype %d", fn, id_dtype);
    if (n < 0 || D < 1 || vocab < 1 || n > 0x7FFFFFFF || D > 0x7FFFFFFF || vocab >= 0x7FFFFFFF)
        return fail(hipErrorInvalidValue, "%s: invalid sizes n=%lld D=%lld vocab=%lld", fn, (long long)n, (long long)D,
                    (long long)vocab);
    const int64_t most = int64_t(1) << 50;
    if (D > most / std::max<int64_t>(n, 1) || D > most / vocab)
        return fail(hipErrorInvalidValue, "%s: tensors too large", fn);
    return 0;
}

// Whether [a, a + an) and [b, b + bn) share a byte.
bool share(const void *a, int64_t an, const void *b, int64_t bn) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return an > 0 && bn > 0 && x < y + uintptr_t(bn) && y < x + uintptr_t(an);
}
int64_t elem_bytes(int dtype) { return dtype == CTATTN_F64 ? 8 : dtype == CTATTN_F32 ? 4 : 2; }
int64_t id_bytes(int id_dtype) { return id_dtype == CTATTN_I64 ? 8 : 4; }

}  // namespace
}  // namespace ctattn

using namespace ctattn;
using ctattn::capi::fail;
using ctattn::capi::finish;
using ctattn::capi::ok;

extern "C" {

int ctattn_embedding_lookup(int dtype, int id_dtype, const void *ids, const void *table, void *out, double scale,
                            int64_t n, int64_t D, int64_t vocab, void *stream) {
    const char *fn = "ctattn_embedding_lookup";
    if (int rc = check(fn, dtype, id_dtype, n, D, vocab)) return rc;
    if (n == 0) return ok();
    if (!ids || !table || !out) return fail(hipErrorInvalidValue, "%s: null pointer", fn);
    const int64_t es = elem_bytes(dtype);
    if (share(out, n * D * es, table, vocab * D * es) || share(out, n * D * es, ids, n * id_bytes(id_dtype)))
        return fail(hipErrorInvalidValue, "%s: out lies on an input's memory", fn);
    hipStream_t st = static_cast<hipStream_t>(stream);
    const hipError_t e = typed(dtype, id_dtype == CTATTN_I64, [&](auto *t, auto *i) {
        using T = std::remove_pointer_t<decltype(t)>;
        using I = std::remove_pointer_t<decltype(i)>;
        return lookup<T, I>(static_cast<const I *>(ids), static_cast<const T *>(table), static_cast<T *>(out), n, D,
                            vocab, scale, st);
    });
    return finish(fn, e, st);
}

int64_t ctattn_embedding_grad_workspace_bytes(int dtype, int64_t n, int64_t D, int64_t vocab) {
    if (check("ctattn_embedding_grad_workspace_bytes", dtype, CTATTN_I32, n, D, vocab) != 0) return -1;
    return n == 0 ? 0 : grad_plan(dtype, n, D, vocab).bytes;
}

int ctattn_embedding_grad(int dtype, int id_dtype, const void *ids, const void *dout, void *dtable, double scale,
                          int accumulate, void *workspace, int64_t workspace_bytes, int64_t n, int64_t D,
                          int64_t vocab, void *stream) {
    const char *fn = "ctattn_embedding_grad";
    if (int rc = check(fn, dtype, id_dtype, n, D, vocab)) return rc;
    if (!dtable) return fail(hipErrorInvalidValue, "%s: null dtable pointer", fn);
    if (n > 0 && (!ids || !dout)) return fail(hipErrorInvalidValue, "%s: null ids/dout pointer", fn);
    const int64_t es = elem_bytes(dtype);
    if (share(dtable, vocab * D * es, dout, n * D * es) || share(dtable, vocab * D * es, ids, n * id_bytes(id_dtype)))
        return fail(hipErrorInvalidValue, "%s: dtable lies on an input's memory", fn);
    const int64_t need = n == 0 ? 0 : grad_plan(dtype, n, D, vocab).bytes;
    if (need > 0 && (!workspace || workspace_bytes < need))
        return fail(hipErrorInvalidValue, "%s: workspace too small (%lld bytes, %lld needed)", fn,
                    (long long)workspace_bytes, (long long)need);
    if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
        return fail(hipErrorInvalidValue, "%s: workspace must be 16-byte aligned", fn);
    if (n == 0 && accumulate) return ok();
    hipStream_t st = static_cast<hipStream_t>(stream);
    const hipError_t e = typed(dtype, id_dtype == CTATTN_I64, [&](auto *t, auto *i) {
        using T = std::remove_pointer_t<decltype(t)>;
        using I = std::remove_pointer_t<decltype(i)>;
        return grad<T, I>(dtype, static_cast<const I *>(ids), static_cast<const T *>(dout), static_cast<T *>(dtable),
                          scale, accumulate != 0, static_cast<char *>(workspace), n, D, vocab, st);
    });
    return finish(fn, e, st);
}

}  // extern "C"
