// Next tokens from logits and given random numbers: temperature, top-k, top-p and min-p.
//
// With M the row's largest logit and w_i = exp((x_i - M) / T) the tokens are ranked by (x, then the lower id), a run
// of the first ranks is kept (ctattn.h), and the token is the first id, in the order of ids, at which the sum of kept w
// passes u times their whole sum.  A draw near a border of two ids must not depend on the order of a sum, so w and
// its sums are held in 64 bits: 2^e by a polynomial of degree 9 of e's fraction, 4e-14 off (a token changes where u is
// that near a border).
//
// A row is pieces of 512 logits, 8 a lane of a wave.  One pass over the logits, spread over the chip, leaves each
// piece's sum of w relative to its maximum, and the maxima of its quarters; a workgroup a row does the rest.  A draw from
// all tokens then needs the pieces' sums and one piece.  Top-k and most nuclei lie among a few hundred tokens: the R-th
// largest of these maxima is a bound that at least R tokens reach, so only quarters that reach it are read again, and
// what reaches it is ranked in LDS (with a maximum a piece instead, 200 of 256 pieces were read for 200 ranks: 27 us of
// the workgroup's 50).  Where that is not enough (a nucleus of thousands of tokens, more than 2048 at the bound) the row is
// put off: all workgroups together count its tokens and sum its w in bins over x, and list those of the border's bin; its
// own workgroup then finds the border in bins over that bin's keys.  Sums that atomics make are of 64-bit integers, whose
// order does not matter.  Few cases are left to a workgroup alone, in as many histograms as they take: top-k beyond the bound
// together with top-p, thousands of equal logits.  Slow are rows with few finite logits: where fewer runs of 128 hold one than
// ranks are asked for the bound is -inf, and every token is counted (256 rows, 20 finite logits each: top-k 50 666 us instead of
// 55, top-p 0.9 349 instead of 173).
//
// Measured, 256 rows of 131072 bf16 logits: the first pass 31 us (2.1 TB/s, of 13 us at 5.1: 18 64-bit operations a logit, but a
// table of 64 roots in LDS, which spares 13 of them, takes 30; around them are two 64-bit divisions a wave and a wave's
// reduction of a maximum and a 64-bit sum for every 8 logits a lane, not timed apart), without filters 38 in all, top-k 50 54 and top-k 200
// 62 (the row's workgroup is latencies: LDS, barriers, a few loads one after the other), each row its own parameters 107 to
// 113, where 18 rows are put off (10 us of bins, 16 of lists, 27 of borders; by their own workgroups alone over 200).  One row
// of 50257, top-k 50: 3 + 18 us.  1024 threads a row instead of 512 cost 20 us more.
#include "attn_common.h"
#include "attn_launch.h"
#include "capi_bytes.h"
#include "capi_util.h"
#include "ctattn.h"
#include "row_vec.h"

#include <algorithm>
#include <math.h>

namespace ctattn {
namespace {

constexpr int kPiece = 512;
constexpr int kMaxPieces = 1024;  // the pieces' sums stay in LDS
constexpr int kParts = 4;         // of a piece, the 128 logits of 16 lanes, each with a maximum of its own
constexpr int kThreads = 512;     // of a row's workgroup
constexpr int kWaves = kThreads / kWave;
constexpr int kList = 2048;       // tokens ranked in LDS
constexpr int kBins = 1024;
constexpr double kLog2e64 = 1.4426950408889634074;

// A bin that holds a border: its keys, how many tokens and how much w are above it, and the w that the border leaves above itself.
struct BorderBin {
    uint32_t lo, hi;
    int64_t above;
    double base, target;
};
// A row whose border is found by all of the chip: tokens and w (in integers) of bins over x, and the tokens of the border's bin.
struct Wide {
    BorderBin border;
    uint64_t mass[kBins];
    uint64_t list[kList];
    uint32_t cnt[kBins];
    double whole;
    float top;
    int32_t count;
};

struct SampleArgs {
    const void *logits;
    const float *u;
    const float *temperature, *top_p, *min_p;  // of each row, or null: the numbers below
    const int32_t *top_k;
    double temperature_all, top_p_all, min_p_all;
    int64_t top_k_all;
    int64_t *tokens;
    float *logprobs;
    float *part_max;  // [rows][pieces][kParts], null: the row's workgroup makes them itself
    double *piece_sum;
    int64_t stride;
    int vocab, pieces, each;  // each: pieces of a wave of the first pass
    Wide *wide;               // of the rows put off, up to `most` of them
    int32_t *put_off;         // their number, and the rows
    int most;
};

// exp((x - m) / t) as 2^((x - m) s).  Below `floor` it is 0.
struct Scale {
    double s, floor;
};
struct Row {
    double t;  // the temperature of w: 1 for a greedy row
    Scale scale;
    bool greedy;
};
__device__ __forceinline__ Row row_of(const SampleArgs &a, int64_t row) {
    const double t = a.temperature != nullptr ? double(a.temperature[row]) : a.temperature_all;
    Row r;
    r.greedy = !(t > 0.0);
    r.t = r.greedy ? 1.0 : t;
    r.scale.s = fmin(fmax(kLog2e64 / r.t, 1e-290), 1e290);  // an infinite t too leaves -inf below the floor, and 0 s is 0
    r.scale.floor = -1100.0 / r.scale.s;
    return r;
}

// w for finite m: 1 where x is m, 0 for x = -inf.  (2^f - 1) / f on [-1/2, 1/2] is a polynomial of degree 8 through its
// values at the Chebyshev points, so that 2^0 is 1 exactly.  Adding 1.5 2^52 rounds to an integer, in the low word.
__device__ __forceinline__ double weight_finite(float x, double m, const Scale &c) {
    constexpr double kMagic = 6755399441055744.0;
    const double d = fmax(double(x) - m, c.floor);
    const double t = fma(d, c.s, kMagic);
    const double f = fma(d, c.s, kMagic - t);
    double p = 1.0203121063391729e-07;
    p = fma(p, f, 1.3255224878668817e-06);
    p = fma(p, f, 1.525268684626772e-05);
    p = fma(p, f, 0.00015403455852453838);
    p = fma(p, f, 0.0013333558179043112);
    p = fma(p, f, 0.0096181291594025584);
    p = fma(p, f, 0.055504108664760424);
    p = fma(p, f, 0.24022650695812989);
    p = fma(p, f, 0.69314718055994529);
    return ldexp(fma(p, f, 1.0), __double2loint(t));
}
// An infinite m is the value of all that is not 0.
__device__ __forceinline__ double weight(float x, float m, const Scale &c) {
    return m == INFINITY ? (x == m ? 1.0 : 0.0) : weight_finite(x, double(m), c);
}

// What a row draws from: the first k ranks, `share` of their w (above 1: all), w of at least `least`.
struct Choice {
    int64_t k;
    double share, least;
    float u;
};
__device__ __forceinline__ Choice choice_of(const SampleArgs &a, int64_t row, bool greedy) {
    Choice c;
    c.u = a.u != nullptr ? a.u[row] : 0.f;
    if (!(c.u >= 0.f)) c.u = 0.f;
    c.k = a.top_k != nullptr ? int64_t(a.top_k[row]) : a.top_k_all;
    const double p = a.top_p != nullptr ? double(a.top_p[row]) : a.top_p_all;
    c.share = p < 1.0 ? p : 2.0;
    c.least = a.min_p != nullptr ? double(a.min_p[row]) : a.min_p_all;
    if (!(c.least > 0.0)) c.least = 0.0;
    if (c.k <= 0 || c.k > a.vocab) c.k = a.vocab;
    if (greedy || c.share <= 0.0 || c.least > 1.0) {
        c.k = 1;
        c.share = 2.0;
        c.least = 0.0;
    }
    return c;
}
__device__ __forceinline__ void finish_row(const SampleArgs &a, int64_t row, int64_t token, float value, float top, double t, double whole) {
    a.tokens[row] = token;
    const double d = value == top ? 0.0 : (double(value) - double(top)) / t;
    a.logprobs[row] = float(d - log(whole));
}

// A double's two words of the lane that DPP control CTRL names, and the sum over a wave in every lane, as wave_sum_dpp.
template <int CTRL> __device__ __forceinline__ double dpp64(double x) {
    return __hiloint2double(__builtin_amdgcn_update_dpp(0, __double2hiint(x), CTRL, 0xf, 0xf, true),
                            __builtin_amdgcn_update_dpp(0, __double2loint(x), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ double wave_sum64(double x) {
    x += dpp64<0xB1>(x);
    x += dpp64<0x4E>(x);
    x += dpp64<0x141>(x);
    x += dpp64<0x140>(x);
    uint32_t lo = uint32_t(__double2loint(x)), hi = uint32_t(__double2hiint(x));
    auto l = __builtin_amdgcn_permlane16_swap(lo, lo, false, false);
    auto h = __builtin_amdgcn_permlane16_swap(hi, hi, false, false);
    x = __hiloint2double(int(h[0]), int(l[0])) + __hiloint2double(int(h[1]), int(l[1]));
    lo = uint32_t(__double2loint(x));
    hi = uint32_t(__double2hiint(x));
    l = __builtin_amdgcn_permlane32_swap(lo, lo, false, false);
    h = __builtin_amdgcn_permlane32_swap(hi, hi, false, false);
    return __hiloint2double(int(h[0]), int(l[0])) + __hiloint2double(int(h[1]), int(l[1]));
}
// The maximum over a wave of what the lanes of each 16 have in common.
__device__ __forceinline__ float max_of_rows(float x) {
    uint32_t b = __float_as_uint(x);
    auto r = __builtin_amdgcn_permlane16_swap(b, b, false, false);
    b = __float_as_uint(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
    r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
template <typename A> __device__ __forceinline__ A wave_scan(A x) {
    const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
        const A y = __shfl_up(x, off, kWave);
        if (lane >= off) x += y;
    }
    return x;
}

// 8 logits of a lane; past the row's end and where there is none -inf; -0 becomes 0.
template <typename T> struct Eight {
    static constexpr int N = sizeof(T) == 2 ? 1 : 2;
    gran_raw g[N];
    int c0;
    __device__ __forceinline__ void load(const T *row, int piece, int vocab) {
        load_at(row, piece * kPiece + int(threadIdx.x & (kWave - 1)) * 8, (piece + 1) * kPiece <= vocab, vocab);
    }
    __device__ __forceinline__ void load_at(const T *row, int at, bool full, int vocab) {
        c0 = at;
        if (full) {
#pragma unroll
            for (int i = 0; i < N; ++i) g[i] = *reinterpret_cast<const typename Gran<T>::raw_t *>(row + c0 + i * Gran<T>::EPC);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) g[i] = Gran<T>::load_tail(row, c0 + i * Gran<T>::EPC, vocab, -INFINITY);
        }
    }
    // As they are, NaN and -0 too.
    __device__ __forceinline__ void get_raw(float (&x)[8]) const {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = Gran<T>::get(g[e / Gran<T>::EPC], e % Gran<T>::EPC);
    }
    __device__ __forceinline__ void get(float (&x)[8]) const {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float y = Gran<T>::get(g[e / Gran<T>::EPC], e % Gran<T>::EPC);
            x[e] = fmaxf(y, -INFINITY) + 0.f;  // fmaxf takes the number of a NaN and a number
        }
    }
};

// Keys in the order of the values.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x);
    return b ^ (b >> 31 ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) {
    return __uint_as_float(k ^ (k >> 31 ? 0x80000000u : 0xFFFFFFFFu));
}

// The maxima of a piece's parts in each lane of theirs, and its sum of w relative to the whole piece's maximum in every lane,
// from raw values: fmaxf and fmax take the number of a NaN and a number, so that a NaN has the w of -inf.
__device__ __forceinline__ void piece_stats(const float (&x)[8], const Scale &c, float &part, double &s) {
    float m = -INFINITY;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = fmaxf(m, x[e]);
    m = fmaxf(m, dpp<0xB1>(m));
    m = fmaxf(m, dpp<0x4E>(m));
    m = fmaxf(m, dpp<0x141>(m));
    part = fmaxf(m, dpp<0x140>(m)) + 0.f;
    m = max_of_rows(part);
    s = 0.0;
    if (m == -INFINITY) return;
    if (m == INFINITY) {
#pragma unroll
        for (int e = 0; e < 8; ++e) s += x[e] == m ? 1.0 : 0.0;
    } else {
        const double md = double(m);
#pragma unroll
        for (int e = 0; e < 8; ++e) s += weight_finite(x[e], md, c);
    }
    s = wave_sum64(s);
}

template <typename T> __global__ __launch_bounds__(256) void sample_stats_kernel(SampleArgs a) {
    const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
    const int64_t row = blockIdx.y;
    const T *x = static_cast<const T *>(a.logits) + row * a.stride;
    const Scale scale = row_of(a, row).scale;
    const int p0 = (blockIdx.x * 4 + wave) * a.each, p1 = p0 + a.each < a.pieces ? p0 + a.each : a.pieces;
    if (a.put_off != nullptr && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) a.put_off[0] = 0;
    if (p0 >= p1) return;
    Eight<T> now, next;
    next.load(x, p0, a.vocab);
    for (int p = p0; p < p1; ++p) {
        now = next;
        if (p + 1 < p1) next.load(x, p + 1, a.vocab);
        float v[8], part;
        double s;
        now.get_raw(v);
        piece_stats(v, scale, part, s);
        if (lane % 16 == 0) a.part_max[(row * a.pieces + p) * kParts + lane / 16] = part;
        if (lane == 0) a.piece_sum[row * a.pieces + p] = s;
    }
}

struct Shared {
    float pm[kMaxPieces];
    double ps[kMaxPieces];
    union {
        struct {
            uint32_t cnt[kBins];
            uint64_t mass[kBins];
        };
        uint64_t comp[kList];  // (key, ~id)
    };
    union {
        double w[kList];
        float part_max[kMaxPieces * kParts];  // until tokens are listed
    };
    union {
        uint64_t sums[kMaxPieces];
        uint16_t wanted[kMaxPieces * kParts];  // parts to list tokens from
    };
    uint32_t sub[kBins];
    uint64_t scratch[2 * kWaves];
    int32_t found, count;
    int32_t place;  // of a row put off; not `count`, which waves may still be reading as the list's length then
    uint32_t key;
    int64_t token;
};

// Running sums of a[0 .. n), n up to N, in place, in one order.
template <int N, typename A> __device__ __forceinline__ void scan_array(A *a, int n, uint64_t *scratch) {
    constexpr int Q = (N + kThreads - 1) / kThreads;
    A *waves = reinterpret_cast<A *>(scratch);
    const int t = threadIdx.x, lane = t & (kWave - 1), wave = t / kWave;
    const int q = (n + kThreads - 1) / kThreads, i0 = t * q;
    A r[Q];
#pragma unroll
    for (int i = 0; i < Q; ++i) r[i] = i < q && i0 + i < n ? a[i0 + i] : A(0);
#pragma unroll
    for (int i = 1; i < Q; ++i) r[i] += r[i - 1];
    const A s = wave_scan(r[Q - 1]);
    if (lane == kWave - 1) waves[wave] = s;
    __syncthreads();
    A run = __shfl_up(s, 1, kWave);
    if (lane == 0) run = 0;
    A before = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) before += w < wave ? waves[w] : A(0);
    run += before;
#pragma unroll
    for (int i = 0; i < Q; ++i)
        if (i < q && i0 + i < n) a[i0 + i] = run + r[i];
    __syncthreads();
}
// The first i of [0, n) that holds, or n, in every thread.
template <typename Fn> __device__ __forceinline__ int first_of(int n, Shared &sh, Fn holds) {
    __syncthreads();
    if (threadIdx.x == 0) sh.found = n;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads)
        if (holds(i)) {
            atomicMin(&sh.found, i);
            break;
        }
    __syncthreads();
    return sh.found;
}
// The wanted pieces, spread over the waves, four pieces' loads ahead; fn(piece, the lane's eight).
template <typename T, typename Want, typename Fn>
__device__ __forceinline__ void each_piece(const T *x, int pieces, int vocab, Want want, Fn fn) {
    constexpr int N = 4;
    static_assert(kMaxPieces <= 2 * kWave * kWaves, "two masks a wave");
    // Which of pieces wave, wave + kWaves, .. are wanted, a bit each.
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x & (kWave - 1);
    const int p0 = wave + kWaves * lane, p1 = p0 + kWaves * kWave;
    uint64_t mask = __ballot(p0 < pieces && want(p0)), rest = __ballot(p1 < pieces && want(p1));
    int from = wave;
    Eight<T> ahead[N];
    int at[N];
    const auto fetch = [&](int i) {
        if (mask == 0) {
            mask = rest;
            rest = 0;
            from = wave + kWaves * kWave;
        }
        at[i] = -1;
        if (mask == 0) return;
        at[i] = from + kWaves * (__ffsll((unsigned long long)mask) - 1);
        mask &= mask - 1;
        ahead[i].load(x, at[i], vocab);
    };
#pragma unroll
    for (int i = 0; i < N; ++i) fetch(i);
    while (at[0] >= 0) {
        const Eight<T> now = ahead[0];
        const int here = at[0];
#pragma unroll
        for (int i = 0; i + 1 < N; ++i) {
            ahead[i] = ahead[i + 1];
            at[i] = at[i + 1];
        }
        fetch(N - 1);
        fn(here, now);
    }
}

// 1024 bins over x, 32 to a factor of two in w; the first holds the largest, the last all of the rest.
struct Bins {
    float m, by;
    __device__ __forceinline__ int of(float v) const { return v == m ? 0 : int(fminf((m - v) * by, float(kBins - 1))); }
    // The lowest key of a bin <= at_most: the bins fall with the key.  A wave's lanes try 64 keys at a time.
    __device__ __forceinline__ uint32_t edge(int at_most) const {
        const uint32_t lane = threadIdx.x & (kWave - 1);
        uint32_t p = key_of(-INFINITY), q = key_of(m);  // it is one of p .. q
        while (p < q) {
            const uint32_t step = q - p < kWave ? 1u : (q - p) / kWave, key = p + lane * step;
            const uint64_t in = __ballot(key >= q || of(value_of(key)) <= at_most);
            if (in == 0) {
                p += (kWave - 1) * step + 1;
                continue;
            }
            const uint32_t first = uint32_t(__ffsll((unsigned long long)in) - 1), at = p + first * step;
            if (first > 0) p = at - step + 1;
            q = at < q ? at : q;
        }
        return q;
    }
    __device__ uint32_t lowest(int b) const { return edge(b); }
    __device__ uint32_t highest(int b) const { return b > 0 ? edge(b - 1) - 1 : key_of(m); }
};
__device__ __forceinline__ Bins bins_of(float m, const Scale &scale) { return {m, float(scale.s * 32.0)}; }
// w in integers, whose sums do not depend on their order: the whole row's sum takes 62 bits, half a step a token is lost.
struct Fixed {
    double fix, unfix;
    __device__ __forceinline__ uint64_t of(double w) const { return uint64_t(fma(w, fix, 0.5)); }
    __device__ __forceinline__ double sum(uint64_t x) const { return double(x) * unfix; }
};
__device__ __forceinline__ Fixed fixed_of(double whole) {
    const int bits = ilogb(whole) + 1;
    return {ldexp(1.0, 62 - bits), ldexp(1.0, bits - 62)};
}

// Which tokens a draw takes: keys above `key` and the first `ties` ids of that key, of w at least `least`.
struct Kept {
    uint32_t key;
    int64_t ties;
    double least;
};

// The first token of a piece at which `base` and the sum of kept w pass `target` (the last with any, where rounding
// lets none; none, where the piece has none), by one wave.  `before`: tokens of the border's key in earlier pieces.
template <typename T>
__device__ __forceinline__ void draw_in_piece(const T *x, int piece, int vocab, float m, const Scale &scale, const Kept &k, int64_t before,
                              double base, double target, Shared &sh) {
    const int lane = threadIdx.x & (kWave - 1);
    Eight<T> g;
    float v[8];
    g.load(x, piece, vocab);
    g.get(v);
    int ties = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) ties += key_of(v[e]) == k.key ? 1 : 0;
    int upto = ties;
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
        const int y = __shfl_up(upto, off, kWave);
        if (lane >= off) upto += y;
    }
    int64_t rank = before + upto - ties;
    double w[8], s = 0.0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint32_t key = key_of(v[e]);
        const double y = weight(v[e], m, scale);
        const bool in = g.c0 + e < vocab && v[e] != -INFINITY && (key > k.key || (key == k.key && rank < k.ties)) && y >= k.least;
        if (key == k.key) ++rank;
        w[e] = in ? y : 0.0;
        s += w[e];
    }
    double sum = s;
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
        const double y = __shfl_up(sum, off, kWave);
        if (lane >= off) sum += y;
    }
    const uint64_t past = __ballot(base + sum > target && s > 0.0), some = __ballot(s > 0.0);
    const int at = past != 0 ? __ffsll((unsigned long long)past) - 1 : 63 - __clzll((long long)some);
    if (lane == at) {
        double run = base + (sum - s);
        int last = -1;
        bool done = false;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (done || !(w[e] > 0.0)) continue;
            run += w[e];
            last = e;
            done = past != 0 && run > target;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e == last) {
                sh.token = g.c0 + e;
                sh.key = key_of(v[e]);
            }
    }
}

// Sorts the n listed tokens (comp) by rank, and puts their weights beside them (w).  Few by counting those before each,
// many by a bitonic network (2048: 66 steps, 25 us; counting takes over 60).
__device__ __forceinline__ void sort_list(Shared &sh, int n, float m, const Scale &scale) {
    const int t = threadIdx.x;
    if (n <= kThreads) {
        const uint64_t mine = t < n ? sh.comp[t] : 0;
        int rank = 0;
        if (t < n) {
#pragma unroll 8
            for (int j = 0; j < n; ++j) rank += sh.comp[j] > mine ? 1 : 0;
        }
        __syncthreads();
        if (t < n) sh.comp[rank] = mine;
    } else {
        int size = 2 * kThreads;
        while (size < n) size *= 2;
        for (int i = n + t; i < size; i += kThreads) sh.comp[i] = 0;
        for (int k = 2; k <= size; k *= 2)
            for (int j = k / 2; j > 0; j /= 2) {
                __syncthreads();
                for (int q = t; q < size / 2; q += kThreads) {
                    const int i = 2 * (q & ~(j - 1)) + (q & (j - 1));
                    const uint64_t x = sh.comp[i], y = sh.comp[i + j];
                    if ((x < y) == ((i & k) == 0)) {
                        sh.comp[i] = y;
                        sh.comp[i + j] = x;
                    }
                }
            }
    }
    __syncthreads();
    for (int i = t; i < n; i += kThreads) sh.w[i] = weight(value_of(uint32_t(sh.comp[i] >> 32)), m, scale);
    __syncthreads();
}
__device__ __forceinline__ uint32_t list_key(const Shared &sh, int i) { return uint32_t(sh.comp[i] >> 32); }
__device__ __forceinline__ int list_id(const Shared &sh, int i) { return int(~uint32_t(sh.comp[i])); }

// The first `keep` listed tokens are kept: the border that says so, and their w, where it is at least `least`, added to
// their pieces' sums in ps, through sums.  In 64-bit integers (the whole row's sum takes 62 bits), whose sum does not
// depend on the order of the atomics.
__device__ __forceinline__ void keep_listed(Shared &sh, int n, int keep, int pieces, float m, const Scale &scale, double whole, Kept &kept) {
    const int t = threadIdx.x;
    const uint32_t key = list_key(sh, keep - 1);
    const int first = first_of(n, sh, [&](int i) { return list_key(sh, i) == key; });
    kept.key = key;
    kept.ties = keep - first;
    const Fixed f = fixed_of(whole);
    for (int i = t; i < keep; i += kThreads) {
        const double w = weight(value_of(list_key(sh, i)), m, scale);
        if (w >= kept.least)
            atomicAdd(reinterpret_cast<unsigned long long *>(&sh.sums[list_id(sh, i) / kPiece]), (unsigned long long)f.of(w));
    }
    __syncthreads();
    for (int p = t; p < pieces; p += kThreads) sh.ps[p] += f.sum(sh.sums[p]);
    __syncthreads();
}
// Lists a piece's tokens with lo <= key <= hi; few lanes have any.  The order in the list is arbitrary.
__device__ __forceinline__ void append(int32_t *count, uint64_t *list, const float (&v)[8], int c0, int vocab, uint32_t lo, uint32_t hi) {
    int in = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint32_t key = key_of(v[e]);
        in |= int(c0 + e < vocab) & int(key >= lo) & int(key <= hi) ? 1 << e : 0;
    }
    if (in == 0) return;
    int at = atomicAdd(count, __popc(in));
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (in >> e & 1) {
            if (at < kList) list[at] = uint64_t(key_of(v[e])) << 32 | uint32_t(~(c0 + e));
            ++at;
        }
}
// Lists the tokens with lo <= key <= hi of the wanted pieces; their number, which may pass the list's length.
template <typename T, typename Want>
__device__ __forceinline__ int collect(const T *x, int pieces, int vocab, uint32_t lo, uint32_t hi, Want want, Shared &sh) {
    __syncthreads();
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    each_piece(x, pieces, vocab, want, [&](int, const Eight<T> &g) {
        float v[8];
        g.get(v);
        append(&sh.count, sh.comp, v, g.c0, vocab, lo, hi);
    });
    __syncthreads();
    return sh.count;
}

struct Border {
    uint32_t key;
    int64_t ties;   // tokens of that key that are kept
    double mass;    // sum of w of all that are kept
};

// The border of a run of ranks: the first `want` of them (by_count), or those whose sum of w before them is less than
// `share` of the whole row's (by_mass: share of `of`, or of the row where that is negative).
template <typename T>
__device__ __forceinline__ Border find_border(const T *x, const SampleArgs &a, float m, const Scale &scale, double whole, bool by_count, int64_t want,
                              double share, double of, Shared &sh) {
    const Fixed f = fixed_of(whole);
    const Bins bins = bins_of(m, scale);
    uint32_t lo = 0, hi = 0xFFFFFFFFu;
    int shift = -1;  // bins over x first, then over keys
    int64_t before = 0;
    uint64_t mass = 0;
    double target = of < 0.0 ? 0.0 : share * of;
    for (;;) {
        __syncthreads();
        for (int i = threadIdx.x; i < kBins; i += kThreads) {
            sh.cnt[i] = 0;
            sh.mass[i] = 0;
        }
        __syncthreads();
        each_piece(x, a.pieces, a.vocab, [](int) { return true; }, [&](int, const Eight<T> &g) {
            float v[8];
            g.get(v);
            const int c0 = g.c0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t key = key_of(v[e]);
                if (c0 + e < a.vocab && key >= lo && key <= hi) {
                    const int b = shift < 0 ? bins.of(v[e]) : int((hi - key) >> shift);
                    atomicAdd(&sh.cnt[b], 1u);
                    const uint64_t w = f.of(weight(v[e], m, scale));
                    if (w != 0) atomicAdd(reinterpret_cast<unsigned long long *>(&sh.mass[b]), (unsigned long long)w);
                }
            }
        });
        __syncthreads();
        scan_array<kBins>(sh.cnt, kBins, sh.scratch);
        scan_array<kBins>(sh.mass, kBins, sh.scratch);
        if (shift < 0 && !by_count && of < 0.0) target = share * (f.sum(sh.mass[kBins - 1]));
        int b = first_of(kBins, sh, [&](int i) {
            return by_count ? before + int64_t(sh.cnt[i]) >= want : f.sum(mass + sh.mass[i]) >= target;
        });
        if (b >= kBins) b = first_of(kBins, sh, [&](int i) { return sh.cnt[i] == sh.cnt[kBins - 1]; });  // the last with any
        const int64_t in = int64_t(sh.cnt[b]) - (b > 0 ? int64_t(sh.cnt[b - 1]) : 0);
        if (b > 0) {
            before += sh.cnt[b - 1];
            mass += sh.mass[b - 1];
        }
        if (shift < 0) {
            lo = bins.lowest(b);
            hi = bins.highest(b);
        } else {
            hi -= uint32_t(b) << shift;
            const uint32_t width = (1u << shift) - 1;
            lo = hi - lo > width ? hi - width : lo;
        }
        if (lo >= hi) {
            const double w = weight(value_of(hi), m, scale);
            int64_t ties = want - before;
            if (!by_count) {
                // As many as have less than the target before them.
                const double need = (target - f.sum(mass)) / w;
                ties = need < double(in) ? int64_t(ceil(need)) : in;
            }
            ties = ties < 1 ? 1 : ties > in ? in : ties;
            return {hi, ties, f.sum(mass) + double(ties) * w};
        }
        if (in <= kList) break;
        const int width = 32 - __clz(hi - lo);
        shift = width > 10 ? width - 10 : 0;
    }
    int n = collect(x, a.pieces, a.vocab, lo, hi, [](int) { return true; }, sh);
    n = n < kList ? n : kList;
    sort_list(sh, n, m, scale);
    scan_array<kList>(sh.w, n, sh.scratch);
    const double base = f.sum(mass);
    int j = by_count ? int(want - before) - 1 : first_of(n, sh, [&](int i) { return base + sh.w[i] >= target; });
    j = j < 0 ? 0 : j >= n ? n - 1 : j;
    const uint32_t key = list_key(sh, j);
    const int first = first_of(n, sh, [&](int i) { return list_key(sh, i) == key; });
    const Border out{key, j - first + 1, base + sh.w[j]};
    __syncthreads();
    return out;
}

// Of the n listed tokens, all with lo <= key <= hi, leaves those of the one of 1024 bins over the keys that holds the border:
// the first `want` listed, or those with less than `target` of w before them.  The w of the ones above are added to their pieces in
// sums, their number and w to `above` and `base`.  Returns how many are left.
__device__ __forceinline__ int narrow(Shared &sh, int n, uint32_t lo, uint32_t hi, bool by_count, int64_t want, double target, double least,
                                      float m, const Scale &scale, double whole, int64_t &above, double &base) {
    const int t = threadIdx.x;
    const int width = 32 - __clz(int((hi - lo) | 1u)), shift = width > 10 ? width - 10 : 0;
    const Fixed f = fixed_of(whole);
    uint64_t *const mass = reinterpret_cast<uint64_t *>(sh.w);
    for (int i = t; i < kBins; i += kThreads) {
        sh.sub[i] = 0;
        mass[i] = 0;
    }
    __syncthreads();
    constexpr int Q = kList / kThreads;
    uint64_t mine[Q], fixed[Q];
    int bin[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const int i = t + q * kThreads;
        mine[q] = fixed[q] = 0;
        bin[q] = kBins;
        if (i >= n) continue;
        mine[q] = sh.comp[i];
        const double w = weight(value_of(uint32_t(mine[q] >> 32)), m, scale);
        fixed[q] = f.of(w);
        bin[q] = int((hi - uint32_t(mine[q] >> 32)) >> shift);
        atomicAdd(&sh.sub[bin[q]], 1u);
        atomicAdd(reinterpret_cast<unsigned long long *>(&mass[bin[q]]), (unsigned long long)fixed[q]);
        if (!(w >= least)) fixed[q] = 0;
    }
    __syncthreads();
    scan_array<kBins>(sh.sub, kBins, sh.scratch);
    scan_array<kBins>(mass, kBins, sh.scratch);
    const int b = first_of(kBins, sh, [&](int i) {
        return by_count ? above + int64_t(sh.sub[i]) >= want : base + f.sum(mass[i]) >= target;
    });
    if (b >= kBins) return 0;
    if (b > 0) {
        above += sh.sub[b - 1];
        base += f.sum(mass[b - 1]);
    }
    if (t == 0) sh.count = 0;
    __syncthreads();
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        if (bin[q] < b)
            atomicAdd(reinterpret_cast<unsigned long long *>(&sh.sums[int(~uint32_t(mine[q])) / kPiece]), (unsigned long long)fixed[q]);
        if (bin[q] == b) sh.comp[atomicAdd(&sh.count, 1)] = mine[q];
    }
    __syncthreads();
    return sh.count;
}

// A value that at least `rank` of v[0 .. n) reach, n up to N, and few more: the upper BITS of the key of that rank, 8 at a
// time in histograms of hist[], 256 numbers of zero for each.  Every wave finds the digits for itself.
template <int BITS, int N> __device__ __forceinline__ float rank_bound(const float *v, int n, int rank, uint32_t *hist) {
    constexpr int Q = N / kThreads;
    const int t = threadIdx.x, lane = t & (kWave - 1);
    uint32_t prefix = 0;
#pragma unroll
    for (int shift = 24; shift >= 32 - BITS; shift -= 8, hist += 256) {
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            if (q * kThreads + t >= n) break;
            const uint32_t key = key_of(v[q * kThreads + t]);
            if (shift == 24 || key >> (shift + 8) == prefix) atomicAdd(&hist[255 - (key >> shift & 255)], 1u);
        }
        __syncthreads();
        uint32_t c[4], sum = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) sum += c[i] = hist[4 * lane + i];
        uint32_t run = wave_scan(sum);
        const uint64_t past = __ballot(run >= uint32_t(rank));
        const int at = past != 0 ? __ffsll((unsigned long long)past) - 1 : kWave - 1;
        run -= sum;
        int digit = 4 * lane + 3, left = rank - int(run);
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (digit == 4 * lane + 3) {
                if (left <= int(c[i])) digit = 4 * lane + i;
                else left -= int(c[i]);
            }
        prefix = prefix << 8 | uint32_t(255 - __builtin_amdgcn_readlane(digit, at));
        rank = __builtin_amdgcn_readlane(left, at);
    }
    const uint32_t key = prefix << (32 - BITS), none = key_of(-INFINITY);
    return value_of(key > none ? key : none);
}
// Lists the tokens that reach the bound, from the parts that hold any, 16 lanes a part; their number, which may pass the list's
// length.
template <typename T> __device__ __forceinline__ int collect_top(const T *x, int parts, int vocab, float bound, Shared &sh) {
    constexpr int N = 16 / sizeof(T), G = kThreads / 16, P = kPiece / kParts;
    const int t = threadIdx.x, lane = t & (kWave - 1);
    __syncthreads();
    if (t == 0) sh.count = sh.found = 0;
    __syncthreads();
    for (int i0 = 0; i0 < parts; i0 += kThreads) {
        const bool want = i0 + t < parts && (bound == -INFINITY || sh.part_max[i0 + t] >= bound);
        const uint64_t mask = __ballot(want);
        if (mask == 0) continue;
        int at = 0;
        if (lane == 0) at = atomicAdd(&sh.found, __popcll(mask));
        at = __builtin_amdgcn_readfirstlane(at) + __popcll(mask & ((uint64_t(1) << lane) - 1));
        if (want) sh.wanted[at] = uint16_t(i0 + t);
    }
    __syncthreads();
    const int n = sh.found;
    const uint32_t lo = key_of(bound);
    for (int i0 = t / 16; i0 < n; i0 += N * G) {
        Eight<T> g[N];
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i0 + i * G < n) {
                const int part = sh.wanted[i0 + i * G];
                g[i].load_at(x, part * P + (t & 15) * 8, (part + 1) * P <= vocab, vocab);
            }
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i0 + i * G < n) {
                float v[8];
                g[i].get(v);
                append(&sh.count, sh.comp, v, g[i].c0, vocab, lo, 0xFFFFFFFFu);
            }
    }
    __syncthreads();
    return sh.count;
}

// What the kernels of a workgroup a row share.
template <typename T> struct RowWork {
    const SampleArgs &a;
    Shared &sh;
    const int64_t row;
    const T *const x;
    const Row r;
    const Choice c;
    const int np, vocab, t, lane;
    float top;
    double whole;

    __device__ __forceinline__ RowWork(const SampleArgs &a_, Shared &sh_, int64_t row_)
        : a(a_), sh(sh_), row(row_), x(static_cast<const T *>(a_.logits) + row_ * a_.stride), r(row_of(a_, row_)),
          c(choice_of(a_, row_, r.greedy)), np(a_.pieces), vocab(a_.vocab), t(threadIdx.x), lane(threadIdx.x & (kWave - 1)) {}

    __device__ __forceinline__ double w_of(float v) const { return weight(v, top, r.scale); }
    __device__ __forceinline__ void finish(int64_t token, float value) const { finish_row(a, row, token, value, top, r.t, whole); }

    // The first pass's maxima of the pieces, and of their parts where asked.
    __device__ __forceinline__ void load_maxima(float *parts) const {
        static_assert(kParts == 4, "16 bytes a piece");
        const float4 *const from = reinterpret_cast<const float4 *>(a.part_max) + row * np;
        for (int p = t; p < np; p += kThreads) {
            const float4 m = from[p];
            sh.pm[p] = fmaxf(fmaxf(m.x, m.y), fmaxf(m.z, m.w));
            if (parts != nullptr) reinterpret_cast<float4 *>(parts)[p] = m;
        }
    }
    // The first token of the first piece that holds the maximum, which every run of ranks keeps.
    __device__ __forceinline__ void largest() {
        const int p = first_of(np, sh, [&](int i) { return sh.pm[i] == top; });
        if (t < kWave) {
            Eight<T> g;
            float v[8];
            g.load(x, p, vocab);
            g.get(v);
            int at = 8;
#pragma unroll
            for (int e = 7; e >= 0; --e)
                if (v[e] == top) at = e;
            const uint64_t some = __ballot(at < 8);
            if (lane == __ffsll((unsigned long long)some) - 1) finish(g.c0 + at, top);
        }
    }
    // The draw from the kept tokens: ps holds the pieces' sums of them (running ones if `running`); `n` listed tokens hold
    // all of the border's key, or with n = 0 cnt the running numbers of such tokens by piece.
    __device__ __forceinline__ void draw(const Kept &kept, int n, bool running) {
        if (!running) scan_array<kMaxPieces>(sh.ps, np, sh.scratch);
        const double total = sh.ps[np - 1], target = double(c.u) * total;
        int p = first_of(np, sh, [&](int i) { return sh.ps[i] > target; });
        if (p >= np) p = first_of(np, sh, [&](int i) { return sh.ps[i] == total; });
        int64_t before = 0;  // tokens of the border's key in earlier pieces
        if (n > 0) {
            if (t == 0) sh.count = 0;
            __syncthreads();
            for (int i = t; i < n; i += kThreads)
                if (list_key(sh, i) == kept.key && list_id(sh, i) < p * kPiece) atomicAdd(&sh.count, 1);
            __syncthreads();
            before = sh.count;
        } else if (p > 0 && !running) {
            before = sh.cnt[p - 1];
        }
        // Piece sums are rounded by themselves: where one is said to hold the draw and does not, the row's largest is taken.
        if (t == 0) sh.token = -1;
        __syncthreads();
        if (t < kWave) draw_in_piece(x, p, vocab, top, r.scale, kept, before, p > 0 ? sh.ps[p - 1] : 0.0, target, sh);
        __syncthreads();
        if (sh.token < 0) largest();
        else if (t == 0) finish(sh.token, value_of(sh.key));
    }
    // The border's bin, the pieces' sums of the tokens above it (ps) and its own tokens (comp), by this workgroup alone: the same
    // integers, and sums in the same order, as sample_bins_kernel and sample_list_kernel leave of a row that has a place.
    __device__ __forceinline__ int list_border(BorderBin &out) {
        const Fixed f = fixed_of(whole);
        const Bins bins = bins_of(top, r.scale);
        __syncthreads();
        for (int i = t; i < kBins; i += kThreads) {
            sh.cnt[i] = 0;
            sh.mass[i] = 0;
        }
        __syncthreads();
        each_piece(x, np, vocab, [](int) { return true; }, [&](int, const Eight<T> &g) {
            float v[8];
            g.get(v);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (g.c0 + e < vocab) {
                    const int b = bins.of(v[e]);
                    atomicAdd(&sh.cnt[b], 1u);
                    const uint64_t w = f.of(w_of(v[e]));
                    if (w != 0) atomicAdd(reinterpret_cast<unsigned long long *>(&sh.mass[b]), (unsigned long long)w);
                }
        });
        __syncthreads();
        scan_array<kBins>(sh.cnt, kBins, sh.scratch);
        scan_array<kBins>(sh.mass, kBins, sh.scratch);
        const double target = c.share * f.sum(sh.mass[kBins - 1]);
        int b = first_of(kBins, sh, [&](int i) { return c.k < vocab ? int64_t(sh.cnt[i]) >= c.k : f.sum(sh.mass[i]) >= target; });
        b = b < kBins ? b : kBins - 1;
        out = {bins.lowest(b), bins.highest(b), b > 0 ? int64_t(sh.cnt[b - 1]) : 0, b > 0 ? f.sum(sh.mass[b - 1]) : 0.0, target};
        __syncthreads();
        if (t == 0) sh.count = 0;
        __syncthreads();
        each_piece(x, np, vocab, [](int) { return true; }, [&](int p, const Eight<T> &g) {
            float v[8];
            g.get(v);
            double s = 0.0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const double w = w_of(v[e]);
                s += key_of(v[e]) > out.hi && w >= c.least ? w : 0.0;
            }
            s = wave_sum64(s);
            if (lane == 0) sh.ps[p] = s;
            append(&sh.count, sh.comp, v, g.c0, vocab, out.lo, out.hi);
        });
        __syncthreads();
        return sh.count;
    }
    // The whole row by this workgroup alone, in as many histograms as it takes.
    __device__ __forceinline__ void draw_alone() {
        Kept kept{0, 0, c.least};
        double of = -1.0;
        for (int by = 0; by < 2; ++by) {
            if (by == 0 ? c.k >= vocab : c.share > 1.0) continue;
            const Border b = find_border(x, a, top, r.scale, whole, by == 0, c.k, c.share, of, sh);
            of = b.mass;
            if (by == 0 || b.key > kept.key || (b.key == kept.key && b.ties < kept.ties)) {
                kept.key = b.key;
                kept.ties = b.ties;
            }
        }
        const double edge = w_of(value_of(kept.key));  // of the border's own tokens
        const bool with_ties = kept.ties > 0 && edge >= c.least;
        __syncthreads();
        each_piece(x, np, vocab, [](int) { return true; }, [&](int p, const Eight<T> &g) {
            float v[8];
            g.get(v);
            const int c0 = g.c0;
            double s = 0.0;
            int ties = 0;
            if (key_of(sh.pm[p]) >= kept.key) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint32_t key = key_of(v[e]);
                    const double w = w_of(v[e]);
                    if (key > kept.key && w >= c.least) s += w;
                    ties += with_ties && c0 + e < vocab && key == kept.key ? 1 : 0;
                }
                s = wave_sum64(s);
#pragma unroll
                for (int off = kWave / 2; off > 0; off >>= 1) ties += __shfl_xor(ties, off, kWave);
            }
            if (lane == 0) {
                sh.ps[p] = s;
                sh.cnt[p] = uint32_t(ties);
            }
        });
        __syncthreads();
        scan_array<kMaxPieces>(sh.cnt, np, sh.scratch);
        for (int p = t; p < np; p += kThreads) {
            const int64_t before = p > 0 ? sh.cnt[p - 1] : 0, here = int64_t(sh.cnt[p]) - before;
            const int64_t room = kept.ties - before, in = room < 0 ? 0 : room < here ? room : here;
            sh.ps[p] += double(in) * edge;
        }
        __syncthreads();
        draw(kept, 0, false);
    }
};

// A workgroup a row: all draws but those whose border is not among the few tokens that reach a bound.  These it puts off
// for the whole chip (PUT_OFF), or makes alone.
template <typename T, bool PUT_OFF> __global__ __launch_bounds__(kThreads) void sample_select_kernel(SampleArgs a) {
    __shared__ Shared sh;
    RowWork<T> w(a, sh, blockIdx.x);
    const int np = w.np, vocab = w.vocab, t = w.t, lane = w.lane;
    const Choice &c = w.c;
    for (int i = t; i < kBins; i += kThreads) sh.sub[i] = 0;
    if (a.part_max != nullptr) {
        w.load_maxima(sh.part_max);
        for (int p = t; p < np; p += kThreads) sh.ps[p] = a.piece_sum[w.row * np + p];
    } else {
        each_piece(w.x, np, vocab, [](int) { return true; }, [&](int p, const Eight<T> &g) {
            float v[8], part;
            double s;
            g.get_raw(v);
            piece_stats(v, w.r.scale, part, s);
            if (lane % 16 == 0) sh.part_max[p * kParts + lane / 16] = part;
            const float m = max_of_rows(part);
            if (lane == 0) {
                sh.pm[p] = m;
                sh.ps[p] = s;
            }
        });
    }
    __syncthreads();
    float top = -INFINITY;
    for (int p = lane; p < np; p += kWave) top = fmaxf(top, sh.pm[p]);
    w.top = top = wave_max_dpp(top);
    if (top == -INFINITY) {  // no token is left
        if (t == 0) {
            a.tokens[w.row] = -1;
            a.logprobs[w.row] = -INFINITY;
        }
        return;
    }
    for (int p = t; p < np; p += kThreads) sh.ps[p] = sh.pm[p] == -INFINITY ? 0.0 : sh.ps[p] * w.w_of(sh.pm[p]);
    __syncthreads();
    scan_array<kMaxPieces>(sh.ps, np, sh.scratch);
    const double whole = w.whole = sh.ps[np - 1];
    if (c.k == 1) {
        w.largest();
        return;
    }
    if (c.k == vocab && c.share > 1.0 && c.least == 0.0) {
        w.draw(Kept{0, 0, 0.0}, 0, true);
        return;
    }
    // A bound that all kept tokens reach, if enough of them do; for rows that fit in the list then all.
    const int parts = np * kParts;
    constexpr int kBits = std::is_same<T, bf16_t>::value ? 16 : 24;  // of a key that a bound looks at
    for (int attempt = vocab > kThreads ? 0 : 1; attempt < (vocab > kList ? 1 : 2); ++attempt) {
        bool complete = true;  // no token that may be kept is below the bound
        float bound = -INFINITY;
        if (attempt == 0) {
            // Tokens of less w than `least`: a little below, for the rounding of the logarithm.
            float low = -INFINITY;
            if (c.least > 0.0 && (c.k == vocab || c.share > 1.0)) {
                const double under = -w.r.t * log(c.least);
                low = isinf(top) ? top : float(double(top) - under - 1e-6 * (fabs(double(top)) + under));
            }
            const int64_t reach = c.k < vocab ? c.k : c.share < 1.0 ? 128 : 0;
            const bool by_thread = reach > parts && reach <= kThreads;  // more ranks than parts: maxima of every thread
            if (reach > parts && !by_thread && low == -INFINITY) continue;
            if (by_thread) {
                float m = -INFINITY;
                each_piece(w.x, np, vocab, [](int) { return true; }, [&](int, const Eight<T> &g) {
                    float v[8];
                    g.get(v);
#pragma unroll
                    for (int e = 0; e < 8; ++e) m = fmaxf(m, v[e]);
                });
                float *const maxima = reinterpret_cast<float *>(sh.comp);
                maxima[t] = m;  // read by itself alone
                bound = rank_bound<kBits, kThreads>(maxima, kThreads, int(reach), sh.sub);
                complete = c.k < vocab || low >= bound;
            } else if (reach > 0 && reach <= parts) {
                bound = rank_bound<kBits, kMaxPieces * kParts>(sh.part_max, parts, int(reach), sh.sub);
                complete = c.k < vocab || low >= bound;
            }
            bound = fmaxf(bound, low);
        }
        const int n = collect_top(w.x, parts, vocab, bound, sh);
        if (n <= kList) {
            sort_list(sh, n, top, w.r.scale);
            scan_array<kList>(sh.w, n, sh.scratch);
            const int kn = c.k < n ? int(c.k) : n;
            const double mass = c.k < vocab ? sh.w[kn - 1] : whole;
            if (complete || sh.w[n - 1] >= c.share * mass) {
                const int keep = first_of(n, sh, [&](int i) {
                    return i > 0 && (i >= kn || !(sh.w[i - 1] < c.share * mass || c.share > 1.0) || !(w.w_of(value_of(list_key(sh, i))) >= c.least));
                });
                for (int p = t; p < np; p += kThreads) {
                    sh.ps[p] = 0.0;
                    sh.sums[p] = 0;
                }
                __syncthreads();
                Kept kept{0, 0, 0.0};  // `least` is in `keep` already
                keep_listed(sh, n, keep, np, top, w.r.scale, whole, kept);
                w.draw(kept, n, false);
                return;
            }
        }
    }
    if constexpr (PUT_OFF) {
        if (t == 0) sh.place = atomicAdd(a.put_off, 1);
        __syncthreads();
        const int at = sh.place;
        if (t == 0) a.put_off[1 + at] = int32_t(w.row);
        if (at >= a.most) return;
        Wide &wide = a.wide[at];
        for (int i = t; i < kBins; i += kThreads) {
            wide.mass[i] = 0;
            wide.cnt[i] = 0;
        }
        if (t == 0) {
            wide.whole = whole;
            wide.top = top;
            wide.count = 0;
        }
    } else {
        w.draw_alone();
    }
}

// Of the rows put off that all workgroups work on together: the place, chunk by chunk of 16 pieces; fn(row, its place, first piece).
constexpr int kChunk = 16;
template <typename Fn> __device__ __forceinline__ void each_chunk(const SampleArgs &a, Fn fn) {
    const int rows = a.put_off[0] < a.most ? a.put_off[0] : a.most;
    const int chunks = (a.pieces + kChunk - 1) / kChunk;
    for (int item = blockIdx.x; item < rows * chunks; item += gridDim.x) {
        const int at = item / chunks;
        fn(int64_t(a.put_off[1 + at]), a.wide[at], (item - at * chunks) * kChunk);
    }
}
// By one alone of top-k and top-p: the other's border would need the first's sum.
__device__ __forceinline__ bool together(const Choice &c, int vocab) { return (c.k < vocab) != (c.share < 1.0); }

template <typename T> __global__ __launch_bounds__(256) void sample_bins_kernel(SampleArgs a) {
    __shared__ uint32_t cnt[kBins];
    __shared__ uint64_t mass[kBins];
    const int t = threadIdx.x, wave = t / kWave;
    each_chunk(a, [&](int64_t row, Wide &wide, int p0) {
        const Row r = row_of(a, row);
        if (!together(choice_of(a, row, r.greedy), a.vocab)) return;
        const T *x = static_cast<const T *>(a.logits) + row * a.stride;
        const Bins bins = bins_of(wide.top, r.scale);
        const Fixed f = fixed_of(wide.whole);
        __syncthreads();
        for (int i = t; i < kBins; i += 256) {
            cnt[i] = 0;
            mass[i] = 0;
        }
        __syncthreads();
        Eight<T> g[kChunk / 4];
#pragma unroll
        for (int q = 0; q < kChunk / 4; ++q)
            if (p0 + 4 * q + wave < a.pieces) g[q].load(x, p0 + 4 * q + wave, a.vocab);
#pragma unroll
        for (int q = 0; q < kChunk / 4; ++q) {
            if (p0 + 4 * q + wave >= a.pieces) break;
            float v[8];
            g[q].get(v);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (g[q].c0 + e < a.vocab) {
                    const int b = bins.of(v[e]);
                    atomicAdd(&cnt[b], 1u);
                    const uint64_t w = f.of(weight(v[e], wide.top, r.scale));
                    if (w != 0) atomicAdd(reinterpret_cast<unsigned long long *>(&mass[b]), (unsigned long long)w);
                }
        }
        __syncthreads();
        for (int i = t; i < kBins; i += 256)
            if (cnt[i] != 0) {
                atomicAdd(&wide.cnt[i], cnt[i]);
                atomicAdd(reinterpret_cast<unsigned long long *>(&wide.mass[i]), (unsigned long long)mass[i]);
            }
    });
}

// The border's bin, as every workgroup of 256 threads finds it for itself from the row's bins, 4 a thread.
__device__ __forceinline__ BorderBin border_bin(const Wide &wide, const Choice &c, int vocab, const Bins &bins, uint64_t *scratch, int *found) {
    constexpr int Q = kBins / 256, W = 256 / kWave;
    const int t = threadIdx.x, lane = t & (kWave - 1), wave = t / kWave;
    const Fixed f = fixed_of(wide.whole);
    uint64_t mass[Q], cnt[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        mass[q] = wide.mass[t * Q + q] + (q > 0 ? mass[q - 1] : 0);
        cnt[q] = wide.cnt[t * Q + q] + (q > 0 ? cnt[q - 1] : 0);
    }
    uint64_t sm = wave_scan(mass[Q - 1]), sc = wave_scan(cnt[Q - 1]);
    __syncthreads();
    if (lane == kWave - 1) {
        scratch[wave] = sm;
        scratch[W + wave] = sc;
    }
    if (t == 0) *found = kBins;
    __syncthreads();
    sm -= mass[Q - 1];
    sc -= cnt[Q - 1];
    uint64_t all = 0;
    for (int v = 0; v < W; ++v) {
        if (v < wave) {
            sm += scratch[v];
            sc += scratch[W + v];
        }
        all += scratch[v];
    }
    const double target = c.share * f.sum(all);  // of the integers' sum, as the bins are
    int b = kBins;
#pragma unroll
    for (int q = Q - 1; q >= 0; --q)
        if (c.k < vocab ? int64_t(sc + cnt[q]) >= c.k : f.sum(sm + mass[q]) >= target) b = t * Q + q;
    if (b < kBins) atomicMin(found, b);
    __syncthreads();
    const int first = *found < kBins ? *found : kBins - 1;
    __syncthreads();
    if (first / Q == t) {
        const int q = first - t * Q;
        uint64_t m = sm, n = sc;
#pragma unroll
        for (int i = 0; i < Q; ++i)
            if (i + 1 == q) {
                m += mass[i];
                n += cnt[i];
            }
        scratch[0] = m;
        scratch[1] = n;
    }
    __syncthreads();
    const BorderBin out{bins.lowest(first), bins.highest(first), int64_t(scratch[1]), f.sum(scratch[0]), target};
    __syncthreads();
    return out;
}

template <typename T> __global__ __launch_bounds__(256) void sample_list_kernel(SampleArgs a) {
    __shared__ uint64_t scratch[8];
    __shared__ int found;
    const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
    each_chunk(a, [&](int64_t row, Wide &wide, int p0) {
        const Row r = row_of(a, row);
        const Choice c = choice_of(a, row, r.greedy);
        if (!together(c, a.vocab)) return;
        const T *x = static_cast<const T *>(a.logits) + row * a.stride;
        Eight<T> g[kChunk / 4];
#pragma unroll
        for (int q = 0; q < kChunk / 4; ++q)
            if (p0 + 4 * q + wave < a.pieces) g[q].load(x, p0 + 4 * q + wave, a.vocab);
        const BorderBin b = border_bin(wide, c, a.vocab, bins_of(wide.top, r.scale), scratch, &found);
        if (p0 == 0 && threadIdx.x == 0) wide.border = b;
#pragma unroll
        for (int q = 0; q < kChunk / 4; ++q) {
            const int p = p0 + 4 * q + wave;
            if (p >= a.pieces) break;
            float v[8];
            g[q].get(v);
            double s = 0.0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const double w = weight(v[e], wide.top, r.scale);
                s += key_of(v[e]) > b.hi && w >= c.least ? w : 0.0;
            }
            s = wave_sum64(s);
            if (lane == 0) a.piece_sum[row * a.pieces + p] = s;  // in place of the sum of all
            append(&wide.count, wide.list, v, g[q].c0, a.vocab, b.lo, b.hi);
        }
    });
}

template <typename T> __global__ __launch_bounds__(kThreads) void sample_finish_kernel(SampleArgs a) {
    __shared__ Shared sh;
    const int rows = a.put_off[0];
    for (int at = blockIdx.x; at < rows; at += gridDim.x) {
        __syncthreads();
        RowWork<T> w(a, sh, a.put_off[1 + at]);
        const int np = w.np, vocab = w.vocab, t = w.t, lane = w.lane;
        const Choice &c = w.c;
        float top = -INFINITY;
        w.load_maxima(nullptr);
        __syncthreads();
        for (int p = lane; p < np; p += kWave) top = fmaxf(top, sh.pm[p]);
        w.top = wave_max_dpp(top);
        int n = 0;
        BorderBin b;
        if (at < a.most) {
            const Wide &wide = a.wide[at];
            w.whole = wide.whole;
            n = together(c, vocab) ? wide.count : 0;
            if (n > 0 && n <= kList) {
                b = wide.border;
                for (int p = t; p < np; p += kThreads) sh.ps[p] = a.piece_sum[w.row * np + p];
                for (int i = t; i < n; i += kThreads) sh.comp[i] = wide.list[i];
            }
        } else {  // no place of its own: its sums are as the first pass left them
            for (int p = t; p < np; p += kThreads) sh.ps[p] = sh.pm[p] == -INFINITY ? 0.0 : a.piece_sum[w.row * np + p] * w.w_of(sh.pm[p]);
            __syncthreads();
            scan_array<kMaxPieces>(sh.ps, np, sh.scratch);
            w.whole = sh.ps[np - 1];
            if (together(c, vocab)) n = w.list_border(b);  // which rows have a place is chance: their tokens are not
        }
        bool drawn = false;
        if (n > 0 && n <= kList) {
            for (int p = t; p < np; p += kThreads) sh.sums[p] = 0;
            __syncthreads();
            // Where min-p leaves nothing of the bin, any border in it will do.
            const bool none = !(w.w_of(value_of(b.hi)) >= c.least);
            const bool by_count = none || c.k < vocab;
            n = narrow(sh, n, b.lo, b.hi, by_count, none ? b.above + 1 : c.k, b.target, c.least, w.top, w.r.scale, w.whole, b.above, b.base);
            if (n > 0) {
                sort_list(sh, n, w.top, w.r.scale);
                scan_array<kList>(sh.w, n, sh.scratch);
                int keep = 1;
                if (by_count) keep = none ? 1 : int(c.k - b.above);
                else keep = 1 + first_of(n, sh, [&](int i) { return b.base + sh.w[i] >= b.target; });
                keep = keep > n ? n : keep;  // the integers' sum passes the target, this one by its rounding may not
                if (keep > 0) {
                    __syncthreads();
                    Kept kept{0, 0, c.least};
                    keep_listed(sh, n, keep, np, w.top, w.r.scale, w.whole, kept);
                    w.draw(kept, n, false);
                    drawn = true;
                }
            }
        }
        if (!drawn) w.draw_alone();
    }
}

// Rows of at most 128 logits, a wave each: logit 64 e + lane is the lane's e-th, ranks are counted over all of them.  (Up to 512
// so, 500 logits take 34 us, a workgroup a row 25.)
constexpr int kSmall = 128;
template <typename T> __global__ __launch_bounds__(256) void sample_small_kernel(SampleArgs a, int64_t rows) {
    __shared__ uint64_t lists[4][kSmall];
    __shared__ double weights[4][kSmall];
    constexpr int E = kSmall / kWave;
    const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
    const int64_t row = int64_t(blockIdx.x) * 4 + wave;
    if (row >= rows) return;  // no barriers below
    const T *x = static_cast<const T *>(a.logits) + row * a.stride;
    const int vocab = a.vocab, used = (vocab + kWave - 1) / kWave;
    const Row r = row_of(a, row);
    const Choice c = choice_of(a, row, r.greedy);
    float v[E], top = -INFINITY;
    double w[E], whole = 0.0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        v[e] = 64 * e + lane < vocab ? fmaxf(to_f32(x[64 * e + lane]), -INFINITY) + 0.f : -INFINITY;
        top = fmaxf(top, v[e]);
    }
    top = wave_max_dpp(top);
    if (top == -INFINITY) {
        if (lane == 0) {
            a.tokens[row] = -1;
            a.logprobs[row] = -INFINITY;
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
        w[e] = e < used ? weight(v[e], top, r.scale) : 0.0;
        whole += w[e];
    }
    whole = wave_sum64(whole);
    if (c.k < vocab || c.share < 1.0 || c.least > 0.0) {
        uint64_t *const list = lists[wave];
        double *const ranked = weights[wave];
        uint64_t mine[E];
        int rank[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            mine[e] = uint64_t(key_of(v[e])) << 32 | uint32_t(~(64 * e + lane));
            rank[e] = 0;
            list[64 * e + lane] = mine[e];
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the wave's own writes
#pragma unroll 8
        for (int j = 0; j < vocab; ++j) {
            const uint64_t o = list[j];
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (e < used) rank[e] += o > mine[e] ? 1 : 0;
        }
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (64 * e + lane < vocab) ranked[rank[e]] = w[e];
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        // A lane sums `used` ranks in a row.
        const int k = int(c.k);
        double mass = 0.0, first = 0.0;
        for (int i = 0; i < used; ++i) {
            const int q = lane * used + i;
            const double y = q < vocab ? ranked[q] : 0.0;
            mass += y;
            first += q < k ? y : 0.0;
        }
        double before = wave_scan(mass) - mass;
        first = wave_sum64(first);
        if (lane == 0) before = 0.0;
        int keep = 0;
        for (int i = 0; i < used; ++i) {
            const int q = lane * used + i;
            if (q >= vocab) break;
            const double y = ranked[q];
            if (q == 0 || (q < k && (c.share > 1.0 || before < c.share * first) && y >= c.least)) ++keep;
            before += y;
        }
#pragma unroll
        for (int off = kWave / 2; off > 0; off >>= 1) keep += __shfl_xor(keep, off, kWave);
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (rank[e] >= keep) w[e] = 0.0;
    }
    // The draw in the order of ids: 64 of them a step.
    double upto[E], total = 0.0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        upto[e] = total;
        if (e < used) {
            upto[e] += wave_scan(w[e]);
            total = __shfl(upto[e], kWave - 1, kWave);
        }
    }
    const double target = double(c.u) * total;
    int64_t token = -1;
    float value = top;
#pragma unroll
    for (int e = E - 1; e >= 0; --e) {
        const uint64_t past = __ballot(upto[e] > target && w[e] > 0.0);
        if (past != 0) {
            const int from = __ffsll((unsigned long long)past) - 1;
            token = 64 * e + from;
            value = __shfl(v[e], from, kWave);
        }
    }
    if (token < 0) {  // rounding passed the last: the last that is kept
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const uint64_t some = __ballot(w[e] > 0.0);
            if (some != 0) {
                const int from = 63 - __clzll((long long)some);
                token = 64 * e + from;
                value = __shfl(v[e], from, kWave);
            }
        }
    }
    if (lane == 0) finish_row(a, row, token, value, top, r.t, whole);
}

// Rows of few pieces need no pass of their own over the chip.
constexpr int kInline = 16;

int64_t pieces_of(int64_t vocab) { return (vocab + kPiece - 1) / kPiece; }
// Sums and maxima of the pieces, the rows put off, and a place for the histogram and list of up to 1024 of them.
struct Space {
    int64_t sums, maxima, put_off, wide, bytes;
    int most;
};
Space space_of(int64_t rows, int64_t vocab) {
    Space s{};
    if (pieces_of(vocab) <= kInline) return s;
    const auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
    s.most = int(std::min<int64_t>(rows, 1024));
    s.maxima = up(rows * pieces_of(vocab) * 8);
    s.put_off = s.maxima + up(rows * pieces_of(vocab) * kParts * 4);
    s.wide = s.put_off + up((rows + 1) * 4);
    s.bytes = s.wide + s.most * int64_t(sizeof(Wide));
    return s;
}

template <typename T> hipError_t sample(SampleArgs &a, int64_t rows, void *workspace, hipStream_t st) {
    if (a.vocab <= kSmall) {
        sample_small_kernel<T><<<unsigned((rows + 3) / 4), 256, 0, st>>>(a, rows);
        return hipGetLastError();
    }
    if (a.pieces <= kInline) {
        sample_select_kernel<T, false><<<unsigned(rows), kThreads, 0, st>>>(a);
        return hipGetLastError();
    }
    const Space space = space_of(rows, a.vocab);
    char *const ws = static_cast<char *>(workspace);
    a.piece_sum = reinterpret_cast<double *>(ws);
    a.part_max = reinterpret_cast<float *>(ws + space.maxima);
    // 4 pieces a wave where that leaves the chip 4096 waves.
    a.each = rows * a.pieces >= 4 * 4096 ? 4 : 1;
    // A border that is not near the top is for the whole chip, unless top-k says that it is (or a bound by min-p alone).
    const bool near = !a.top_k && ((a.top_k_all > 0 && a.top_k_all <= a.pieces * kParts) ||
                                   (!a.top_p && !(a.top_p_all < 1.0) && (a.top_k_all <= 0 || a.top_k_all >= a.vocab)));
    if (!near) {
        a.put_off = reinterpret_cast<int32_t *>(ws + space.put_off);
        a.wide = reinterpret_cast<Wide *>(ws + space.wide);
        a.most = space.most;
    }
    const dim3 grid(unsigned((a.pieces + 4 * a.each - 1) / (4 * a.each)), unsigned(rows));
    sample_stats_kernel<T><<<grid, 256, 0, st>>>(a);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    if (near) {
        sample_select_kernel<T, false><<<unsigned(rows), kThreads, 0, st>>>(a);
        return hipGetLastError();
    }
    sample_select_kernel<T, true><<<unsigned(rows), kThreads, 0, st>>>(a);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    const int64_t chunks = std::min<int64_t>(1024, rows * ((a.pieces + kChunk - 1) / kChunk));
    sample_bins_kernel<T><<<unsigned(chunks), 256, 0, st>>>(a);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    sample_list_kernel<T><<<unsigned(chunks), 256, 0, st>>>(a);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    sample_finish_kernel<T><<<unsigned(std::min<int64_t>(rows, 512)), kThreads, 0, st>>>(a);
    return hipGetLastError();
}

int64_t workspace_of(int64_t rows, int64_t vocab) { return space_of(rows, vocab).bytes; }
int check_sizes(const char *fn, int64_t rows, int64_t vocab) {
    if (rows < 0 || rows > 65535 || vocab < 1 || vocab > int64_t(kMaxPieces) * kPiece)
        return capi::fail(hipErrorInvalidValue, "%s: %lld rows (up to 65535) of %lld logits (1 to %d)", fn, (long long)rows,
                          (long long)vocab, kMaxPieces * kPiece);
    return 0;
}

}  // namespace
}  // namespace ctattn

using namespace ctattn;
using namespace ctattn::capi;

extern "C" {

int64_t ctattn_sample_workspace_bytes(int64_t rows, int64_t vocab) {
    if (check_sizes("ctattn_sample_workspace_bytes", rows, vocab) != 0) return -1;
    return workspace_of(rows, vocab);
}

int ctattn_sample(int dtype, const void *logits, const float *u, const float *temperature, const int32_t *top_k,
                  const float *top_p, const float *min_p, double temperature_all, int64_t top_k_all, double top_p_all,
                  double min_p_all, int64_t *tokens, float *logprobs, void *workspace, int64_t workspace_bytes, int64_t rows,
                  int64_t vocab, int64_t stride, void *stream) {
    const char *fn = "ctattn_sample";
    if (dtype != CTATTN_F32 && dtype != CTATTN_BF16 && dtype != CTATTN_F16)
        return fail(dtype == CTATTN_F64 ? hipErrorNotSupported : hipErrorInvalidValue, "%s: dtype %d unsupported (0 = f32, 1 = bf16, 2 = f16)",
                    fn, dtype);
    if (int rc = check_sizes(fn, rows, vocab)) return rc;
    if (rows > 1 && stride != 0 && (stride < vocab || stride > (int64_t(1) << 40)))  // 0: one row for all
        return fail(hipErrorInvalidValue, "%s: rows %lld apart of %lld logits", fn, (long long)stride, (long long)vocab);
    if (rows == 0) return ok();
    if (!logits || !tokens || !logprobs) return fail(hipErrorInvalidValue, "%s: null pointer", fn);
    if (!u && (temperature || temperature_all > 0.0))
        return fail(hipErrorInvalidValue, "%s: random numbers may be left out for greedy rows alone", fn);
    const int64_t need = workspace_of(rows, vocab), es = dtype == CTATTN_F32 ? 4 : 2;
    if (need > 0 && (!workspace || workspace_bytes < need))
        return fail(hipErrorInvalidValue, "%s: workspace too small (%lld bytes, %lld needed)", fn, (long long)workspace_bytes,
                    (long long)need);
    if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
        return fail(hipErrorInvalidValue, "%s: workspace must be 16-byte aligned", fn);
    const int64_t r4 = rows * 4;
    const Bytes in[] = {run_of(logits, ((rows - 1) * stride + vocab) * es), run_of(u, u ? r4 : 0), run_of(temperature, temperature ? r4 : 0),
                        run_of(top_k, top_k ? r4 : 0), run_of(top_p, top_p ? r4 : 0), run_of(min_p, min_p ? r4 : 0)};
    const Bytes out[] = {run_of(tokens, rows * 8), run_of(logprobs, r4), run_of(workspace, need)};
    if (int rc = check_apart(fn, in, out)) return rc;
    SampleArgs a{};
    a.logits = logits;
    a.u = u;
    a.temperature = temperature;
    a.top_p = top_p;
    a.min_p = min_p;
    a.top_k = top_k;
    a.temperature_all = temperature_all;
    a.top_p_all = top_p_all;
    a.min_p_all = min_p_all;
    a.top_k_all = top_k_all;
    a.tokens = tokens;
    a.logprobs = logprobs;
    a.stride = rows > 1 ? stride : 0;
    a.vocab = int(vocab);
    a.pieces = int(pieces_of(vocab));
    hipStream_t st = static_cast<hipStream_t>(stream);
    hipError_t e;
    switch (dtype) {
    case CTATTN_F32: e = sample<float>(a, rows, workspace, st); break;
    case CTATTN_BF16: e = sample<bf16_t>(a, rows, workspace, st); break;
    default: e = sample<f16_t>(a, rows, workspace, st); break;
    }
    return finish(fn, e, st);
}

}  // extern "C"
