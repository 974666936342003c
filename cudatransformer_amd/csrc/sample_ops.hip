// Next tokens from logits and given random numbers: temperature, top-k, top-p and min-p.
//
// With M the row's largest logit and w_i = exp((x_i - M) / T) the tokens are ranked by (x, then the lower id), a run
// of the first ranks is kept (ctattn.h), and the token is the first id, in the order of ids, at which the sum of kept w
// passes u times their whole sum.  A draw near a border of two ids must not depend on the order of a sum, so w and
// its sums are held in 64 bits: 2^e by a polynomial of degree 9 of e's fraction, 4e-14 off (a token changes where u is
// that near a border).
//
// A row is pieces of 512 logits, 8 a lane of a wave.  One pass over the logits, spread over the chip, leaves each
// piece's maximum and its sum of w relative to it; a workgroup a row does the rest.  A draw from all tokens then needs
// the pieces' sums and one piece.  Top-k and most nuclei lie among a few hundred tokens: the R-th largest of the pieces'
// maxima is a bound that at least R tokens reach, so only pieces that reach it are read again, and what reaches it is
// ranked in LDS.  Where that is not enough (a nucleus of thousands of tokens, more than 2048 at the bound), the border is
// found in a histogram of the whole row over x, with counts and sums of w in 64-bit integers (sums of integers do not
// depend on the order of the atomics), refined to a bin of at most 2048 tokens, or to one value, and ranked there.
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
constexpr int kThreads = 512;     // of a row's workgroup
constexpr int kWaves = kThreads / kWave;
constexpr int kList = 2048;       // tokens ranked in LDS
constexpr int kBins = 1024;
constexpr double kLog2e64 = 1.4426950408889634074;

struct SampleArgs {
    const void *logits;
    const float *u;
    const float *temperature, *top_p, *min_p;  // of each row, or null: the numbers below
    const int32_t *top_k;
    double temperature_all, top_p_all, min_p_all;
    int64_t top_k_all;
    int64_t *tokens;
    float *logprobs;
    float *piece_max;  // [rows][pieces], null: the row's workgroup makes them itself
    double *piece_sum;
    int64_t stride;
    int vocab, pieces, each;  // each: pieces of a wave of the first pass
};

struct Row {
    double t;      // the temperature of w: 1 for a greedy row
    double scale;  // log2(e) / t
    bool greedy;
};
__device__ __forceinline__ Row row_of(const SampleArgs &a, int64_t row) {
    const double t = a.temperature != nullptr ? double(a.temperature[row]) : a.temperature_all;
    Row r;
    r.greedy = !(t > 0.0);
    r.t = r.greedy ? 1.0 : t;
    r.scale = kLog2e64 / r.t;
    return r;
}

// exp((x - m) / t), 1 where x is m (infinite too), 0 for x = -inf.  (2^f - 1) / f on [-1/2, 1/2] is a polynomial of
// degree 8 through its values at the Chebyshev points, so that 2^0 is 1 exactly.
__device__ __forceinline__ double weight(float x, float m, double scale) {
    const double e = x == m ? 0.0 : fmax((double(x) - double(m)) * scale, -1100.0);
    const double n = rint(e), f = e - n;
    double p = 1.0203121063391729e-07;
    p = fma(p, f, 1.3255224878668817e-06);
    p = fma(p, f, 1.525268684626772e-05);
    p = fma(p, f, 0.00015403455852453838);
    p = fma(p, f, 0.0013333558179043112);
    p = fma(p, f, 0.0096181291594025584);
    p = fma(p, f, 0.055504108664760424);
    p = fma(p, f, 0.24022650695812989);
    p = fma(p, f, 0.69314718055994529);
    return ldexp(fma(p, f, 1.0), int(n));
}

// 8 logits of a lane; past the row's end and where there is none -inf; -0 becomes 0.
template <typename T> struct Eight {
    static constexpr int N = sizeof(T) == 2 ? 1 : 2;
    gran_raw g[N];
    int c0;
    __device__ __forceinline__ void load(const T *row, int piece, int vocab) {
        c0 = piece * kPiece + int(threadIdx.x & (kWave - 1)) * 8;
#pragma unroll
        for (int i = 0; i < N; ++i) g[i] = Gran<T>::load_tail(row, c0 + i * Gran<T>::EPC, vocab, -INFINITY);
    }
    __device__ __forceinline__ void get(float (&x)[8]) const {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float y = Gran<T>::get(g[e / Gran<T>::EPC], e % Gran<T>::EPC);
            x[e] = y == y ? y + 0.f : -INFINITY;
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

// A piece's maximum and its sum of w relative to it, the same in every lane.
__device__ __forceinline__ void piece_stats(const float (&x)[8], double scale, float &m, double &s) {
    m = x[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) m = fmaxf(m, x[e]);
    m = wave_max(m);
    s = 0.0;
    if (m == -INFINITY) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) s += weight(x[e], m, scale);
    s = wave_sum(s);
}

template <typename T> __global__ __launch_bounds__(256) void sample_stats_kernel(SampleArgs a) {
    const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
    const int64_t row = blockIdx.y;
    const T *x = static_cast<const T *>(a.logits) + row * a.stride;
    const double scale = row_of(a, row).scale;
    const int p0 = (blockIdx.x * 4 + wave) * a.each, p1 = p0 + a.each < a.pieces ? p0 + a.each : a.pieces;
    if (p0 >= p1) return;
    Eight<T> now, next;
    next.load(x, p0, a.vocab);
    for (int p = p0; p < p1; ++p) {
        now = next;
        if (p + 1 < p1) next.load(x, p + 1, a.vocab);
        float v[8], m;
        double s;
        now.get(v);
        piece_stats(v, scale, m, s);
        if (lane == 0) {
            a.piece_max[row * a.pieces + p] = m;
            a.piece_sum[row * a.pieces + p] = s;
        }
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
    double w[kList];
    uint64_t sorted[kList];
    uint64_t scratch[2 * kWaves];
    int32_t found, count;
    uint32_t key;
    double sum;
    int64_t token;
};

// Running sums of a[0 .. n), in place, in one order.
template <typename A> __device__ void scan_array(A *a, int n, uint64_t *scratch) {
    A *waves = reinterpret_cast<A *>(scratch);
    const int t = threadIdx.x, lane = t & (kWave - 1), wave = t / kWave;
    const int q = (n + kThreads - 1) / kThreads, i0 = t * q, i1 = i0 + q < n ? i0 + q : n;
    A s = 0;
    for (int i = i0; i < i1; ++i) s += a[i];
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
        const A y = __shfl_up(s, off, kWave);
        if (lane >= off) s += y;
    }
    __syncthreads();
    if (lane == kWave - 1) waves[wave] = s;
    __syncthreads();
    A run = __shfl_up(s, 1, kWave);
    if (lane == 0) run = 0;
    A before = 0;
    for (int w = 0; w < wave; ++w) before += waves[w];
    run += before;
    for (int i = i0; i < i1; ++i) {
        run += a[i];
        a[i] = run;
    }
    __syncthreads();
}
// The first i of [0, n) that holds, or n, in every thread.
template <typename Fn> __device__ int first_of(int n, Shared &sh, Fn holds) {
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
// The row's pieces, one after the other a wave's, the next one's loads ahead; fn(piece, values).
template <typename T, typename Want, typename Fn>
__device__ __forceinline__ void each_piece(const T *x, int pieces, int vocab, Want want, Fn fn) {
    int p = threadIdx.x / kWave;
    while (p < pieces && !want(p)) p += kWaves;
    Eight<T> now, next;
    if (p < pieces) next.load(x, p, vocab);
    while (p < pieces) {
        now = next;
        int q = p + kWaves;
        while (q < pieces && !want(q)) q += kWaves;
        if (q < pieces) next.load(x, q, vocab);
        float v[8];
        now.get(v);
        fn(p, v, now.c0);
        p = q;
    }
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
__device__ void draw_in_piece(const T *x, int piece, int vocab, float m, double scale, const Kept &k, int64_t before,
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

// Ranks the n listed tokens (comp): sorted[rank] = comp, w[rank] = its weight.  Thread t keeps its own tokens' ranks.
__device__ __forceinline__ void rank_list(Shared &sh, int n, float m, double scale, uint64_t (&mine)[4], int (&rank)[4], int (&place)[4]) {
    const int t = threadIdx.x;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        mine[k] = t + k * kThreads < n ? sh.comp[t + k * kThreads] : 0;
        rank[k] = place[k] = 0;
    }
    // Beside the rank by value the place by id: ids are complemented in the low half.
    const int used = (n + kThreads - 1) / kThreads;
    for (int j = 0; j < n; ++j) {
        const uint64_t c = sh.comp[j];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (k >= used) break;
            rank[k] += c > mine[k] ? 1 : 0;
            place[k] += uint32_t(c) > uint32_t(mine[k]) ? 1 : 0;
        }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (t + k * kThreads < n) {
            sh.sorted[rank[k]] = mine[k];
            sh.w[rank[k]] = weight(value_of(uint32_t(mine[k] >> 32)), m, scale);
        }
    __syncthreads();
}
// Lists the tokens with lo <= key <= hi of the wanted pieces; their number, which may pass the list's length.
template <typename T, typename Want>
__device__ int collect(const T *x, int pieces, int vocab, uint32_t lo, uint32_t hi, Want want, Shared &sh) {
    __syncthreads();
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    each_piece(x, pieces, vocab, want, [&](int, const float (&v)[8], int c0) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t key = key_of(v[e]);
            if (c0 + e < vocab && key >= lo && key <= hi) {
                const int at = atomicAdd(&sh.count, 1);
                if (at < kList) sh.comp[at] = uint64_t(key) << 32 | uint32_t(~(c0 + e));
            }
        }
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
__device__ Border find_border(const T *x, const SampleArgs &a, float m, double scale, double whole, bool by_count, int64_t want,
                              double share, double of, Shared &sh) {
    // The whole row's sum takes 62 bits, half a step a token is lost.
    const int bits = ilogb(whole) + 1;
    const double fix = ldexp(1.0, 62 - bits), unfix = ldexp(1.0, bits - 62);
    const float bins = float(scale * 32.0);  // 32 bins to a factor of two in w
    const auto linear = [&](float v) { return v == m ? 0 : int(fminf((m - v) * bins, float(kBins - 1))); };
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
        each_piece(x, a.pieces, a.vocab, [](int) { return true; }, [&](int, const float (&v)[8], int c0) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t key = key_of(v[e]);
                if (c0 + e < a.vocab && key >= lo && key <= hi) {
                    const int b = shift < 0 ? linear(v[e]) : int((hi - key) >> shift);
                    atomicAdd(&sh.cnt[b], 1u);
                    const uint64_t w = uint64_t(fma(weight(v[e], m, scale), fix, 0.5));
                    if (w != 0) atomicAdd(reinterpret_cast<unsigned long long *>(&sh.mass[b]), (unsigned long long)w);
                }
            }
        });
        __syncthreads();
        scan_array(sh.cnt, kBins, sh.scratch);
        scan_array(sh.mass, kBins, sh.scratch);
        if (shift < 0 && !by_count && of < 0.0) target = share * (double(sh.mass[kBins - 1]) * unfix);
        int b = first_of(kBins, sh, [&](int i) {
            return by_count ? before + int64_t(sh.cnt[i]) >= want : double(mass + sh.mass[i]) * unfix >= target;
        });
        if (b >= kBins) b = first_of(kBins, sh, [&](int i) { return sh.cnt[i] == sh.cnt[kBins - 1]; });  // the last with any
        const int64_t in = int64_t(sh.cnt[b]) - (b > 0 ? int64_t(sh.cnt[b - 1]) : 0);
        if (b > 0) {
            before += sh.cnt[b - 1];
            mass += sh.mass[b - 1];
        }
        if (shift < 0) {
            // The bin's keys: the bins fall with the key.
            uint32_t l = key_of(-INFINITY), h = key_of(m);
            const auto edge = [&](int at_most) {  // the lowest key of a bin <= at_most
                uint32_t p = l, q = h;
                while (p < q) {
                    const uint32_t mid = p + (q - p) / 2;
                    if (linear(value_of(mid)) <= at_most) q = mid;
                    else p = mid + 1;
                }
                return p;
            };
            lo = edge(b);
            hi = b > 0 ? edge(b - 1) - 1 : h;
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
                const double need = (target - double(mass) * unfix) / w;
                ties = need < double(in) ? int64_t(ceil(need)) : in;
            }
            ties = ties < 1 ? 1 : ties > in ? in : ties;
            return {hi, ties, double(mass) * unfix + double(ties) * w};
        }
        if (in <= kList) break;
        const int width = 32 - __clz(hi - lo);
        shift = width > 10 ? width - 10 : 0;
    }
    int n = collect(x, a.pieces, a.vocab, lo, hi, [](int) { return true; }, sh);
    n = n < kList ? n : kList;
    uint64_t mine[4];
    int rank[4], place[4];
    rank_list(sh, n, m, scale, mine, rank, place);
    scan_array(sh.w, n, sh.scratch);
    const double base = double(mass) * unfix;
    int j = by_count ? int(want - before) - 1 : first_of(n, sh, [&](int i) { return base + sh.w[i] >= target; });
    j = j < 0 ? 0 : j >= n ? n - 1 : j;
    const uint32_t key = uint32_t(sh.sorted[j] >> 32);
    const int first = first_of(n, sh, [&](int i) { return uint32_t(sh.sorted[i] >> 32) == key; });
    const Border out{key, j - first + 1, base + sh.w[j]};
    __syncthreads();
    return out;
}

template <typename T> __global__ __launch_bounds__(kThreads) void sample_select_kernel(SampleArgs a) {
    __shared__ Shared sh;
    const int t = threadIdx.x, lane = t & (kWave - 1);
    const int64_t row = blockIdx.x;
    const T *x = static_cast<const T *>(a.logits) + row * a.stride;
    const Row r = row_of(a, row);
    const int np = a.pieces, vocab = a.vocab;
    const auto every = [](int) { return true; };

    if (a.piece_max != nullptr) {
        for (int p = t; p < np; p += kThreads) {
            sh.pm[p] = a.piece_max[row * np + p];
            sh.ps[p] = a.piece_sum[row * np + p];
        }
    } else {
        each_piece(x, np, vocab, every, [&](int p, const float (&v)[8], int) {
            float m;
            double s;
            piece_stats(v, r.scale, m, s);
            if (lane == 0) {
                sh.pm[p] = m;
                sh.ps[p] = s;
            }
        });
    }
    __syncthreads();
    float top = -INFINITY;
    for (int p = lane; p < np; p += kWave) top = fmaxf(top, sh.pm[p]);
    top = wave_max(top);
    if (top == -INFINITY) {  // no token is left
        if (t == 0) {
            a.tokens[row] = -1;
            a.logprobs[row] = -INFINITY;
        }
        return;
    }
    for (int p = t; p < np; p += kThreads) sh.ps[p] = sh.pm[p] == -INFINITY ? 0.0 : sh.ps[p] * weight(sh.pm[p], top, r.scale);
    __syncthreads();
    scan_array(sh.ps, np, sh.scratch);
    const double whole = sh.ps[np - 1];

    float u = a.u != nullptr ? a.u[row] : 0.f;
    if (!(u >= 0.f)) u = 0.f;
    int64_t k = a.top_k != nullptr ? int64_t(a.top_k[row]) : a.top_k_all;
    const double p_ = a.top_p != nullptr ? double(a.top_p[row]) : a.top_p_all;
    const double share = p_ < 1.0 ? p_ : 2.0;  // 2: no nucleus
    double least = a.min_p != nullptr ? double(a.min_p[row]) : a.min_p_all;
    if (!(least > 0.0)) least = 0.0;
    if (k <= 0 || k > vocab) k = vocab;
    if (r.greedy || share <= 0.0 || least > 1.0) k = 1;
    const auto finish = [&](int64_t token, float value) {
        a.tokens[row] = token;
        const double d = value == top ? 0.0 : (double(value) - double(top)) / r.t;
        a.logprobs[row] = float(d - log(whole));
    };

    // The first token of the first piece that holds the maximum, which every run of ranks keeps.
    const auto largest = [&]() {
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
    };
    // A draw from piece p on, whose earlier ones sum to `base`; piece sums are rounded by themselves, and where one is said to
    // hold the draw and does not, the row's largest is taken.
    const auto draw = [&](int p, const Kept &kept, int64_t before, double base, double target) {
        if (t == 0) sh.token = -1;
        __syncthreads();
        if (t < kWave) draw_in_piece(x, p, vocab, top, r.scale, kept, before, base, target, sh);
        __syncthreads();
        if (sh.token < 0) largest();
        else if (t == 0) finish(sh.token, value_of(sh.key));
    };
    if (k == 1) {
        largest();
        return;
    }
    if (k == vocab && share > 1.0 && least == 0.0) {
        const double target = double(u) * whole;
        int p = first_of(np, sh, [&](int i) { return sh.ps[i] > target; });
        if (p >= np) p = first_of(np, sh, [&](int i) { return sh.ps[i] == whole; });
        draw(p, Kept{0, 0, 0.0}, 0, p > 0 ? sh.ps[p - 1] : 0.0, target);
        return;
    }

    // A bound that all kept tokens reach, if enough of them do.
    bool listed = true, complete = true;
    float bound = -INFINITY;
    if (vocab > kList) {
        // Tokens of less w than `least`: a little below, for the rounding of the logarithm.
        float low = -INFINITY;
        if (least > 0.0 && (k == vocab || share > 1.0)) {
            const double under = -r.t * log(least);
            low = isinf(top) ? top : float(double(top) - under - 1e-6 * (fabs(double(top)) + under));
        }
        const int64_t reach = k < vocab ? k : share < 1.0 ? 128 : 0;
        if (reach == 0) {
            bound = low;
        } else if (reach <= np) {
            // The piece whose maximum has that rank.
            __syncthreads();
            for (int i = t; i < np; i += kThreads) {
                const float mi = sh.pm[i];
                int rank = 0;
                for (int j = 0; j < np; ++j) rank += sh.pm[j] > mi || (sh.pm[j] == mi && j < i) ? 1 : 0;
                if (rank == int(reach) - 1) sh.key = key_of(mi);
            }
            __syncthreads();
            bound = fmaxf(value_of(sh.key), low);
            complete = k < vocab || bound == low;
        } else if (low > -INFINITY) {
            bound = low;
        } else {
            listed = false;
        }
    }
    if (listed) {
        const float b = bound;
        const int n = collect(x, np, vocab, key_of(b), 0xFFFFFFFFu, [&](int p) { return sh.pm[p] >= b; }, sh);
        if (n <= kList) {
            uint64_t mine[4];
            int rank[4], place[4];
            rank_list(sh, n, top, r.scale, mine, rank, place);
            // w by rank, then its running sums; the weights themselves come back from the keys.
            scan_array(sh.w, n, sh.scratch);
            const int kn = k < n ? int(k) : n;
            const double mass = k < vocab ? sh.w[kn - 1] : whole;
            if (complete || sh.w[n - 1] >= share * mass) {
                const int keep = first_of(n, sh, [&](int i) {
                    return i > 0 && (i >= kn || !(sh.w[i - 1] < share * mass || share > 1.0) ||
                                     !(weight(value_of(uint32_t(sh.sorted[i] >> 32)), top, r.scale) >= least));
                });
                __syncthreads();
                // The kept ones' weights in the order of ids, at the places of all that are listed.
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if (t + q * kThreads < n) {
                        const uint32_t key = uint32_t(mine[q] >> 32);
                        sh.w[place[q]] = rank[q] < keep ? weight(value_of(key), top, r.scale) : 0.0;
                        sh.sorted[place[q]] = mine[q];
                    }
                __syncthreads();
                scan_array(sh.w, n, sh.scratch);
                const double total = sh.w[n - 1], target = double(u) * total;
                int at = first_of(n, sh, [&](int i) { return sh.w[i] > target; });
                if (at >= n) at = first_of(n, sh, [&](int i) { return sh.w[i] == total; });
                if (t == 0) finish(int64_t(~uint32_t(sh.sorted[at])), value_of(uint32_t(sh.sorted[at] >> 32)));
                return;
            }
        }
    }

    // The whole row.
    Kept kept{0, 0, least};
    double of = -1.0;
    if (k < vocab) {
        const Border b = find_border(x, a, top, r.scale, whole, true, k, 0.0, 0.0, sh);
        kept.key = b.key;
        kept.ties = b.ties;
        of = b.mass;
    }
    if (share < 1.0) {
        const Border b = find_border(x, a, top, r.scale, whole, false, 0, share, of, sh);
        if (b.key > kept.key || (b.key == kept.key && b.ties < kept.ties)) {
            kept.key = b.key;
            kept.ties = b.ties;
        }
    }
    const double edge = weight(value_of(kept.key), top, r.scale);  // of the border's own tokens
    const bool with_ties = kept.ties > 0 && edge >= least;
    __syncthreads();
    each_piece(x, np, vocab, every, [&](int p, const float (&v)[8], int c0) {
        double s = 0.0;
        int ties = 0;
        if (key_of(sh.pm[p]) >= kept.key) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t key = key_of(v[e]);
                const double w = weight(v[e], top, r.scale);
                if (key > kept.key && w >= least) s += w;
                ties += with_ties && c0 + e < vocab && key == kept.key ? 1 : 0;
            }
            s = wave_sum(s);
#pragma unroll
            for (int off = kWave / 2; off > 0; off >>= 1) ties += __shfl_xor(ties, off, kWave);
        }
        if (lane == 0) {
            sh.ps[p] = s;
            sh.cnt[p] = uint32_t(ties);
        }
    });
    __syncthreads();
    scan_array(sh.cnt, np, sh.scratch);
    for (int p = t; p < np; p += kThreads) {
        const int64_t before = p > 0 ? sh.cnt[p - 1] : 0, here = int64_t(sh.cnt[p]) - before;
        const int64_t room = kept.ties - before, in = room < 0 ? 0 : room < here ? room : here;
        sh.ps[p] += double(in) * edge;
    }
    __syncthreads();
    scan_array(sh.ps, np, sh.scratch);
    const double total = sh.ps[np - 1], target = double(u) * total;
    int p = first_of(np, sh, [&](int i) { return sh.ps[i] > target; });
    if (p >= np) p = first_of(np, sh, [&](int i) { return sh.ps[i] == total; });
    draw(p, kept, p > 0 ? int64_t(sh.cnt[p - 1]) : 0, p > 0 ? sh.ps[p - 1] : 0.0, target);
}

// Rows of few pieces need no pass of their own over the chip.
constexpr int kInline = 16;

template <typename T> hipError_t sample(SampleArgs &a, int64_t rows, void *workspace, hipStream_t st) {
    if (a.pieces > kInline) {
        a.piece_sum = static_cast<double *>(workspace);
        a.piece_max = reinterpret_cast<float *>(a.piece_sum + rows * a.pieces);
        // 4 pieces a wave where that leaves the chip 4096 waves.
        a.each = rows * a.pieces >= 4 * 4096 ? 4 : 1;
        const dim3 grid(unsigned((a.pieces + 4 * a.each - 1) / (4 * a.each)), unsigned(rows));
        sample_stats_kernel<T><<<grid, 256, 0, st>>>(a);
        if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    sample_select_kernel<T><<<unsigned(rows), kThreads, 0, st>>>(a);
    return hipGetLastError();
}

int64_t pieces_of(int64_t vocab) { return (vocab + kPiece - 1) / kPiece; }
int64_t workspace_of(int64_t rows, int64_t vocab) {
    return pieces_of(vocab) > kInline ? rows * pieces_of(vocab) * 12 : 0;
}
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
    if (rows > 1 && (stride < vocab || stride > (int64_t(1) << 40)))
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
