// The bookkeeping of a paged key / value cache on the device, and writes into it.
//
// ctattn_page_reserve gives a step's requests the pages that their new tokens need, from a ring of free ones, and
// says where every token goes; ctattn_page_release gives a finished request's pages back; ctattn_cache_write puts
// keys and values there.  No length crosses to the host, so that a captured step replays on other lengths.
//
// Pages are dealt in the order of the requests: two running sums, of new tokens (a request's first row) and of
// the pages needed by those that fit.  Every workgroup computes both sums for itself over all requests, thread t over
// ceil(B / threads) of them in a row, instead of waiting for another launch, and then writes its share: the
// requests of its own threads (table, lengths, starts) and a window of 2 rows a thread.  A row finds its request
// by a running maximum over marks that requests leave in LDS at their first row of the window.  All outputs are
// functions of the inputs, whose order is fixed: no atomics.
//
// Latency bounds the bookkeeping: a token of each of 256 requests 5.6 us, prompts of 60 tokens of 2048 requests (61
// workgroups, 122880 rows) 12.9, a third of 1024 requests with 125 pages each given back 6.8.
#include "attn_common.h"
#include "attn_launch.h"
#include "capi_bytes.h"
#include "capi_util.h"
#include "ctattn.h"

#include <algorithm>

namespace ctattn {
namespace {

__device__ __forceinline__ int64_t least(int64_t a, int64_t b) { return a < b ? a : b; }
__device__ __forceinline__ int64_t most(int64_t a, int64_t b) { return a > b ? a : b; }

// Inclusive sums or maxima over a workgroup's threads.
template <int NT, typename Op> __device__ __forceinline__ int64_t block_scan(int64_t x, int64_t *waves, Op op) {
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
        const int64_t y = __shfl_up(x, off, kWave);
        if (lane >= off) x = op(x, y);
    }
    __syncthreads();  // the last scan's reads of `waves` are done
    if (lane == kWave - 1) waves[wave] = x;
    __syncthreads();
    for (int w = 0; w < wave; ++w) x = op(x, waves[w]);
    return x;
}
struct Sum {
    __device__ int64_t operator()(int64_t a, int64_t b) const { return a + b; }
};
struct Max {
    __device__ int64_t operator()(int64_t a, int64_t b) const { return a > b ? a : b; }
};

// (base + x) mod n for 0 <= base < n, 0 <= x <= n.
__device__ __forceinline__ int64_t around(int64_t base, int64_t x, int64_t n) {
    const int64_t y = base + x;
    return y >= n ? y - n : y;
}
__device__ __forceinline__ int64_t mod(int64_t x, int64_t n) {
    const int64_t r = x % n;
    return r < 0 ? r + n : r;
}

struct Pool {
    int32_t *free;  // a ring of n places; the free pages are in taken .. given - 1
    const int64_t *counters;
    int64_t *counters_out;
    int64_t n;
};

struct ReserveArgs {
    const int32_t *lens, *fresh, *offsets;
    int32_t *table;
    int64_t table_row;
    Pool pool;
    int64_t *slots, *positions;
    int32_t *starts, *lens_out;
    int64_t requests, width, tokens;
    int shift;
};

template <int NT> __global__ __launch_bounds__(NT) void page_reserve_kernel(ReserveArgs a) {
    constexpr int ROWS = 2 * NT;
    __shared__ int64_t waves[NT / kWave];
    __shared__ int32_t mark[ROWS], req[ROWS];
    __shared__ int32_t base[ROWS];  // of the request's first fresh page among the free ones; -1: it got none
    __shared__ int64_t head_start, end;
    __shared__ int32_t head_req, head_base;
    const int t = threadIdx.x, lane = t & (kWave - 1);
    const int64_t each = (a.requests + NT - 1) / NT, i0 = t * each, i1 = least(a.requests, i0 + each);
    const int64_t w0 = int64_t(blockIdx.x) * ROWS;
    const int64_t page = int64_t(1) << a.shift;
    const bool mine = int64_t(t) * gridDim.x / NT == blockIdx.x;  // this thread's requests are written here
    const int64_t taken = a.pool.counters[0], given = a.pool.counters[1];
    const int64_t avail = least(most(given - taken, int64_t(0)), a.pool.n);
    const int64_t ring = a.pool.n > 0 ? mod(taken, a.pool.n) : 0;

    for (int r = t; r < ROWS; r += NT) mark[r] = -1;
    if (t == 0) head_req = -1;
    int64_t tok = 0;
    for (int64_t i = i0; i < i1; ++i) tok += most(a.fresh[i], 0);
    const int64_t upto = block_scan<NT>(tok, waves, Sum{});
    if (t == NT - 1) end = upto;
    struct One {
        int64_t len, add, held, need;
        bool fits;
    };
    // Request i, whose tokens begin at row `start`.
    const auto one = [&](int64_t i, int64_t start) {
        One x;
        x.len = most(a.lens[i], 0);
        x.add = most(a.fresh[i], 0);
        x.held = (x.len + page - 1) >> a.shift;
        const int64_t pages = (x.len + x.add + page - 1) >> a.shift;
        x.fits = pages <= a.width && start + x.add <= a.tokens;
        x.need = x.fits ? pages - x.held : 0;
        return x;
    };
    int64_t need = 0, start = upto - tok;
    for (int64_t i = i0; i < i1; ++i) {
        const One x = one(i, start);
        need += x.need;
        start += x.add;
    }
    int64_t at = block_scan<NT>(need, waves, Sum{}) - need, used = 0;
    start = upto - tok;
    for (int64_t k = 0; k < each; ++k) {
        const int64_t i = i0 + k;
        One x{0, 0, 0, 0, false};
        bool ok = false;
        if (i < i1) {
            x = one(i, start);
            ok = x.fits && (x.need == 0 || at + x.need <= avail);
            if (ok && x.need > 0) used = at + x.need;
            if (mine) {
                a.starts[i] = int32_t(least(start, int64_t(0x7FFFFFFF)));
                a.lens_out[i] = ok ? int32_t(x.len + x.add) : a.lens[i];
            }
            if (x.add > 0 && start < w0 + ROWS && start + x.add > w0) {
                const int32_t b = ok ? int32_t(at) : -1;
                if (start >= w0) {
                    const int r = int(start - w0);
                    mark[r] = r;
                    req[r] = int32_t(i);
                    base[r] = b;
                } else {
                    head_start = start;
                    head_req = int32_t(i);
                    head_base = b;
                }
            }
        }
        // Few pages by the thread itself, many by its wave.
        const bool write = mine && ok && x.need > 0;
        if (write && x.need <= 16)
            for (int64_t j = 0; j < x.need; ++j)
                a.table[i * a.table_row + x.held + j] = a.pool.free[around(ring, at + j, a.pool.n)];
        for (uint64_t big = __ballot(write && x.need > 16); big != 0; big &= big - 1) {
            const int from = __ffsll((unsigned long long)big) - 1;
            const int64_t bi = __shfl(i, from, kWave), bh = __shfl(x.held, from, kWave);
            const int64_t bn = __shfl(x.need, from, kWave), ba = __shfl(at, from, kWave);
            for (int64_t j = lane; j < bn; j += kWave)
                a.table[bi * a.table_row + bh + j] = a.pool.free[around(ring, ba + j, a.pool.n)];
        }
        at += x.need;
        start += x.add;
    }
    used = block_scan<NT>(used, waves, Max{});
    if (blockIdx.x == 0 && t == NT - 1) {
        a.starts[a.requests] = int32_t(least(end, int64_t(0x7FFFFFFF)));
        a.pool.counters_out[0] = taken + used;
        a.pool.counters_out[1] = given;
    }
    // The last marked row at or before each: where its request's rows begin.
    const int64_t before = t == 0 ? -1 : most(mark[2 * t - 2], mark[2 * t - 1]);
    int from = int(block_scan<NT>(before, waves, Max{}));
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int r = 2 * t + k;
        const int64_t row = w0 + r;
        if (row >= a.tokens) break;
        from = int(most(from, mark[r]));
        const int64_t i = from >= 0 ? req[from] : head_req;
        const int64_t b = from >= 0 ? base[from] : head_base;
        int64_t slot = -1, pos = 0;
        if (row < end && i >= 0 && b >= 0) {
            const int64_t len = most(a.lens[i], 0), held = (len + page - 1) >> a.shift;
            pos = len + row - (from >= 0 ? w0 + from : head_start);
            const int64_t p = pos >> a.shift;
            const int32_t id = p < held ? a.table[i * a.table_row + p] : a.pool.free[around(ring, b + p - held, a.pool.n)];
            slot = int64_t(id) * page + (pos & (page - 1));
            if (a.offsets != nullptr) pos += a.offsets[i];
        }
        a.slots[row] = slot;
        a.positions[row] = pos;
    }
}

struct ReleaseArgs {
    const uint8_t *done;
    const int32_t *lens, *table;
    int64_t table_row;
    Pool pool;
    int32_t *lens_out;
    int64_t requests, width;
    int shift;
};

template <int NT> __global__ __launch_bounds__(NT) void page_release_kernel(ReleaseArgs a) {
    __shared__ int64_t waves[NT / kWave];
    const int t = threadIdx.x, lane = t & (kWave - 1);
    const int64_t each = (a.requests + NT - 1) / NT, i0 = t * each, i1 = least(a.requests, i0 + each);
    const bool mine = int64_t(t) * gridDim.x / NT == blockIdx.x;
    const int64_t taken = a.pool.counters[0], given = a.pool.counters[1];
    const int64_t room = least(most(a.pool.n - (given - taken), int64_t(0)), a.pool.n);
    const int64_t ring = a.pool.n > 0 ? mod(given, a.pool.n) : 0;
    const auto back = [&](int64_t i) {
        if (!a.done[i]) return int64_t(0);
        const int64_t held = (int64_t(most(a.lens[i], 0)) + (int64_t(1) << a.shift) - 1) >> a.shift;
        return least(held, a.width);
    };
    int64_t n = 0;
    for (int64_t i = i0; i < i1; ++i) n += back(i);
    int64_t at = block_scan<NT>(n, waves, Sum{}) - n, used = 0;
    for (int64_t k = 0; k < each; ++k) {
        const int64_t i = i0 + k;
        int64_t pages = 0;
        bool ok = false;
        if (i < i1) {
            pages = back(i);
            ok = a.done[i] && at + pages <= room;
            if (ok) used = at + pages;
            if (mine) a.lens_out[i] = ok ? 0 : a.lens[i];
        }
        for (uint64_t some = __ballot(mine && ok && pages > 0); some != 0; some &= some - 1) {
            const int from = __ffsll((unsigned long long)some) - 1;
            const int64_t bi = __shfl(i, from, kWave), bn = __shfl(pages, from, kWave), ba = __shfl(at, from, kWave);
            for (int64_t j = lane; j < bn; j += kWave)
                a.pool.free[around(ring, ba + j, a.pool.n)] = a.table[bi * a.table_row + j];
        }
        at += pages;
    }
    used = block_scan<NT>(used, waves, Max{});
    if (blockIdx.x == 0 && t == NT - 1) {
        a.pool.counters_out[0] = taken;
        a.pool.counters_out[1] = given + used;
    }
}

// ---- writes into the cache ----

struct Rows {
    const char *p;
    int64_t row, head;  // bytes
};
struct Pages {
    char *p;
    int64_t page, token, head;
};

// A unit (16 bytes, or an element where something lies off 16) of a row's keys and of its values a thread.  HBM bounds it:
// 40000 rows of 8 bf16 heads of 128 (328 MB read and written) 60 us, 5.4 TB/s; 256 such rows 2.9 us.
template <typename U>
__global__ __launch_bounds__(256) void cache_write_kernel(Rows k, Rows v, Pages kc, Pages vc,
                                                          const int64_t *__restrict__ slots, int64_t rows, int hkv,
                                                          int per, int64_t places, int shift) {
    const int units = hkv * per;
    const int64_t total = rows * units;
    for (int64_t x = int64_t(blockIdx.x) * 256 + threadIdx.x; x < total; x += int64_t(gridDim.x) * 256) {
        // 64-bit division only where a tensor has as many units.
        const int64_t n = total <= 0x7FFFFFFF ? int64_t(uint32_t(x) / uint32_t(units)) : x / units;
        const int u = int(x - n * units), h = u / per, c = (u - h * per) * int(sizeof(U));
        const int64_t slot = slots[n];
        if (slot < 0 || slot >= places) continue;
        const int64_t page = slot >> shift, in = slot & ((int64_t(1) << shift) - 1);
        const U a = *reinterpret_cast<const U *>(k.p + n * k.row + h * k.head + c);
        const U b = *reinterpret_cast<const U *>(v.p + n * v.row + h * v.head + c);
        *reinterpret_cast<U *>(kc.p + page * kc.page + in * kc.token + h * kc.head + c) = a;
        *reinterpret_cast<U *>(vc.p + page * vc.page + in * vc.token + h * vc.head + c) = b;
    }
}

template <typename U>
hipError_t write(const Rows &k, const Rows &v, const Pages &kc, const Pages &vc, const int64_t *slots, int64_t rows,
                 int64_t hkv, int64_t bytes, int64_t places, int shift, hipStream_t st) {
    const int per = int(bytes / int64_t(sizeof(U)));
    cache_write_kernel<U><<<stride_grid((rows * hkv * per + 255) / 256, 256), 256, 0, st>>>(
        k, v, kc, vc, slots, rows, int(hkv), per, places, shift);
    return hipGetLastError();
}

int shift_of(int64_t page_size) {
    int s = 0;
    while ((int64_t(1) << s) < page_size) ++s;
    return s;
}

constexpr int64_t kMost = 0x7FFFFFFF;

int check_pages(const char *fn, int64_t requests, int64_t table_row, int64_t width, int64_t free_places, int64_t page_size) {
    using capi::fail;
    if (page_size < 1 || page_size > (1 << 20) || (page_size & (page_size - 1)) != 0)
        return fail(hipErrorInvalidValue, "%s: page size %lld (a power of two up to 2^20)", fn, (long long)page_size);
    if (requests < 0 || requests > (1 << 24) || width < 0 || width > kMost || free_places < 0 || free_places > kMost)
        return fail(hipErrorInvalidValue, "%s: invalid sizes: %lld requests, table %lld wide, %lld places for free pages", fn,
                    (long long)requests, (long long)width, (long long)free_places);
    if (width * page_size > kMost)
        return fail(hipErrorInvalidValue, "%s: a table of %lld pages of %lld tokens passes 2^31 - 1 tokens", fn, (long long)width,
                    (long long)page_size);
    if (requests > 1 && (table_row < width || table_row > (int64_t(1) << 40)))
        return fail(hipErrorInvalidValue, "%s: table rows %lld apart, %lld wide", fn, (long long)table_row, (long long)width);
    return 0;
}

}  // namespace
}  // namespace ctattn

using namespace ctattn;
using namespace ctattn::capi;

extern "C" {

int ctattn_page_reserve(const int32_t *lens, const int32_t *new_lens, const int32_t *offsets, int32_t *table,
                        const int32_t *free_pages, const int64_t *counters, int64_t *slots, int64_t *positions,
                        int32_t *starts, int32_t *lens_out, int64_t *counters_out, int64_t requests, int64_t table_row,
                        int64_t table_width, int64_t free_places, int64_t page_size, int64_t max_tokens, void *stream) {
    const char *fn = "ctattn_page_reserve";
    if (int rc = check_pages(fn, requests, table_row, table_width, free_places, page_size)) return rc;
    if (max_tokens < 0 || max_tokens > kMost)
        return fail(hipErrorInvalidValue, "%s: max_tokens %lld", fn, (long long)max_tokens);
    if (!counters || !starts || !counters_out || (max_tokens > 0 && (!slots || !positions)) ||
        (requests > 0 && (!lens || !new_lens || !lens_out || (!table && table_width > 0))) || (free_places > 0 && !free_pages))
        return fail(hipErrorInvalidValue, "%s: null pointer", fn);
    const int64_t b4 = requests * 4;
    const Bytes in[] = {run_of(lens, b4), run_of(new_lens, b4), run_of(offsets, offsets ? b4 : 0), run_of(free_pages, free_places * 4),
                        run_of(counters, 16)};
    const Bytes out[] = {run_of(table, requests > 0 ? ((requests - 1) * table_row + table_width) * 4 : 0), run_of(slots, max_tokens * 8),
                         run_of(positions, max_tokens * 8), run_of(starts, b4 + 4), run_of(lens_out, b4), run_of(counters_out, 16)};
    if (int rc = check_apart(fn, in, out)) return rc;
    ReserveArgs a{lens, new_lens, offsets, table, table_row, {const_cast<int32_t *>(free_pages), counters, counters_out, free_places},
                  slots, positions, starts, lens_out, requests, table_width, max_tokens, shift_of(page_size)};
    hipStream_t st = static_cast<hipStream_t>(stream);
    // 1024 threads where either sum is long; 256 start sooner.
    if (requests <= 256 && max_tokens <= 512) {
        page_reserve_kernel<256><<<1, 256, 0, st>>>(a);
    } else {
        const int64_t blocks = std::max<int64_t>(1, (max_tokens + 2047) / 2048);
        if (!grid_fits(blocks, 1024)) return fail(hipErrorInvalidValue, "%s: max_tokens %lld", fn, (long long)max_tokens);
        page_reserve_kernel<1024><<<unsigned(blocks), 1024, 0, st>>>(a);
    }
    return finish(fn, hipGetLastError(), st);
}

int ctattn_page_release(const void *done, const int32_t *lens, const int32_t *table, int32_t *free_pages,
                        const int64_t *counters, int32_t *lens_out, int64_t *counters_out, int64_t requests,
                        int64_t table_row, int64_t table_width, int64_t free_places, int64_t page_size, void *stream) {
    const char *fn = "ctattn_page_release";
    if (int rc = check_pages(fn, requests, table_row, table_width, free_places, page_size)) return rc;
    if (!counters || !counters_out || (requests > 0 && (!done || !lens || !lens_out || (!table && table_width > 0))) ||
        (free_places > 0 && !free_pages))
        return fail(hipErrorInvalidValue, "%s: null pointer", fn);
    const int64_t b4 = requests * 4;
    const Bytes in[] = {run_of(done, requests), run_of(lens, b4), run_of(counters, 16),
                        run_of(table, requests > 0 ? ((requests - 1) * table_row + table_width) * 4 : 0)};
    const Bytes out[] = {run_of(free_pages, free_places * 4), run_of(lens_out, b4), run_of(counters_out, 16)};
    if (int rc = check_apart(fn, in, out)) return rc;
    ReleaseArgs a{static_cast<const uint8_t *>(done), lens, table, table_row, {free_pages, counters, counters_out, free_places},
                  lens_out, requests, table_width, shift_of(page_size)};
    hipStream_t st = static_cast<hipStream_t>(stream);
    // A workgroup for 8 requests, whose pages a wave copies one request after the other (1024 requests, a third done: 16
    // workgroups 11.8 us, 128 6.8 us).
    const unsigned blocks = unsigned(std::max<int64_t>(1, std::min<int64_t>(128, requests / 8)));
    if (requests <= 256) page_release_kernel<256><<<blocks, 256, 0, st>>>(a);
    else page_release_kernel<1024><<<blocks, 1024, 0, st>>>(a);
    return finish(fn, hipGetLastError(), st);
}

int ctattn_cache_write(int dtype, const void *k, const void *v, void *k_cache, void *v_cache, const int64_t *slots,
                       const int64_t *strides, int64_t rows, int64_t hkv, int64_t d, int64_t pages, int64_t page_size,
                       void *stream) {
    const char *fn = "ctattn_cache_write";
    if (dtype != CTATTN_F32 && dtype != CTATTN_BF16 && dtype != CTATTN_F16 && dtype != CTATTN_F64)
        return fail(hipErrorInvalidValue, "%s: unknown dtype %d (0 = f32, 1 = bf16, 2 = f16, 3 = f64)", fn, dtype);
    if (rows < 0 || rows > kMost || hkv < 1 || hkv > kMost || d < 1 || d > kMost || hkv * d > (1 << 28) || pages < 0 || pages > kMost)
        return fail(hipErrorInvalidValue, "%s: invalid sizes rows=%lld hkv=%lld d=%lld pages=%lld", fn, (long long)rows,
                    (long long)hkv, (long long)d, (long long)pages);
    if (page_size < 1 || page_size > (1 << 20) || (page_size & (page_size - 1)) != 0)
        return fail(hipErrorInvalidValue, "%s: page size %lld (a power of two up to 2^20)", fn, (long long)page_size);
    if (!strides) return fail(hipErrorInvalidValue, "%s: null strides", fn);
    if (rows == 0 || pages == 0) return ok();
    if (!k || !v || !k_cache || !v_cache || !slots) return fail(hipErrorInvalidValue, "%s: null pointer", fn);
    const int64_t es = dtype == CTATTN_F64 ? 8 : dtype == CTATTN_F32 ? 4 : 2;
    int64_t st_[10];
    const int64_t extent[10] = {rows, hkv, rows, hkv, pages, page_size, hkv, pages, page_size, hkv};
    if (int rc = check_strides(fn, strides, extent, 10, st_)) return rc;
    for (int64_t &s : st_) s *= es;
    const Rows kr{static_cast<const char *>(k), st_[0], st_[1]}, vr{static_cast<const char *>(v), st_[2], st_[3]};
    const Pages kc{static_cast<char *>(k_cache), st_[4], st_[5], st_[6]}, vc{static_cast<char *>(v_cache), st_[7], st_[8], st_[9]};
    const Bytes in[] = {span_of(k, st_, extent, 2, d * es), span_of(v, st_ + 2, extent + 2, 2, d * es), run_of(slots, rows * 8)};
    // The two caches may be slices of one buffer.
    const Bytes out[] = {span_of(k_cache, st_ + 4, extent + 4, 3, d * es), span_of(v_cache, st_ + 7, extent + 7, 3, d * es)};
    for (const Bytes &o : out)
        for (const Bytes &i : in)
            if (may_overlap(o, i)) return fail(hipErrorInvalidValue, "%s: a cache lies on an input's memory", fn);
    int64_t all = reinterpret_cast<intptr_t>(k) | reinterpret_cast<intptr_t>(v) | reinterpret_cast<intptr_t>(k_cache) |
                  reinterpret_cast<intptr_t>(v_cache) | (d * es);
    for (int64_t s : st_) all |= s;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int64_t places = pages * page_size, bytes = d * es;
    const int shift = shift_of(page_size);
    hipError_t e;
    if (all % 16 == 0) e = write<uint4>(kr, vr, kc, vc, slots, rows, hkv, bytes, places, shift, st);
    else if (es == 8) e = write<uint64_t>(kr, vr, kc, vc, slots, rows, hkv, bytes, places, shift, st);
    else if (es == 4) e = write<uint32_t>(kr, vr, kc, vc, slots, rows, hkv, bytes, places, shift, st);
    else e = write<uint16_t>(kr, vr, kc, vc, slots, rows, hkv, bytes, places, shift, st);
    return finish(fn, e, st);
}

}  // extern "C"
