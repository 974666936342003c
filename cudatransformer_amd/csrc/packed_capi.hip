// C-ABI entry points of attention on packed sequences (declared in include/ctattn.h): the plan, the
// checks of arguments and the choice between the MFMA and the generic kernels.
#include "attn_launch.h"
#include "attn_packed.h"
#include "capi_util.h"
#include "ctattn.h"

#include <algorithm>
#include <cstring>
#include <initializer_list>
#include <new>
#include <vector>

using namespace ctattn;
using ctattn::capi::fail;
using ctattn::capi::finish;
using ctattn::capi::ok;

namespace {

// Row indices are 32-bit, and the kernels add up to 128 keys' rows to one.
constexpr int64_t kMaxRows = (int64_t(1) << 31) - (int64_t(1) << 20);
constexpr int64_t kMaxGroup = 4096;

int64_t tiles_of(int64_t len, int64_t group, int kind) {
    const int64_t n = kind >= kKeys32 ? len : len * group;
    return (n + kPackedTileSize[kind] - 1) / kPackedTileSize[kind];
}

// Sizes of a plan: the header with its offsets and counts filled in.  0 or an error code.
int plan_header(const char *fn, const int64_t *lens, int64_t nseq, int64_t group, PackedHeader &h) {
    if (nseq < 0 || nseq > 0x7FFFFFFF) return fail(hipErrorInvalidValue, "%s: invalid sequence count %lld", fn, (long long)nseq);
    if (nseq > 0 && !lens) return fail(hipErrorInvalidValue, "%s: null lengths", fn);
    if (group < 1 || group > kMaxGroup)
        return fail(hipErrorInvalidValue, "%s: group of %lld query heads (1 to %lld)", fn, (long long)group,
                    (long long)kMaxGroup);
    std::memset(&h, 0, sizeof(h));
    h.magic = kPackedMagic;
    h.nseq = nseq;
    h.group = group;
    int64_t counts[kPackedTiles] = {};
    for (int64_t i = 0; i < nseq; ++i) {
        if (lens[i] < 0) return fail(hipErrorInvalidValue, "%s: length %lld of sequence %lld", fn, (long long)lens[i], (long long)i);
        if (lens[i] > kMaxRows || (h.tokens += lens[i]) > kMaxRows / group)
            return fail(hipErrorInvalidValue, "%s: more than %lld tokens for groups of %lld heads", fn,
                        (long long)(kMaxRows / group), (long long)group);
        h.max_len = std::max(h.max_len, lens[i]);
        h.pairs += lens[i] * lens[i];  // lengths are below 2^31 and sum to less: at most 2^62
        h.pairs_causal += lens[i] * (lens[i] + 1) / 2;
        for (int k = 0; k < kPackedTiles; ++k) counts[k] += tiles_of(lens[i], group, k);
    }
    auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
    int64_t at = up(sizeof(PackedHeader));
    h.cu_offset = at;
    at += up((nseq + 1) * int64_t(sizeof(int32_t)));
    for (int causal = 0; causal < 2; ++causal)
        for (int k = 0; k < kPackedTiles; ++k) {
            h.table[causal][k] = {at, counts[k]};
            at += up(counts[k] * int64_t(sizeof(PackedItem)));
        }
    h.bytes = at;
    return 0;
}

// What a tile costs: the keys its rows see, or the rows that see its keys.
int64_t tile_cost(const PackedItem &it, int64_t group, int kind, bool causal) {
    if (!causal) return it.len;
    const int64_t size = kPackedTileSize[kind];
    if (kind >= kKeys32) return it.len - it.tile * size;
    return std::min<int64_t>(it.len, (it.tile * size + size - 1) / group + 1);
}

struct Sides {
    const void *p;
    const PackedStride *s;
};

int check_call(const char *fn, int dtype, const void *plan_host, const void *plan, int64_t rows, int64_t hq,
               int64_t hkv, int64_t d, const int64_t *strides, PackedCall &c) {
    if (dtype != CTATTN_F32 && dtype != CTATTN_BF16 && dtype != CTATTN_F16 && dtype != CTATTN_F64)
        return fail(hipErrorInvalidValue, "%s: unknown dtype %d (0 = f32, 1 = bf16, 2 = f16, 3 = f64)", fn, dtype);
    if (!plan_host) return fail(hipErrorInvalidValue, "%s: null plan", fn);
    const PackedHeader *h = static_cast<const PackedHeader *>(plan_host);
    if (h->magic != kPackedMagic) return fail(hipErrorInvalidValue, "%s: not a plan of ctattn_packed_plan", fn);
    if (hq < 1 || hkv < 1 || hq % hkv != 0 || hq > 0x7FFFFFFF)
        return fail(hipErrorInvalidValue, "%s: %lld query heads on %lld key heads", fn, (long long)hq, (long long)hkv);
    if (hq / hkv != h->group)
        return fail(hipErrorInvalidValue, "%s: %lld query heads to a key head, the plan has %lld", fn,
                    (long long)(hq / hkv), (long long)h->group);
    if (d < 1 || d > 256)
        return fail(hipErrorNotSupported, "%s: head dim d=%lld unsupported (1 <= d <= 256)", fn, (long long)d);
    if (rows < h->tokens)
        return fail(hipErrorInvalidValue, "%s: tensors of %lld rows, the plan has %lld tokens", fn, (long long)rows,
                    (long long)h->tokens);
    if (h->tokens > 0 && double(h->tokens) * double(hq) > double(kMaxRows) * 64.0)
        return fail(hipErrorInvalidValue, "%s: tokens * heads too large", fn);
    if (!strides) return fail(hipErrorInvalidValue, "%s: null strides", fn);
    if (h->tokens > 0 && !plan) return fail(hipErrorInvalidValue, "%s: null device plan", fn);
    c.dtype = dtype;
    c.host = h;
    c.dev = static_cast<const char *>(plan);
    c.hq = hq;
    c.hkv = hkv;
    c.d = d;
    return 0;
}

// Whether an output's elements are all its own: rows within heads or heads within rows, none folded on another.
bool separate(const PackedStride &s, int64_t rows, int64_t heads, int64_t d) {
    const auto within = [&](int64_t inner, int64_t n_inner, int64_t outer, int64_t n_outer) {
        const int64_t span = n_inner > 1 ? (n_inner - 1) * inner + d : d;
        return (n_inner <= 1 || inner >= d) && (n_outer <= 1 || outer >= span);
    };
    return within(s.head, heads, s.row, rows) || within(s.row, rows, s.head, heads);
}
int check_outputs(const char *fn, std::initializer_list<const PackedStride *> outs, std::initializer_list<int64_t> heads,
                  int64_t rows, int64_t d) {
    auto h = heads.begin();
    for (const PackedStride *s : outs) {
        if (s->row > (int64_t(1) << 40) || s->head > (int64_t(1) << 40) || !separate(*s, rows, *h++, d))
            return fail(hipErrorInvalidValue, "%s: an output's rows or heads overlap (strides %lld, %lld)", fn,
                        (long long)s->row, (long long)s->head);
    }
    return 0;
}

// The bytes of a [rows, heads, d] tensor: `lo`, `hi` its first and last; within a row from `lo` on `span` of them
// every `row`, unless heads lie further apart than rows.
struct Bytes {
    intptr_t lo, hi, row, span;
};
Bytes bytes_of(const void *p, const PackedStride &s, int64_t rows, int64_t heads, int64_t d, int64_t es) {
    const intptr_t at = reinterpret_cast<intptr_t>(p);
    const auto end = [&](int64_t n, int64_t step) { return n > 1 ? (n - 1) * step : 0; };
    const int64_t up = std::max<int64_t>(0, end(rows, s.row)) + std::max<int64_t>(0, end(heads, s.head));
    const int64_t down = std::min<int64_t>(0, end(rows, s.row)) + std::min<int64_t>(0, end(heads, s.head));
    return {at + down * es, at + (up + d) * es, s.row * es, (end(heads, s.head) + d) * es};
}
// Whether two tensors may share a byte.  Slices of one row-major buffer (a projection's q, k, v) do not: their rows are
// equally far apart and each lies in its own part of a row.
bool may_overlap(const Bytes &a, const Bytes &b) {
    if (a.hi <= b.lo || b.hi <= a.lo) return false;
    if (a.row != b.row || a.row <= 0 || a.span <= 0 || b.span <= 0 || a.span > a.row || b.span > a.row) return true;
    const intptr_t shift = ((b.lo - a.lo) % a.row + a.row) % a.row;
    return !(a.span <= shift && shift + b.span <= a.row);
}

// `n` bytes from p on, whole.
Bytes run_of(const void *p, int64_t n) {
    const intptr_t at = reinterpret_cast<intptr_t>(p);
    return {at, at + n, 0, 0};
}

int64_t elem_bytes(int dtype) { return dtype == CTATTN_F64 ? 8 : dtype == CTATTN_F32 ? 4 : 2; }

// A stride that is never stepped along (one head, one token) may hold anything: 0, so that it decides nothing.
void settle(PackedCall &c) {
    const int64_t heads[] = {c.hq, c.hkv, c.hkv, c.hq, c.hq, c.hq, c.hkv, c.hkv};
    PackedStride *const all[] = {&c.sq, &c.sk, &c.sv, &c.so, &c.sdo, &c.sdq, &c.sdk, &c.sdv};
    for (int i = 0; i < 8; ++i) {
        if (heads[i] == 1) all[i]->head = 0;
        if (c.tokens() <= 1) all[i]->row = 0;
    }
}

// The MFMA kernels move 16 bytes per access: pointers and strides on 16 bytes.
bool on16(const Sides &x, int dtype) {
    const int64_t e = elem_bytes(dtype);
    return reinterpret_cast<uintptr_t>(x.p) % 16 == 0 && (x.s->row * e) % 16 == 0 && (x.s->head * e) % 16 == 0;
}

Bytes lse_bytes(const void *lse, const PackedCall &c) {
    return run_of(lse, c.tokens() * c.hq * (c.dtype == CTATTN_F64 ? 8 : 4));
}

bool mfma(const PackedCall &c) {
    return ctattn_get_policy() != CTATTN_POLICY_GENERIC && packed_mfma_supported(c.dtype, c.d, c.group());
}

int64_t scratch_bytes(const PackedCall &c) {
    const int64_t generic = c.tokens() * c.hq * (c.dtype == CTATTN_F64 ? 8 : 4);
    return packed_mfma_supported(c.dtype, c.d, c.group()) ? std::max(generic, packed_bwd_scratch_bytes(c)) : generic;
}

}  // namespace

extern "C" {

int64_t ctattn_packed_plan_bytes(const int64_t *seqlens, int64_t nseq, int64_t group) {
    PackedHeader h;
    if (plan_header("ctattn_packed_plan_bytes", seqlens, nseq, group, h) != 0) return -1;
    return h.bytes;
}

int ctattn_packed_plan(const int64_t *seqlens, int64_t nseq, int64_t group, void *out, int64_t bytes) {
    const char *fn = "ctattn_packed_plan";
    PackedHeader h;
    if (int rc = plan_header(fn, seqlens, nseq, group, h)) return rc;
    if (!out) return fail(hipErrorInvalidValue, "%s: null buffer", fn);
    if (bytes < h.bytes)
        return fail(hipErrorInvalidValue, "%s: buffer too small (%lld bytes, %lld needed)", fn, (long long)bytes,
                    (long long)h.bytes);
    try {
        char *p = static_cast<char *>(out);
        std::memset(p, 0, size_t(h.bytes));
        std::memcpy(p, &h, sizeof(h));
        int32_t *cu = reinterpret_cast<int32_t *>(p + h.cu_offset);
        for (int64_t i = 0; i < nseq; ++i) cu[i + 1] = cu[i] + int32_t(seqlens[i]);
        std::vector<int64_t> place(size_t(h.max_len) + 2);
        for (int causal = 0; causal < 2; ++causal)
            for (int k = 0; k < kPackedTiles; ++k) {
                // By cost, the largest first, in one counting pass and one that places; equal ones in order. A
                // cost is at most the longest sequence, and both passes over `place` are as long: 26 documents of
                // 14.7k tokens, the longest 3011, 45 to 79 us of one core (a stable sort of the items 424), one sequence of
                // 8192 tokens 71, of 131072 1.2 ms, of a million 14 ms.
                PackedItem *items = reinterpret_cast<PackedItem *>(p + h.table[causal][k].offset);
                std::fill(place.begin(), place.end(), 0);
                const auto each = [&](auto fn) {
                    for (int64_t i = 0; i < nseq; ++i)
                        for (int64_t t = 0, e = tiles_of(seqlens[i], group, k); t < e; ++t) {
                            const PackedItem it{cu[i], int32_t(seqlens[i]), int32_t(t), int32_t(i)};
                            fn(it, size_t(h.max_len - tile_cost(it, group, k, causal != 0)));
                        }
                };
                each([&](const PackedItem &, size_t c) { ++place[c + 1]; });
                for (size_t c = 1; c < place.size(); ++c) place[c] += place[c - 1];
                each([&](const PackedItem &it, size_t c) { items[place[c]++] = it; });
            }
    } catch (const std::exception &) {
        return fail(hipErrorOutOfMemory, "%s: out of host memory", fn);
    }
    return ok();
}

int ctattn_packed_fwd(int dtype, const void *q, const void *k, const void *v, void *o, void *lse,
                      const int64_t *strides, const void *plan_host, const void *plan, int64_t rows, int64_t hq,
                      int64_t hkv, int64_t d, int causal, void *stream) {
    const char *fn = "ctattn_packed_fwd";
    PackedCall c{};
    if (int rc = check_call(fn, dtype, plan_host, plan, rows, hq, hkv, d, strides, c)) return rc;
    c.causal = causal != 0;
    c.sq = {strides[0], strides[1]};
    c.sk = {strides[2], strides[3]};
    c.sv = {strides[4], strides[5]};
    c.so = {strides[6], strides[7]};
    settle(c);
    if (c.tokens() == 0) return ok();
    if (int rc = check_outputs(fn, {&c.so}, {hq}, c.tokens(), d)) return rc;
    if (!q || !k || !v || !o) return fail(hipErrorInvalidValue, "%s: null q/k/v/o pointer", fn);
    const int64_t es = elem_bytes(dtype);
    const Bytes bo = bytes_of(o, c.so, c.tokens(), hq, d, es);
    const Bytes in[] = {bytes_of(q, c.sq, c.tokens(), hq, d, es), bytes_of(k, c.sk, c.tokens(), hkv, d, es),
                        bytes_of(v, c.sv, c.tokens(), hkv, d, es)};
    for (const Bytes &b : in) {
        if (may_overlap(bo, b)) return fail(hipErrorInvalidValue, "%s: o lies on an input's memory", fn);
        if (lse && may_overlap(lse_bytes(lse, c), b)) return fail(hipErrorInvalidValue, "%s: lse lies on an input's memory", fn);
    }
    if (lse && may_overlap(lse_bytes(lse, c), bo)) return fail(hipErrorInvalidValue, "%s: lse lies on o's memory", fn);
    hipStream_t st = static_cast<hipStream_t>(stream);
    const Sides all[] = {{q, &c.sq}, {k, &c.sk}, {v, &c.sv}, {o, &c.so}};
    const bool fast = mfma(c) && std::all_of(std::begin(all), std::end(all), [&](const Sides &x) { return on16(x, dtype); });
    return finish(fn,
                  fast ? launch_packed_fwd(c, q, k, v, o, static_cast<float *>(lse), st)
                       : launch_packed_generic_fwd(c, q, k, v, o, lse, st),
                  st);
}

int64_t ctattn_packed_bwd_workspace_bytes(int dtype, const void *plan_host, int64_t hq, int64_t hkv, int64_t d) {
    PackedCall c{};
    const int64_t any[16] = {};  // strides and rows play no part
    if (check_call("ctattn_packed_bwd_workspace_bytes", dtype, plan_host, any, kMaxRows, hq, hkv, d, any, c) != 0) return -1;
    return scratch_bytes(c);
}

int ctattn_packed_bwd(int dtype, const void *q, const void *k, const void *v, const void *o, const void *dout,
                      const void *lse, void *dq, void *dk, void *dv, void *workspace, int64_t workspace_bytes,
                      const int64_t *strides, const void *plan_host, const void *plan, int64_t rows, int64_t hq,
                      int64_t hkv, int64_t d, int causal, void *stream) {
    const char *fn = "ctattn_packed_bwd";
    PackedCall c{};
    if (int rc = check_call(fn, dtype, plan_host, plan, rows, hq, hkv, d, strides, c)) return rc;
    c.causal = causal != 0;
    PackedStride *const to[] = {&c.sq, &c.sk, &c.sv, &c.so, &c.sdo, &c.sdq, &c.sdk, &c.sdv};
    for (int i = 0; i < 8; ++i) *to[i] = {strides[2 * i], strides[2 * i + 1]};
    settle(c);
    if (c.tokens() == 0) return ok();
    if (int rc = check_outputs(fn, {&c.sdq, &c.sdk, &c.sdv}, {hq, hkv, hkv}, c.tokens(), d)) return rc;
    if (!q || !k || !v || !o || !dout || !lse || !dq || !dk || !dv)
        return fail(hipErrorInvalidValue, "%s: null tensor pointer", fn);
    const int64_t es = elem_bytes(dtype), n = c.tokens();
    const Bytes in[] = {bytes_of(q, c.sq, n, hq, d, es),  bytes_of(k, c.sk, n, hkv, d, es), bytes_of(v, c.sv, n, hkv, d, es),
                        bytes_of(o, c.so, n, hq, d, es),  bytes_of(dout, c.sdo, n, hq, d, es), lse_bytes(lse, c)};
    const Bytes out[] = {bytes_of(dq, c.sdq, n, hq, d, es), bytes_of(dk, c.sdk, n, hkv, d, es), bytes_of(dv, c.sdv, n, hkv, d, es)};
    for (int i = 0; i < 3; ++i) {
        for (const Bytes &b : in)
            if (may_overlap(out[i], b)) return fail(hipErrorInvalidValue, "%s: a gradient lies on an input's memory", fn);
        for (int j = 0; j < i; ++j)
            if (may_overlap(out[i], out[j])) return fail(hipErrorInvalidValue, "%s: two gradients share memory", fn);
    }
    const int64_t need = scratch_bytes(c);
    if (!workspace || workspace_bytes < need)
        return fail(hipErrorInvalidValue, "%s: workspace too small (%lld bytes, %lld needed)", fn,
                    (long long)workspace_bytes, (long long)need);
    if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
        return fail(hipErrorInvalidValue, "%s: workspace must be 16-byte aligned", fn);
    const Bytes ws = run_of(workspace, need);
    const auto on_ws = [&](const Bytes &b) { return may_overlap(ws, b); };
    if (std::any_of(std::begin(in), std::end(in), on_ws) || std::any_of(std::begin(out), std::end(out), on_ws))
        return fail(hipErrorInvalidValue, "%s: workspace lies on a tensor's memory", fn);
    hipStream_t st = static_cast<hipStream_t>(stream);
    const Sides all[] = {{q, &c.sq}, {k, &c.sk}, {v, &c.sv}, {o, &c.so}, {dout, &c.sdo}, {dq, &c.sdq}, {dk, &c.sdk}, {dv, &c.sdv}};
    const bool fast = mfma(c) && std::all_of(std::begin(all), std::end(all), [&](const Sides &x) { return on16(x, dtype); });
    return finish(fn,
                  fast ? launch_packed_bwd(c, q, k, v, o, dout, static_cast<const float *>(lse), workspace, dq, dk, dv, st)
                       : launch_packed_generic_bwd(c, q, k, v, o, dout, lse, workspace, dq, dk, dv, st),
                  st);
}

}  // extern "C"
