// C-ABI entry point of attention of requests that share a prompt (declared in include/ctattn.h): the checks of
// arguments and the choice between the MFMA and the generic kernels.
#include "attn_shared.h"
#include "capi_bytes.h"
#include "capi_util.h"
#include "ctattn.h"

#include <algorithm>

using namespace ctattn;
using namespace ctattn::capi;

namespace {

constexpr int64_t kMost = (int64_t(1) << 31) - (int64_t(1) << 20);  // rows of (token, head), tokens of a table

int64_t elem_bytes(int dtype) { return dtype == CTATTN_F64 ? 8 : dtype == CTATTN_F32 ? 4 : 2; }

int check_sizes(const char *fn, const SharedCall &c) {
    if (c.dtype != CTATTN_F32 && c.dtype != CTATTN_BF16 && c.dtype != CTATTN_F16 && c.dtype != CTATTN_F64)
        return fail(hipErrorInvalidValue, "%s: unknown dtype %d (0 = f32, 1 = bf16, 2 = f16, 3 = f64)", fn, c.dtype);
    if (c.hq < 1 || c.hkv < 1 || c.hq > 65536 || c.hq % c.hkv != 0)
        return fail(hipErrorInvalidValue, "%s: %lld query heads on %lld key heads", fn, (long long)c.hq, (long long)c.hkv);
    if (c.d < 1 || c.d > 256)
        return fail(hipErrorNotSupported, "%s: head dim d=%lld unsupported (1 <= d <= 256)", fn, (long long)c.d);
    if (c.page_size < 1 || c.page_size > (1 << 20) || (c.page_size & (c.page_size - 1)) != 0)
        return fail(hipErrorInvalidValue, "%s: page size %lld (a power of two up to 2^20)", fn, (long long)c.page_size);
    if (c.rows < 0 || c.rows > kMost / c.hq || c.requests < 0 || c.requests > (1 << 24) || c.groups < 0 || c.groups > (1 << 24))
        return fail(hipErrorInvalidValue, "%s: invalid sizes: %lld rows of %lld heads, %lld requests in %lld groups", fn,
                    (long long)c.rows, (long long)c.hq, (long long)c.requests, (long long)c.groups);
    if (c.pages < 0 || c.pages > 0x7FFFFFFF || c.table_width < 0 || c.prefix_width < 0 || c.table_width > kMost / c.page_size ||
        c.prefix_width > kMost / c.page_size)
        return fail(hipErrorInvalidValue, "%s: tables of %lld and %lld pages of %lld tokens", fn, (long long)c.table_width,
                    (long long)c.prefix_width, (long long)c.page_size);
    return 0;
}

// Whether an output's elements are all its own.
bool separate(const SharedStride &s, int64_t rows, int64_t heads, int64_t d) {
    const auto within = [&](int64_t inner, int64_t n_inner, int64_t outer, int64_t n_outer) {
        const int64_t span = n_inner > 1 ? (n_inner - 1) * inner + d : d;
        return (n_inner <= 1 || inner >= d) && (n_outer <= 1 || outer >= span);
    };
    return within(s.head, heads, s.row, rows) || within(s.row, rows, s.head, heads);
}

}  // namespace

extern "C" {

int64_t ctattn_shared_prefix_workspace_bytes(int dtype, int64_t rows, int64_t requests, int64_t groups, int64_t hq,
                                             int64_t hkv, int64_t d, int64_t page_size, int64_t table_width,
                                             int64_t prefix_width) {
    SharedCall c{};
    c.dtype = dtype;
    c.rows = rows;
    c.requests = requests;
    c.groups = groups;
    c.hq = hq;
    c.hkv = hkv;
    c.d = d;
    c.page_size = page_size;
    c.table_width = table_width;
    c.prefix_width = prefix_width;
    if (check_sizes("ctattn_shared_prefix_workspace_bytes", c) != 0) return -1;
    return rows > 0 && shared_mfma_supported(dtype, d, c.group()) ? shared_workspace_most(c) : 0;
}

int ctattn_shared_prefix_fwd(int dtype, const void *q, const void *k_cache, const void *v_cache, const int32_t *table,
                             const int32_t *lens, const int32_t *prefix_table, const int32_t *prefix_lens,
                             const int32_t *group_starts, const int32_t *starts, void *o, void *lse, void *workspace,
                             int64_t workspace_bytes, const int64_t *strides, int64_t rows, int64_t requests,
                             int64_t groups, int64_t hq, int64_t hkv, int64_t d, int64_t pages, int64_t page_size,
                             int64_t table_width, int64_t prefix_width, int fill, void *stream) {
    const char *fn = "ctattn_shared_prefix_fwd";
    SharedCall c{dtype, rows, requests, groups, hq, hkv, d, pages, page_size, table_width, prefix_width};
    if (int rc = check_sizes(fn, c)) return rc;
    if (!strides) return fail(hipErrorInvalidValue, "%s: null strides", fn);
    if (rows == 0) return ok();
    if (!q || !o || (requests > 0 && (!lens || (!table && table_width > 0))) ||
        (groups > 0 && (!prefix_lens || (!prefix_table && prefix_width > 0))) ||
        (pages > 0 && (!k_cache || !v_cache)))
        return fail(hipErrorInvalidValue, "%s: null pointer", fn);
    if (!starts && rows != requests)
        return fail(hipErrorInvalidValue, "%s: %lld rows of %lld requests, and no starts", fn, (long long)rows, (long long)requests);
    if (groups > 0 && !group_starts && requests % groups != 0)
        return fail(hipErrorInvalidValue, "%s: %lld requests in %lld equal groups", fn, (long long)requests, (long long)groups);
    // A cache without pages has no keys.
    if (pages == 0) c.table_width = c.prefix_width = 0;
    // row and head of q and o, page, token and head of each cache, rows of the two tables
    const int64_t extent[12] = {rows, hq, rows, hq, pages, page_size, hkv, pages, page_size, hkv, requests, groups};
    int64_t s[12], b[12];
    if (int rc = check_strides(fn, strides, extent, 12, s)) return rc;
    const int64_t es = elem_bytes(dtype);
    for (int i = 0; i < 12; ++i) b[i] = s[i] * (i < 10 ? es : 4);
    c.sq = {s[0], s[1]};
    c.so = {s[2], s[3]};
    c.sk = {s[4], s[5], s[6]};
    c.sv = {s[7], s[8], s[9]};
    c.table_row = s[10];
    c.prefix_row = s[11];
    if (!separate(c.so, rows, hq, d)) return fail(hipErrorInvalidValue, "%s: o's rows or heads overlap", fn);
    c.q = q;
    c.k = k_cache;
    c.v = v_cache;
    c.o = o;
    c.lse = lse;
    c.table = table;
    c.lens = lens;
    c.prefix_table = prefix_table;
    c.prefix_lens = prefix_lens;
    c.group_starts = group_starts;
    c.starts = starts;
    c.fill = fill != 0;
    const int64_t run = d * es, per = c.group();
    int64_t all = reinterpret_cast<intptr_t>(q) | reinterpret_cast<intptr_t>(o) | reinterpret_cast<intptr_t>(k_cache) |
                  reinterpret_cast<intptr_t>(v_cache);
    for (int i = 0; i < 10; ++i) all |= b[i];
    const bool fast = ctattn_get_policy() != CTATTN_POLICY_GENERIC && shared_mfma_supported(dtype, d, per) && all % 16 == 0;
    const int64_t need = fast ? shared_workspace_bytes(c) : 0;
    const int64_t pr = groups > 0 ? groups : 0;
    const Bytes in[] = {span_of(q, b, extent, 2, run),
                        span_of(k_cache, b + 4, extent + 4, 3, pages > 0 ? run : 0),
                        span_of(v_cache, b + 7, extent + 7, 3, pages > 0 ? run : 0),
                        run_of(table, requests > 0 ? ((requests - 1) * s[10] + c.table_width) * 4 : 0),
                        run_of(prefix_table, pr > 0 ? ((pr - 1) * s[11] + c.prefix_width) * 4 : 0),
                        run_of(lens, requests * 4),
                        run_of(prefix_lens, pr * 4),
                        run_of(group_starts, group_starts ? (pr + 1) * 4 : 0),
                        run_of(starts, starts ? (requests + 1) * 4 : 0)};
    const Bytes out[] = {span_of(o, b + 2, extent + 2, 2, run), run_of(lse, lse ? rows * hq * (dtype == CTATTN_F64 ? 8 : 4) : 0),
                         run_of(workspace, need)};
    if (int rc = check_apart(fn, in, out)) return rc;
    if (need > 0 && (!workspace || workspace_bytes < need))
        return fail(hipErrorInvalidValue, "%s: workspace too small (%lld bytes, %lld needed)", fn, (long long)workspace_bytes,
                    (long long)need);
    if (need > 0 && reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
        return fail(hipErrorInvalidValue, "%s: workspace must be 16-byte aligned", fn);
    hipStream_t st = static_cast<hipStream_t>(stream);
    return finish(fn, fast ? launch_shared(c, workspace, st) : launch_shared_generic(c, st), st);
}

}  // extern "C"
