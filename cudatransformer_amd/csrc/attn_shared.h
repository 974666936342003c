// Attention of requests that share a prompt, keys and values in a paged cache: the call and the launcher
// interface between the C-ABI layer (paged_capi.hip) and the kernels (attn_shared.hip,
// attn_shared_generic.hip).
//
// A cache is pages of page_size tokens.  Requests are in groups, one behind the other; a group's prompt lies in
// the pages of its row of prefix_table, a request's own tokens in those of its row of table.  All lengths,
// tables and offsets are device memory and are read by the kernels alone, so that a captured graph replays on
// other contents; grids come from the tensors' shapes.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ctattn {

struct SharedStride {
    int64_t row, head;  // of a [rows, heads, d] tensor, in elements
};
struct CacheStride {
    int64_t page, token, head;
};

struct SharedCall {
    int dtype;  // 0 fp32, 1 bf16, 2 fp16, 3 fp64
    int64_t rows, requests, groups, hq, hkv, d;
    int64_t pages, page_size, table_width, prefix_width;
    const void *q, *k, *v;
    void *o, *lse;
    const int32_t *table, *lens, *prefix_table, *prefix_lens, *group_starts, *starts;
    int64_t table_row, prefix_row;
    SharedStride sq, so;
    CacheStride sk, sv;
    bool fill;  // rows of no request: zeros (lse -inf) instead of left as they are
    int64_t group() const { return hq / hkv; }
    int64_t max_own() const { return table_width * page_size; }
    int64_t max_prefix() const { return groups > 0 ? prefix_width * page_size : 0; }
};

// What the kernels read of a call to find out whose row is whose.  Every number that comes from device memory is
// brought into range where it is read: a wrong length or table makes a wrong result, not a wrong access.
struct SharedLayout {
    const int32_t *table, *lens, *prefix_table, *prefix_lens, *group_starts, *starts;
    int64_t table_row, prefix_row;
    int rows, requests, groups, hkv, group;
    int max_own, max_prefix;
    int shift, pages;

    static __device__ __forceinline__ int within(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }
    // First row of request i (0 .. requests).
    __device__ __forceinline__ int first_row(int i) const { return starts != nullptr ? within(starts[i], 0, rows) : i; }
    // First request of group g (0 .. groups), and its first row.
    __device__ __forceinline__ int first_request(int g) const {
        if (group_starts != nullptr) return within(group_starts[g], 0, requests);
        return int(int64_t(requests) * g / groups);
    }
    __device__ __forceinline__ int group_row(int g) const { return first_row(first_request(g)); }
    __device__ __forceinline__ int own_len(int i) const { return within(lens[i], 0, max_own); }
    __device__ __forceinline__ int prefix_len(int g) const { return within(prefix_lens[g], 0, max_prefix); }
    // A page outside the cache is read as page 0.
    __device__ __forceinline__ int page_at(const int32_t *pages_of, int key) const {
        const int p = pages_of[key >> shift];
        return uint32_t(p) < uint32_t(pages) ? p : 0;
    }
};
inline SharedLayout layout_of(const SharedCall &c) {
    int shift = 0;
    while ((int64_t(1) << shift) < c.page_size) ++shift;
    return {c.table,         c.lens,          c.prefix_table,      c.prefix_lens,      c.group_starts, c.starts,
            c.table_row,     c.prefix_row,    int(c.rows),         int(c.requests),    int(c.groups),  int(c.hkv),
            int(c.group()),  int(c.max_own()), int(c.max_prefix()), shift,             int(c.pages)};
}

// Any 1 <= d <= 256, any type, strides and alignment; no workspace.
hipError_t launch_shared_generic(const SharedCall &c, hipStream_t stream);

// MFMA kernels: fp32, bf16, fp16; d whole 16-byte chunks up to 128, at most 128 query heads to a key head;
// pointers and strides of q, o and the caches on 16 bytes.
bool shared_mfma_supported(int dtype, int64_t d, int64_t group);
// What a call needs, and the most that any call of these sizes does, with or without starts and group_starts.
int64_t shared_workspace_bytes(const SharedCall &c);
int64_t shared_workspace_most(const SharedCall &c);
hipError_t launch_shared(const SharedCall &c, void *workspace, hipStream_t stream);

}  // namespace ctattn
