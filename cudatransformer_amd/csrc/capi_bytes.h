// Which memory an entry point's tensors cover, for the checks that no output lies on another tensor.
#pragma once

#include "capi_util.h"

#include <algorithm>
#include <stdint.h>

namespace ctattn {
namespace capi {

// The bytes of a [rows, heads, d] tensor: `lo`, `hi` its first and last; within a row from `lo` on `span` of them
// every `row`, unless heads lie further apart than rows.
struct Bytes {
    intptr_t lo, hi, row, span;
};
// Whether two tensors may share a byte.  Slices of one row-major buffer (a projection's q, k and v) do not: their rows are
// equally far apart and each lies in its own part of a row.
inline bool may_overlap(const Bytes &a, const Bytes &b) {
    if (a.hi <= b.lo || b.hi <= a.lo || a.hi <= a.lo || b.hi <= b.lo) return false;
    if (a.row != b.row || a.row <= 0 || a.span <= 0 || b.span <= 0 || a.span > a.row || b.span > a.row) return true;
    const intptr_t shift = ((b.lo - a.lo) % a.row + a.row) % a.row;
    return !(a.span <= shift && shift + b.span <= a.row);
}
// `n` bytes from p on, whole.
inline Bytes run_of(const void *p, int64_t n) {
    const intptr_t at = reinterpret_cast<intptr_t>(p);
    return {at, at + n, 0, 0};
}
// A tensor of `dims` strided dimensions (strides in bytes, the outermost first) of runs of `run` bytes.
inline Bytes span_of(const void *p, const int64_t *strides, const int64_t *extent, int dims, int64_t run) {
    const intptr_t at = reinterpret_cast<intptr_t>(p);
    Bytes b{at, at + run, strides[0], run};
    for (int i = 0; i < dims; ++i) {
        const int64_t end = extent[i] > 1 ? (extent[i] - 1) * strides[i] : 0;
        (end < 0 ? b.lo : b.hi) += end;
        if (i > 0) b.span += end;
    }
    return b;
}

// Strides in elements into `out`; one that is never stepped along (an extent of one) may hold anything and becomes 0.
inline int check_strides(const char *fn, const int64_t *strides, const int64_t *extent, int n, int64_t *out) {
    for (int i = 0; i < n; ++i) {
        out[i] = extent[i] > 1 ? strides[i] : 0;
        if (out[i] < 0 || out[i] > (int64_t(1) << 48) / std::max<int64_t>(1, extent[i]))
            return fail(hipErrorInvalidValue, "%s: stride %lld", fn, (long long)strides[i]);
    }
    return 0;
}

// No output may share memory with an input or another output.
template <size_t N, size_t M> int check_apart(const char *fn, const Bytes (&in)[N], const Bytes (&out)[M]) {
    for (size_t i = 0; i < M; ++i) {
        for (const Bytes &b : in)
            if (may_overlap(out[i], b)) return fail(hipErrorInvalidValue, "%s: an output lies on an input's memory", fn);
        for (size_t j = 0; j < i; ++j)
            if (may_overlap(out[i], out[j])) return fail(hipErrorInvalidValue, "%s: two outputs share memory", fn);
    }
    return 0;
}

}  // namespace capi
}  // namespace ctattn
