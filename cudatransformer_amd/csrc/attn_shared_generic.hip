// Attention of requests that share a prompt, generic kernel: any head dim 1 <= d <= 256, fp32, bf16, fp16 or fp64
// storage, any strides and alignment.  One wave per query row and head, which walks the prompt's keys and
// then the request's own up to the row's place, 64 at a time, with a running maximum and sum; scalar FMAs in the
// storage type's accumulation type.  Every row reads its prompt by itself.  It serves the calls that the MFMA
// kernels do not take and every call under the GENERIC policy, their cross-check, and is bound by its own
// instruction issue.
#include "attn_common.h"
#include "attn_launch.h"
#include "attn_shared.h"

#include <math.h>

namespace ctattn {
namespace {

constexpr int kMaxD = 256;
constexpr int kSlots = kMaxD / kWave;  // d elements per lane

template <typename T> struct Rows {
    T *p;
    int64_t row, head;
    __device__ T *at(int64_t n, int h) const { return p + n * row + h * head; }
};
template <typename T> struct Cache {
    const T *p;
    int64_t page, token, head;
    __device__ const T *at(int64_t pg, int64_t t, int h) const { return p + pg * page + t * token + h * head; }
};

template <typename T, typename A = acc_t<T>>
__global__ __launch_bounds__(kWave) void shared_generic_kernel(SharedLayout a, Rows<const T> q, Cache<T> k, Cache<T> v,
                                                              Rows<T> o, A *__restrict__ lse, int d, int fill) {
    __shared__ A qs[kMaxD];
    __shared__ A ps[kWave];
    __shared__ int64_t at[kWave];
    const int lane = threadIdx.x;
    const int hq = a.hkv * a.group;
    const A scale = A(1) / acc_sqrt(A(d));
    for (int64_t row = blockIdx.x; row < int64_t(a.rows) * hq; row += gridDim.x) {
        __syncthreads();  // the previous row's reads are done
        const int n = int(row / hq), h = int(row % hq), kvh = h / a.group;
        // The last request that begins at or before the row (empty ones begin with the next), and its group.
        int i = 0, g = 0;
        for (int hi = a.requests - 1; i < hi;) {
            const int mid = (i + hi + 1) / 2;
            if (a.first_row(mid) <= n) i = mid;
            else hi = mid - 1;
        }
        const int r0 = a.requests < 1 ? 0 : a.first_row(i), r1 = a.requests < 1 ? 0 : a.first_row(i + 1);
        if (a.requests < 1 || n < r0 || n >= r1) {
            if (fill) {
                for (int c = lane; c < d; c += kWave) o.at(n, h)[c] = from_acc<T>(A(0));
                if (lse != nullptr && lane == 0) lse[row] = -INFINITY;
            }
            continue;
        }
        for (int hi = a.groups - 1; g < hi;) {
            const int mid = (g + hi + 1) / 2;
            if (a.first_request(mid) <= i) g = mid;
            else hi = mid - 1;
        }
        const bool prompt = a.groups > 0 && i >= a.first_request(g) && i < a.first_request(g + 1);
        const int np = prompt ? a.prefix_len(g) : 0;
        const int len = a.own_len(i);
        const int own = a.within(len - (r1 - r0) + (n - r0) + 1, 0, len);
        for (int c = lane; c < d; c += kWave) qs[c] = to_acc(q.at(n, h)[c]);
        __syncthreads();
        A m = -INFINITY, l = 0;
        A acc[kSlots] = {0, 0, 0, 0};
        for (int part = 0; part < 2; ++part) {
            const int nkeys = part == 0 ? np : own;
            const int32_t *pages = part == 0 ? a.prefix_table + g * a.prefix_row : a.table + i * a.table_row;
            for (int j0 = 0; j0 < nkeys; j0 += kWave) {
                const int j = j0 + lane;
                A s = -INFINITY;
                if (j < nkeys) {
                    const int page = a.page_at(pages, j), token = j & ((1 << a.shift) - 1);
                    const T *kr = k.at(page, token, kvh);
                    A dot = 0;
                    for (int c = 0; c < d; ++c) dot += qs[c] * to_acc(kr[c]);
                    s = dot * scale;
                    at[lane] = v.at(page, token, kvh) - v.p;
                }
                const A mnew = fmax(m, wave_max(s));
                // A row that has met nothing but -inf has no maximum yet.
                const A base = mnew == -INFINITY ? A(0) : mnew;
                const A rescale = acc_exp(m - base);
                const A p = (j < nkeys) ? acc_exp(s - base) : A(0);
                l = l * rescale + wave_sum(p);
                ps[lane] = p;
                __syncthreads();
                const int cnt = nkeys - j0 < kWave ? nkeys - j0 : kWave;
#pragma unroll
                for (int r = 0; r < kSlots; ++r) {
                    const int c = lane + r * kWave;
                    if (c < d) {
                        A x = acc[r] * rescale;
                        for (int jj = 0; jj < cnt; ++jj) x += ps[jj] * to_acc(v.p[at[jj] + c]);
                        acc[r] = x;
                    }
                }
                __syncthreads();
                m = mnew;
            }
        }
        const A inv = l == A(0) ? A(0) : A(1) / l;  // no key, or none but -inf: zeros
#pragma unroll
        for (int r = 0; r < kSlots; ++r) {
            const int c = lane + r * kWave;
            if (c < d) o.at(n, h)[c] = from_acc<T>(l == A(0) ? A(0) : acc[r] * inv);
        }
        if (lse != nullptr && lane == 0) lse[row] = l == A(0) ? -INFINITY : m + acc_log(l);
    }
}

template <typename T> hipError_t run(const SharedCall &c, hipStream_t stream) {
    using A = acc_t<T>;
    const Rows<const T> q{static_cast<const T *>(c.q), c.sq.row, c.sq.head};
    const Rows<T> o{static_cast<T *>(c.o), c.so.row, c.so.head};
    const Cache<T> k{static_cast<const T *>(c.k), c.sk.page, c.sk.token, c.sk.head};
    const Cache<T> v{static_cast<const T *>(c.v), c.sv.page, c.sv.token, c.sv.head};
    shared_generic_kernel<T><<<stride_grid(c.rows * c.hq, kWave), kWave, 0, stream>>>(
        layout_of(c), q, k, v, o, static_cast<A *>(c.lse), int(c.d), c.fill ? 1 : 0);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_shared_generic(const SharedCall &c, hipStream_t stream) {
    switch (c.dtype) {
    case 0: return run<float>(c, stream);
    case 1: return run<bf16_t>(c, stream);
    case 2: return run<f16_t>(c, stream);
    default: return run<double>(c, stream);
    }
}

}  // namespace ctattn
