// Generic kernels of attention on packed sequences: any head dim 1 <= d <= 256, fp32, bf16, fp16 or
// fp64 storage, any strides and alignment.  One wave per query row (forward, dQ) or per key of a
// key head (dK, dV); scalar FMAs in the storage type's accumulation type.  They serve the calls
// that the MFMA kernels do not take (fp64, head dims off 16 bytes or above 128, tensors off 16
// bytes) and every call under the GENERIC policy, the cross-check of those kernels.  They are
// bound by their own instruction issue, far above the memory's floor.
//
// With P = exp(S / sqrt(d) - L), L the log of the row's sum: dV_j = sum P_ij dO_i,
// dS_ij = P_ij (dO_i V_j - delta_i), delta_i = dO_i O_i, dQ_i = sum_j dS_ij K_j / sqrt(d),
// dK_j = sum dS_ij Q_i / sqrt(d); dK and dV sum over the group's query heads as well, token by
// token and head by head in one order: no atomics.
#include "attn_common.h"
#include "attn_launch.h"
#include "attn_packed.h"

#include <math.h>

namespace ctattn {
namespace {

constexpr int kMaxD = 256;
constexpr int kSlots = kMaxD / kWave;  // d elements per lane

// The sequence that holds token n: the last one that starts at or before it (empty ones share
// their start with the next).
__device__ __forceinline__ int find_seq(const int32_t *cu, int nseq, int n) {
    int lo = 0, hi = nseq - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (cu[mid] <= n) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

template <typename T> struct Mat {
    T *p;
    int64_t row, head;
    __device__ T *at(int64_t n, int h) const { return p + n * row + h * head; }
};

template <typename T, typename A = acc_t<T>>
__global__ __launch_bounds__(kWave) void packed_generic_fwd_kernel(Mat<const T> q, Mat<const T> k, Mat<const T> v,
                                                                  Mat<T> o, A *__restrict__ lse,
                                                                  const int32_t *__restrict__ cu, int nseq,
                                                                  int64_t rows, int hq, int group, int d, int causal) {
    __shared__ A qs[kMaxD];
    __shared__ A ps[kWave];
    const int lane = threadIdx.x;
    const A scale = A(1) / acc_sqrt(A(d));
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        __syncthreads();  // the previous row's reads of qs / ps are done
        const int n = int(row / hq), h = int(row % hq), kvh = h / group;
        const int s0 = find_seq(cu, nseq, n);
        const int start = cu[s0], nkeys = causal ? n + 1 - start : cu[s0 + 1] - start;
        for (int c = lane; c < d; c += kWave) qs[c] = to_acc(q.at(n, h)[c]);
        __syncthreads();
        A m = -INFINITY, l = 0;
        A acc[kSlots] = {0, 0, 0, 0};
        for (int j0 = 0; j0 < nkeys; j0 += kWave) {
            const int j = j0 + lane;
            A s = -INFINITY;
            if (j < nkeys) {
                A dot = 0;
                const T *kr = k.at(int64_t(start) + j, kvh);
                for (int c = 0; c < d; ++c) dot += qs[c] * to_acc(kr[c]);
                s = dot * scale;
            }
            const A mnew = fmax(m, wave_max(s));
            const A rescale = (m == -INFINITY) ? A(0) : acc_exp(m - mnew);
            const A p = (j < nkeys) ? acc_exp(s - mnew) : A(0);
            l = l * rescale + wave_sum(p);
            ps[lane] = p;
            __syncthreads();
            const int cnt = nkeys - j0 < kWave ? nkeys - j0 : kWave;
#pragma unroll
            for (int r = 0; r < kSlots; ++r) {
                const int c = lane + r * kWave;
                if (c < d) {
                    A a = acc[r] * rescale;
                    for (int jj = 0; jj < cnt; ++jj) a += ps[jj] * to_acc(v.at(int64_t(start) + j0 + jj, kvh)[c]);
                    acc[r] = a;
                }
            }
            __syncthreads();
            m = mnew;
        }
#pragma unroll
        for (int r = 0; r < kSlots; ++r) {
            const int c = lane + r * kWave;
            if (c < d) o.at(n, h)[c] = from_acc<T>(acc[r] / l);
        }
        if (lse != nullptr && lane == 0) lse[row] = m + acc_log(l);
    }
}

// delta[n][h] = sum_c dO O, one wave a row.
template <typename T, typename A = acc_t<T>>
__global__ __launch_bounds__(kWave) void packed_generic_delta_kernel(Mat<const T> o, Mat<const T> dout,
                                                                    A *__restrict__ delta, int64_t rows, int hq,
                                                                    int d) {
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const int64_t n = row / hq;
        const int h = int(row % hq);
        A s = 0;
        for (int c = threadIdx.x; c < d; c += kWave) s += to_acc(o.at(n, h)[c]) * to_acc(dout.at(n, h)[c]);
        s = wave_sum(s);
        if (threadIdx.x == 0) delta[row] = s;
    }
}

template <typename T, typename A = acc_t<T>>
__global__ __launch_bounds__(kWave) void packed_generic_dq_kernel(Mat<const T> q, Mat<const T> k, Mat<const T> v,
                                                                 Mat<const T> dout, const A *__restrict__ lse,
                                                                 const A *__restrict__ delta, Mat<T> dq,
                                                                 const int32_t *__restrict__ cu, int nseq,
                                                                 int64_t rows, int hq, int group, int d, int causal) {
    __shared__ A qs[kMaxD];
    __shared__ A dos[kMaxD];
    __shared__ A dss[kWave];
    const int lane = threadIdx.x;
    const A scale = A(1) / acc_sqrt(A(d));
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        __syncthreads();
        const int n = int(row / hq), h = int(row % hq), kvh = h / group;
        const int s0 = find_seq(cu, nseq, n);
        const int start = cu[s0], nkeys = causal ? n + 1 - start : cu[s0 + 1] - start;
        for (int c = lane; c < d; c += kWave) {
            qs[c] = to_acc(q.at(n, h)[c]);
            dos[c] = to_acc(dout.at(n, h)[c]);
        }
        __syncthreads();
        const A L = lse[row], dl = delta[row];
        A acc[kSlots] = {0, 0, 0, 0};
        for (int j0 = 0; j0 < nkeys; j0 += kWave) {
            const int j = j0 + lane;
            A ds = 0;
            if (j < nkeys) {
                A dot = 0, dp = 0;
                const T *kr = k.at(int64_t(start) + j, kvh), *vr = v.at(int64_t(start) + j, kvh);
                for (int c = 0; c < d; ++c) {
                    dot += qs[c] * to_acc(kr[c]);
                    dp += dos[c] * to_acc(vr[c]);
                }
                ds = acc_exp(dot * scale - L) * (dp - dl);
            }
            dss[lane] = ds;
            __syncthreads();
            const int cnt = nkeys - j0 < kWave ? nkeys - j0 : kWave;
#pragma unroll
            for (int r = 0; r < kSlots; ++r) {
                const int c = lane + r * kWave;
                if (c < d)
                    for (int jj = 0; jj < cnt; ++jj)
                        acc[r] += dss[jj] * to_acc(k.at(int64_t(start) + j0 + jj, kvh)[c]);
            }
            __syncthreads();
        }
#pragma unroll
        for (int r = 0; r < kSlots; ++r) {
            const int c = lane + r * kWave;
            if (c < d) dq.at(n, h)[c] = from_acc<T>(acc[r] * scale);
        }
    }
}

// One wave per (key token, key head); lanes over the rows (token, head of the group).
template <typename T, typename A = acc_t<T>>
__global__ __launch_bounds__(kWave) void packed_generic_dkdv_kernel(Mat<const T> q, Mat<const T> k, Mat<const T> v,
                                                                   Mat<const T> dout, const A *__restrict__ lse,
                                                                   const A *__restrict__ delta, Mat<T> dk, Mat<T> dv,
                                                                   const int32_t *__restrict__ cu, int nseq,
                                                                   int64_t keys, int hkv, int group, int d,
                                                                   int causal) {
    __shared__ A ks[kMaxD];
    __shared__ A vs[kMaxD];
    __shared__ A ps[kWave];
    __shared__ A dss[kWave];
    const int lane = threadIdx.x;
    const int hq = hkv * group;
    const A scale = A(1) / acc_sqrt(A(d));
    for (int64_t row = blockIdx.x; row < keys; row += gridDim.x) {
        __syncthreads();
        const int n = int(row / hkv), kvh = int(row % hkv);
        const int s0 = find_seq(cu, nseq, n);
        const int first = causal ? n : cu[s0];
        const int64_t total = int64_t(cu[s0 + 1] - first) * group;
        for (int c = lane; c < d; c += kWave) {
            ks[c] = to_acc(k.at(n, kvh)[c]);
            vs[c] = to_acc(v.at(n, kvh)[c]);
        }
        __syncthreads();
        A ak[kSlots] = {0, 0, 0, 0}, av[kSlots] = {0, 0, 0, 0};
        for (int64_t r0 = 0; r0 < total; r0 += kWave) {
            const int64_t r = r0 + lane;
            A p = 0, ds = 0;
            if (r < total) {
                const int64_t t = first + r / group;
                const int h = kvh * group + int(r % group);
                const T *qr = q.at(t, h), *gr = dout.at(t, h);
                A dot = 0, dp = 0;
                for (int c = 0; c < d; ++c) {
                    dot += to_acc(qr[c]) * ks[c];
                    dp += to_acc(gr[c]) * vs[c];
                }
                p = acc_exp(dot * scale - lse[t * hq + h]);
                ds = p * (dp - delta[t * hq + h]);
            }
            ps[lane] = p;
            dss[lane] = ds;
            __syncthreads();
            const int cnt = int(total - r0 < kWave ? total - r0 : kWave);
            for (int rr = 0; rr < cnt; ++rr) {
                const int64_t t = first + (r0 + rr) / group;
                const int h = kvh * group + int((r0 + rr) % group);
                const T *qr = q.at(t, h), *gr = dout.at(t, h);
#pragma unroll
                for (int s = 0; s < kSlots; ++s) {
                    const int c = lane + s * kWave;
                    if (c < d) {
                        ak[s] += dss[rr] * to_acc(qr[c]);
                        av[s] += ps[rr] * to_acc(gr[c]);
                    }
                }
            }
            __syncthreads();
        }
#pragma unroll
        for (int s = 0; s < kSlots; ++s) {
            const int c = lane + s * kWave;
            if (c < d) {
                dk.at(n, kvh)[c] = from_acc<T>(ak[s] * scale);
                dv.at(n, kvh)[c] = from_acc<T>(av[s]);
            }
        }
    }
}

template <typename T> Mat<T> mat(void *p, const PackedStride &s) { return {static_cast<T *>(p), s.row, s.head}; }
template <typename T> Mat<const T> cmat(const void *p, const PackedStride &s) {
    return {static_cast<const T *>(p), s.row, s.head};
}
const int32_t *cu_of(const PackedCall &c) { return reinterpret_cast<const int32_t *>(c.dev + c.host->cu_offset); }

template <typename T>
hipError_t generic_fwd(const PackedCall &c, const void *q, const void *k, const void *v, void *o, void *lse,
                       hipStream_t stream) {
    const int64_t rows = c.tokens() * c.hq;
    hipLaunchKernelGGL(packed_generic_fwd_kernel<T>, dim3(stride_grid(rows, kWave)), dim3(kWave), 0, stream,
                       cmat<T>(q, c.sq), cmat<T>(k, c.sk), cmat<T>(v, c.sv), mat<T>(o, c.so),
                       static_cast<acc_t<T> *>(lse), cu_of(c), int(c.host->nseq), rows, int(c.hq), int(c.group()),
                       int(c.d), int(c.causal));
    return hipGetLastError();
}

template <typename T>
hipError_t generic_bwd(const PackedCall &c, const void *q, const void *k, const void *v, const void *o,
                       const void *dout, const void *lse, void *delta, void *dq, void *dk, void *dv,
                       hipStream_t stream) {
    using A = acc_t<T>;
    const int64_t rows = c.tokens() * c.hq, keys = c.tokens() * c.hkv;
    hipLaunchKernelGGL(packed_generic_delta_kernel<T>, dim3(stride_grid(rows, kWave)), dim3(kWave), 0, stream,
                       cmat<T>(o, c.so), cmat<T>(dout, c.sdo), static_cast<A *>(delta), rows, int(c.hq), int(c.d));
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(packed_generic_dq_kernel<T>, dim3(stride_grid(rows, kWave)), dim3(kWave), 0, stream,
                       cmat<T>(q, c.sq), cmat<T>(k, c.sk), cmat<T>(v, c.sv), cmat<T>(dout, c.sdo),
                       static_cast<const A *>(lse), static_cast<const A *>(delta), mat<T>(dq, c.sdq), cu_of(c),
                       int(c.host->nseq), rows, int(c.hq), int(c.group()), int(c.d), int(c.causal));
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(packed_generic_dkdv_kernel<T>, dim3(stride_grid(keys, kWave)), dim3(kWave), 0, stream,
                       cmat<T>(q, c.sq), cmat<T>(k, c.sk), cmat<T>(v, c.sv), cmat<T>(dout, c.sdo),
                       static_cast<const A *>(lse), static_cast<const A *>(delta), mat<T>(dk, c.sdk),
                       mat<T>(dv, c.sdv), cu_of(c), int(c.host->nseq), keys, int(c.hkv), int(c.group()), int(c.d),
                       int(c.causal));
    return hipGetLastError();
}

}  // namespace

hipError_t launch_packed_generic_fwd(const PackedCall &c, const void *q, const void *k, const void *v, void *o,
                                     void *lse, hipStream_t stream) {
    switch (c.dtype) {
        case 0: return generic_fwd<float>(c, q, k, v, o, lse, stream);
        case 1: return generic_fwd<bf16_t>(c, q, k, v, o, lse, stream);
        case 2: return generic_fwd<f16_t>(c, q, k, v, o, lse, stream);
        default: return generic_fwd<double>(c, q, k, v, o, lse, stream);
    }
}

hipError_t launch_packed_generic_bwd(const PackedCall &c, const void *q, const void *k, const void *v, const void *o,
                                     const void *dout, const void *lse, void *delta, void *dq, void *dk, void *dv,
                                     hipStream_t stream) {
    switch (c.dtype) {
        case 0: return generic_bwd<float>(c, q, k, v, o, dout, lse, delta, dq, dk, dv, stream);
        case 1: return generic_bwd<bf16_t>(c, q, k, v, o, dout, lse, delta, dq, dk, dv, stream);
        case 2: return generic_bwd<f16_t>(c, q, k, v, o, dout, lse, delta, dq, dk, dv, stream);
        default: return generic_bwd<double>(c, q, k, v, o, dout, lse, delta, dq, dk, dv, stream);
    }
}

}  // namespace ctattn
