// Device helpers shared by the token-model kernels.
#pragma once

#include "zn_internal.h"

__device__ __forceinline__ float zn_warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float zn_warp_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// Records a token id outside the vocabulary in the context's status word; the first code stays.
__device__ __forceinline__ void zn_bad_token(int *status) { atomicCAS_system(status, 0, (int)ZN_DEVICE_BAD_TOKEN); }

// Sums and maxima of a block of THREADS threads, valid in every thread.  `part` holds one value per warp.
template <int THREADS>
__device__ __forceinline__ float zn_block_sum(float v, float *part) {
    v = zn_warp_sum(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) s += part[i];
    return s;
}
template <int THREADS>
__device__ __forceinline__ float zn_block_max(float v, float *part) {
    v = zn_warp_max(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = part[0];
#pragma unroll
    for (int i = 1; i < THREADS / 32; ++i) s = fmaxf(s, part[i]);
    return s;
}

// 2^v, at most two steps off; results below 2^-126 become zero.
__device__ __forceinline__ float zn_exp2(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float zn_nan() { return __int_as_float(0x7fffffff); }

// Softmax statistics kept on the way over a row: with m the largest logit so far, s = sum 2^((x - m) c) and
// w = sum 2^((x - m) c) (x - m), where c = log2(e) / T.  The difference is formed before the scaling: a product x c could
// leave the range of float where x - m does not.  A column at -inf adds nothing to either; a NaN or +inf makes s NaN.
struct zn_softmax {
    float m, s, w;
};
// A difference so low that its term is zero, kept finite: zero times -inf would be NaN (and 2^31 of these still fit).
__device__ __forceinline__ float zn_above(float d) { return fmaxf(d, -1e28f); }
// N values at once, with one change of the maximum at most.
template <int N, bool ENTROPY>
__device__ __forceinline__ void zn_softmax_add(zn_softmax &a, const float (&x)[N], float c) {
    float top = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) top = fmaxf(top, x[i]);
    if (top > a.m) {
        if (a.m > -INFINITY) {
            const float d = a.m - top, f = zn_exp2(d * c);
            if (ENTROPY) a.w = f * (a.w + a.s * zn_above(d));
            a.s *= f;
        }
        a.m = top;
    }
    const float base = a.m == -INFINITY ? 0.f : a.m;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float d = x[i] - base, e = zn_exp2(d * c);
        a.s += e;
        if (ENTROPY) a.w = fmaf(e, zn_above(d), a.w);
    }
}
// b joined to a.
__device__ __forceinline__ void zn_softmax_join(zn_softmax &a, const zn_softmax &b, float c) {
    const float m = fmaxf(a.m, b.m);
    if (m == -INFINITY) {
        a.s += b.s;                                             // zero, or NaN from a NaN among columns at -inf
        return;
    }
    const float da = a.m - m, db = b.m - m, fa = zn_exp2(da * c), fb = zn_exp2(db * c);
    a.w = fa * (a.w + a.s * zn_above(da)) + fb * (b.w + b.s * zn_above(db));
    a.s = a.s * fa + b.s * fb;
    a.m = m;
}
__device__ __forceinline__ zn_softmax zn_softmax_shuffle(const zn_softmax &a, int o) {
    return {__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o), __shfl_xor_sync(0xffffffffu, a.w, o)};
}
// Over the block: the same result in every thread.  The lower lane or warp always stands first, so that all threads of a
// pair form the same bits.
template <int THREADS>
__device__ __forceinline__ zn_softmax zn_softmax_block(zn_softmax a, float c, zn_softmax *part) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const zn_softmax b = zn_softmax_shuffle(a, o);
        if (threadIdx.x & o) {
            zn_softmax t = b;
            zn_softmax_join(t, a, c);
            a = t;
        } else {
            zn_softmax_join(a, b, c);
        }
    }
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = a;
    __syncthreads();
    a = part[0];
#pragma unroll
    for (int i = 1; i < THREADS / 32; ++i) zn_softmax_join(a, part[i], c);
    return a;
}

// First index of [0, n) at which `p + index` stands on 16 bytes, n if there is none.
__device__ __forceinline__ int64_t zn_aligned_from(const float *p, int64_t n) {
    const int64_t lead = (int64_t)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / 4;
    return lead < n ? lead : n;
}
