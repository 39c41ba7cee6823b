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
