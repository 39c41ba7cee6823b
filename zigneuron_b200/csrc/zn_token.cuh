// Device helpers shared by the token-model kernels.
#pragma once

#include "zn_internal.h"

__device__ __forceinline__ float zn_warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float zn_warp_max(float v) {       // NaN only where every lane has one
    float m;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
    return m;
}

// Records a token id outside the vocabulary in the context's status word; the first code stays.
__device__ __forceinline__ void zn_bad_token(int *status) { atomicCAS_system(status, 0, (int)ZN_DEVICE_BAD_TOKEN); }

// 2^v, at most two steps off; results below 2^-126 become zero.
__device__ __forceinline__ float zn_exp2(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float zn_nan() { return __int_as_float(0x7fffffff); }

// Softmax statistics kept on the way over a row: with m the largest logit so far, c = log2(e) / T and y = (x - m) c,
// s = sum 2^y and w = sum 2^y y.  The difference is formed before the scaling: a product x c could leave the range of float
// where x - m does not.  A column at -inf adds nothing to either; a NaN or +inf makes s NaN.
struct zn_softmax {
    float m, s, w;
};
// An exponent so low that its power is zero, kept finite (zero times -inf would be NaN); NaN stays NaN.
__device__ __forceinline__ float zn_exponent(float y) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(y), "f"(-200.f));
    return r;
}
// The statistics brought to a larger maximum m.
template <bool ENTROPY>
__device__ __forceinline__ void zn_softmax_raise(zn_softmax &a, float m, float c) {
    const float y = a.m == m ? 0.f : zn_exponent((a.m - m) * c), f = zn_exp2(y);       // both at -inf: no difference
    if (ENTROPY) a.w = f * (a.w + a.s * y);
    a.s *= f;
    a.m = m;
}
// N values at once, `top` the largest, with one change of the maximum at most.
template <int N>
__device__ __forceinline__ float zn_largest(const float (&x)[N]) {
    float top = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) top = fmaxf(top, x[i]);
    return top;
}
template <int N, bool ENTROPY>
__device__ __forceinline__ void zn_softmax_add(zn_softmax &a, const float (&x)[N], float top, float c) {
    if (top > a.m) zn_softmax_raise<ENTROPY>(a, top, c);
    const float base = a.m == -INFINITY ? 0.f : a.m;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float y = ENTROPY ? zn_exponent((x[i] - base) * c) : (x[i] - base) * c, e = zn_exp2(y);
        a.s += e;
        if (ENTROPY) a.w = fmaf(e, y, a.w);
    }
}
// Over the first THREADS threads of a block, all of which get the same result: first the maximum, then the sums, which
// takes one exponential per thread.  `sync` is a barrier among them; `part` holds one entry per warp.
template <int THREADS, bool ENTROPY, typename S>
__device__ __forceinline__ zn_softmax zn_softmax_block(zn_softmax a, float c, zn_softmax *part, S sync) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float m = zn_warp_max(a.m);
    if (THREADS > 32) {
        if (lane == 0) part[warp].m = m;
        sync();
        m = part[0].m;
#pragma unroll
        for (int i = 1; i < THREADS / 32; ++i) m = fmaxf(m, part[i].m);
    }
    zn_softmax_raise<ENTROPY>(a, m, c);
    a.s = zn_warp_sum(a.s);
    if (ENTROPY) a.w = zn_warp_sum(a.w);
    if (THREADS > 32) {
        if (lane == 0) {
            part[warp].s = a.s;
            if (ENTROPY) part[warp].w = a.w;
        }
        sync();
        a.s = part[0].s;
        if (ENTROPY) a.w = part[0].w;
#pragma unroll
        for (int i = 1; i < THREADS / 32; ++i) {
            a.s += part[i].s;
            if (ENTROPY) a.w += part[i].w;
        }
    }
    return a;
}
// Several statistics joined in their order.
template <bool ENTROPY, typename F>
__device__ __forceinline__ zn_softmax zn_softmax_join(int n, float c, F get) {
    float m = get(0).m;
    for (int i = 1; i < n; ++i) m = fmaxf(m, get(i).m);
    zn_softmax a{m, 0.f, 0.f};
    for (int i = 0; i < n; ++i) {
        zn_softmax b = get(i);
        zn_softmax_raise<ENTROPY>(b, m, c);
        a.s += b.s;
        if (ENTROPY) a.w += b.w;
    }
    return a;
}

// First index of [0, n) at which `p + index` stands on 16 bytes, n if there is none.
__device__ __forceinline__ int64_t zn_aligned_from(const float *p, int64_t n) {
    const int64_t lead = (int64_t)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / 4;
    return lead < n ? lead : n;
}

// ---- mbarriers and bulk copies ------------------------------------------------------------------

__device__ __forceinline__ uint32_t zn_smem(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void zn_bar_init(uint64_t *bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(zn_smem(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void zn_bar_init_done() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
__device__ __forceinline__ void zn_bar_arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(zn_smem(bar)) : "memory");
}
__device__ __forceinline__ void zn_bar_expect(uint64_t *bar, uint32_t bytes) {       // an arrival that also announces bytes
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(zn_smem(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool zn_bar_try(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t"
        "}"
        : "=r"(ok) : "r"(zn_smem(bar)), "r"(parity) : "memory");
    return ok != 0;
}
// Waits a second or so at most; then the code goes to the status word and the caller carries on, so that every block
// of a launch still takes the same steps to its end.
constexpr long long ZN_TOKEN_WAIT_CYCLES = 2000000000ll;
__device__ __forceinline__ void zn_bar_wait(uint64_t *bar, uint32_t parity, int *status, int code) {
    if (zn_bar_try(bar, parity)) return;
    const long long t0 = clock64();
    while (!zn_bar_try(bar, parity))
        if (clock64() - t0 > ZN_TOKEN_WAIT_CYCLES) {
            atomicCAS_system(status, 0, code);
            return;
        }
}
// Both ends on 16 bytes, size a multiple of 16.
__device__ __forceinline__ void zn_bulk_load(void *dst, const void *src, uint32_t bytes, uint64_t *bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(zn_smem(dst)), "l"(src), "r"(bytes), "r"(zn_smem(bar)) : "memory");
}
// Four bytes in the background, zero where there are none; this thread's arrival on `bar` once all it asked for is there.
__device__ __forceinline__ void zn_async_word(void *dst, const void *src, bool there) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(zn_smem(dst)), "l"(src), "r"(there ? 4 : 0) : "memory");
}
__device__ __forceinline__ void zn_async_words_arrive(uint64_t *bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(zn_smem(bar)) : "memory");
}
__device__ __forceinline__ void zn_cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void zn_cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// Two floats to the same place in block `rank` of the cluster; they count 8 bytes on that block's `bar`.
__device__ __forceinline__ void zn_cluster_send(float *p, float v0, float v1, uint64_t *bar, uint32_t rank) {
    uint32_t to, at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(zn_smem(p)), "r"(rank));
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(zn_smem(bar)), "r"(rank));
    asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];"
                 ::"r"(to), "f"(v0), "f"(v1), "r"(at) : "memory");
}
// Shared memory to global memory, both ends on 16 bytes, and the wait until shared memory has been read.  What other
// threads wrote there needs their zn_async_fence before this thread is told of it.
__device__ __forceinline__ void zn_bulk_store(void *dst, const void *src, uint32_t bytes) {
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(zn_smem(src)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void zn_bulk_store_read() {
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
}
__device__ __forceinline__ void zn_async_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// A barrier among the first `threads` threads of a block.
__device__ __forceinline__ void zn_part_sync(int threads) { asm volatile("bar.sync 1, %0;" ::"r"(threads) : "memory"); }
