// Distillation from a teacher's top logits: loss and gradient of a row in one pass over it.
//
// The row is read from HBM once and the gradient written once: a cluster of blocks holds the row in shared memory, each
// block a slice of it.  While a slice comes in, each thread keeps the softmax statistics of what it loads; the slices'
// statistics are exchanged through distributed shared memory, and the gradient is formed from the copy on chip.
#include <cooperative_groups.h>

#include <utility>

#include "zn_token.cuh"

namespace {

namespace cg = cooperative_groups;
constexpr int TPB = 256;
constexpr int MAX_SHARE = 8;

struct Shared {
    zn_softmax part[TPB / 32];
    zn_softmax slice[MAX_SHARE];                 // statistics of every slice of the row, in their order
    float q[ZN_TEACHER_MAX], x[ZN_TEACHER_MAX];  // the teacher's probability and the student's logit of an entry
    int32_t id[ZN_TEACHER_MAX];                  // its token, -1 for no entry
    float loss_q, ubad;
    int wrong, some;
};

// The teacher's entries of a row, by one warp: q = softmax(u / T) over them.
__device__ void read_teacher(Shared &s, const zn_distill_args &a, int64_t r, const float *x, int lane, bool report, int *status) {
    const float inv_t = 1.f / a.temperature;
    float um = -INFINITY;
    bool wrong = false, ubad = false;
    for (int j = lane; j < a.k; j += 32) {
        const int32_t t = a.ids[r * a.k + j];
        const float u = a.teacher[r * a.k + j];
        const bool entry = t >= 0 && u != -INFINITY;
        wrong = wrong || (entry && t >= a.vocab);
        ubad = ubad || (entry && !(u < INFINITY));
        const bool fine = entry && t < a.vocab;
        s.id[j] = fine ? t : -1;
        s.x[j] = fine ? x[t] : 0.f;
        s.q[j] = u;
        if (entry) um = fmaxf(um, u);
    }
    um = zn_warp_max(um);
    wrong = __any_sync(0xffffffffu, wrong);
    ubad = __any_sync(0xffffffffu, ubad);
    if (wrong && report && lane == 0) zn_bad_token(status);
    const float c = 1.4426950408889634f * inv_t;
    float mass = 0.f;
    for (int j = lane; j < a.k; j += 32)
        if (s.id[j] >= 0) mass += zn_exp2((s.q[j] - um) * c);
    mass = zn_warp_sum(mass);
    const float inv_mass = 1.f / mass, log_mass = logf(mass);
    float lq = 0.f;                              // sum q log q
    for (int j = lane; j < a.k; j += 32) {
        const float d = s.q[j] - um, q = s.id[j] >= 0 ? zn_exp2(d * c) * inv_mass : 0.f;
        if (q > 0.f) lq += q * (d * inv_t - log_mass);
        s.q[j] = q;
    }
    lq = zn_warp_sum(lq);
    if (lane == 0) {
        s.loss_q = lq;
        s.ubad = ubad ? 1.f : 0.f;
        s.wrong = wrong;
        s.some = um > -INFINITY || ubad;
    }
}

// Stores n values from i = 0 on: four at a time by vec(i) from `from` on where g and the copy on chip stand alike on 16
// bytes, one at a time by one(i) elsewhere (neighbouring lanes take neighbouring values: whole lines, no bank conflicts).
template <typename V, typename F>
__device__ __forceinline__ void store_slice(float *g, int64_t n, int64_t from, V vec, F one) {
    int64_t lo = 0;
    if (((reinterpret_cast<uintptr_t>(g + from)) & 15) == 0) {
        const int64_t vecs = (n - from) / 4;
#pragma unroll 4
        for (int64_t i = threadIdx.x; i < vecs; i += TPB) __stcs(reinterpret_cast<float4 *>(g + from + 4 * i), vec(from + 4 * i));
        if (threadIdx.x < from) g[threadIdx.x] = one(threadIdx.x);
        lo = from + 4 * vecs;
    }
#pragma unroll 4
    for (int64_t i = lo + threadIdx.x; i < n; i += TPB) __stcs(g + i, one(i));
}

__global__ void __launch_bounds__(TPB) distill_kernel(zn_distill_args a, int share, int64_t slice, int64_t keep, int *status) {
    extern __shared__ __align__(16) float kept[];          // the first `keep` values of the slice, shifted to the row's alignment
    __shared__ Shared s;
    cg::cluster_group cluster = cg::this_cluster();
    // before another block's shared memory is written it has to have started: the wait is far below
    auto started = cluster.barrier_arrive();
    const int64_t r = blockIdx.x / share;
    const int rank = (int)(blockIdx.x % share);
    const int64_t lo = min((int64_t)rank * slice, a.vocab), n = min(a.vocab, lo + slice) - lo;
    const float *row = a.logits + r * a.ld, *x = row + lo;
    const float w = a.weights ? a.weights[r] : 1.f, inv_t = 1.f / a.temperature, c = 1.4426950408889634f * inv_t, nan = zn_nan();
    if (threadIdx.x < 32) read_teacher(s, a, r, row, threadIdx.x, rank == 0, status);
    // the slice, and its statistics on the way
    const int64_t from = zn_aligned_from(x, n), vecs = (n - from) / 4, to = from + 4 * vecs;
    const int64_t shift = (4 - from) & 3;
    zn_softmax st{-INFINITY, 0.f, 0.f};
    if (w != 0.f) {
        for (int64_t i0 = 0; i0 < vecs; i0 += 4 * TPB) {
            float v[16];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t i = i0 + j * TPB + threadIdx.x;
                float4 f = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                if (i < vecs) f = *reinterpret_cast<const float4 *>(x + from + 4 * i);
                v[4 * j] = f.x; v[4 * j + 1] = f.y; v[4 * j + 2] = f.z; v[4 * j + 3] = f.w;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t at = from + 4 * (i0 + j * TPB + threadIdx.x);
                if (at + 4 <= keep && at < to)
                    *reinterpret_cast<float4 *>(kept + shift + at) = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
            }
            zn_softmax_add<16, false>(st, v, c);
        }
        float v[1] = {-INFINITY};
        int64_t end = -1;
        if (threadIdx.x < from) end = threadIdx.x;
        else if (threadIdx.x >= 32 && threadIdx.x - 32 < n - to) end = to + threadIdx.x - 32;
        if (end >= 0) {
            v[0] = x[end];
            if (end < keep) kept[shift + end] = v[0];
        }
        zn_softmax_add<1, false>(st, v, c);
    }
    st = zn_softmax_block<TPB>(st, c, s.part);
    cluster.barrier_wait(std::move(started));
    if (share > 1) {
        if (threadIdx.x < share) cluster.map_shared_rank(s.slice, threadIdx.x)[rank] = st;
        cluster.sync();                          // also: nobody still reads logits that another block may now overwrite
        st = s.slice[0];
        for (int i = 1; i < share; ++i) zn_softmax_join(st, s.slice[i], c);
    } else {
        __syncthreads();
    }
    const bool bad = !(st.s >= 0.f) || s.ubad != 0.f, empty = st.m == -INFINITY;
    const bool none = w == 0.f || s.wrong != 0 || !s.some;
    const float ls = logf(st.s), inv_s = 1.f / st.s, wt = w * a.temperature;
    if (a.loss && rank == 0 && threadIdx.x < 32) {
        // sum q (log q - log p) = sum q log q - sum q log p
        float lp = 0.f;
        for (int j = threadIdx.x; j < a.k; j += 32)
            if (s.q[j] > 0.f) lp += s.q[j] * (empty ? -INFINITY : (s.x[j] - st.m) * inv_t - ls);
        lp = zn_warp_sum(lp);
        if (threadIdx.x == 0) a.loss[r] = none ? (w != 0.f && s.wrong ? nan : 0.f) : bad ? nan : wt * a.temperature * (s.loss_q - lp);
    }
    if (!a.grad) return;
    float *g = a.grad + r * a.ld_grad + lo;
    if (none || bad || empty) {
        const float fill = none ? 0.f : bad ? nan : 0.f;
        store_slice(g, n, from, [&](int64_t) { return make_float4(fill, fill, fill, fill); }, [&](int64_t) { return fill; });
    } else {
        const float f = wt * inv_s;
        const float *mine = kept + shift;
        const auto p = [&](float v) { return f * zn_exp2((v - st.m) * c); };
        const auto p4 = [&](const float *at) {
            const float4 v = *reinterpret_cast<const float4 *>(at);
            return make_float4(p(v.x), p(v.y), p(v.z), p(v.w));
        };
        const int64_t on_chip = n <= keep ? n : from + (keep - from) / 4 * 4;
        if (n <= keep)
            store_slice(g, n, from, [&](int64_t i) { return p4(mine + i); }, [&](int64_t i) { return p(mine[i]); });
        else
            store_slice(g, n, from, [&](int64_t i) { return p4(i < on_chip ? mine + i : x + i); },
                        [&](int64_t i) { return p(i < on_chip ? mine[i] : x[i]); });
    }
    if (none || bad) return;
    __syncthreads();
    // the listed tokens of this slice: the first place of an id takes the q of all its places
    for (int j = threadIdx.x; j < a.k; j += TPB) {
        const int32_t id = s.id[j];
        if (id < lo || id >= lo + n) continue;
        float sum = 0.f;
        bool first = true;
        for (int i = 0; i < a.k; ++i)
            if (s.id[i] == id) {
                if (i < j) first = false;
                sum += s.q[i];
            }
        if (first) g[id - lo] = wt * ((empty ? 0.f : zn_exp2((s.x[j] - st.m) * c) * inv_s) - sum);
    }
}

// Blocks per row and values of a slice kept on chip.  Three blocks share an SM while a slice has at most KEEP_3 values, so
// that one loads while another stores; a vocabulary above 8 slices of that size gets larger ones, and what no longer fits
// is read a second time.  Fewer rows than SMs are spread over more blocks, down to 2048 values each.
constexpr int64_t KEEP_3 = 16640, KEEP_1 = 55000;
struct Plan {
    int share;
    int64_t slice, keep;
};
Plan distill_plan(int64_t rows, int64_t vocab, int sms) {
    int share = 1;
    while (share < MAX_SHARE && (vocab > share * KEEP_3 || (rows * share < 2 * sms && vocab > share * 2048))) share *= 2;
    const int64_t slice = ((vocab + share - 1) / share + 3) / 4 * 4;
    const int64_t keep = slice <= KEEP_1 ? slice : KEEP_1;
    return {share, slice, keep};
}

}   // namespace

zn_token_plan zn_plan_distill(size_t rows, size_t vocab, size_t k, int sms) {
    (void)k;
    const Plan d = distill_plan((int64_t)rows, (int64_t)vocab, sms);
    zn_token_plan p;
    p.threads = TPB;
    p.share = d.share;
    p.blocks = (int64_t)rows * d.share;
    p.smem = (size_t)(d.keep + 4) * sizeof(float);
    return p;
}

zn_status zn_k_distill(zn_ctx *ctx, const zn_distill_args &a) {
    const Plan d = distill_plan(a.rows, a.vocab, ctx->sm_count);
    const zn_token_plan p = zn_plan_distill((size_t)a.rows, (size_t)a.vocab, (size_t)a.k, ctx->sm_count);
    ZN_CUDA(ctx, cudaFuncSetAttribute(distill_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)((KEEP_1 + 4) * sizeof(float))));
    zn_launch_scope scope(ctx, ZN_PROF_LOSS, 6.0 * a.rows * a.vocab, (a.grad ? 8.0 : 4.0) * a.rows * a.vocab);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)p.blocks);
    cfg.blockDim = dim3(p.threads);
    cfg.dynamicSmemBytes = p.smem;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)d.share;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    ZN_CUDA(ctx, cudaLaunchKernelEx(&cfg, distill_kernel, a, d.share, d.slice, d.keep, ctx->status_dev));
    return ZN_OK;
}
