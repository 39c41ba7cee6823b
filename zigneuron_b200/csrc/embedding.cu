// Embedding lookup with scaling and its gradient.
//
// The gradient is a sum of rows per token.  The positions are sorted by token first (a stable radix sort, so that a
// token's rows are added in the order of their positions), then fixed pieces of the sorted order are summed, however the
// tokens are distributed: one token in every position costs the same as all different ones.  A token whose run crosses
// pieces leaves partial sums, which a last kernel adds in their order.  Nothing is added by atomics.
#include "zn_token.cuh"

namespace {

constexpr int TPB = 256;

template <bool VEC> struct Unit;
template <> struct Unit<true> {
    using type = float4;
    static __device__ __forceinline__ float4 zero() { return make_float4(0.f, 0.f, 0.f, 0.f); }
    static __device__ __forceinline__ float4 add(float4 a, float4 b) { return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w); }
    static __device__ __forceinline__ float4 mul(float s, float4 a) { return make_float4(s * a.x, s * a.y, s * a.z, s * a.w); }
};
template <> struct Unit<false> {
    using type = float;
    static __device__ __forceinline__ float zero() { return 0.f; }
    static __device__ __forceinline__ float add(float a, float b) { return a + b; }
    static __device__ __forceinline__ float mul(float s, float a) { return s * a; }
};

// A block takes `wide` units (16 bytes where rows allow it) of TPB / wide * ROWS rows; a thread has ROWS loads on their way.
template <bool VEC, int ROWS>
__global__ void __launch_bounds__(TPB) embed_kernel(const float *__restrict__ table, const int32_t *__restrict__ tokens, float *__restrict__ out,
                                                    int64_t rows, int64_t vocab, int64_t units, int wide, int cuts, float scale, int *status) {
    using U = Unit<VEC>;
    using T = typename U::type;
    const int64_t c = (int64_t)(blockIdx.x % cuts) * wide + threadIdx.x % wide;
    const int step = TPB / wide;
    const int64_t r0 = (int64_t)(blockIdx.x / cuts) * step * ROWS + threadIdx.x / wide;
    if (c >= units) return;
    const T *from = reinterpret_cast<const T *>(table);
    T *to = reinterpret_cast<T *>(out);
    int32_t id[ROWS];
    T v[ROWS];
#pragma unroll
    for (int j = 0; j < ROWS; ++j) id[j] = r0 + j * step < rows ? __ldg(tokens + r0 + j * step) : -1;
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
        v[j] = U::zero();
        if (id[j] >= 0 && id[j] < vocab) v[j] = U::mul(scale, __ldg(from + id[j] * units + c));
        else if (id[j] >= 0 && c == 0) zn_bad_token(status);
    }
#pragma unroll
    for (int j = 0; j < ROWS; ++j)
        if (r0 + j * step < rows) __stcs(to + (r0 + j * step) * units + c, v[j]);
}

// ---- sort ---------------------------------------------------------------------------------------------

constexpr int SORT_THREADS = 1024, SORT_WARPS = SORT_THREADS / 32, SORT_BLOCKS = 8, RADIX = 256;

struct SortArgs {
    const int32_t *tokens;
    int32_t *buffer;              // four times `rows`: keys and positions, twice
    float *table;                 // to be cleared by the blocks that do not sort; null: nothing to clear
    int64_t rows, vocab, clear;
    int passes, bits;
};

// One cluster of eight blocks sorts the positions by token, `bits` of it at a time, the lowest first; a position without a
// token counts as token `vocab` and comes last.  Every warp owns a stretch of the positions and keeps its own counts, so
// places follow from sums alone and equal tokens keep their order.  The other blocks of the launch clear the table
// meanwhile.  The sort is bound by latency (two cluster barriers a pass); it hides behind the clearing where there is one.
__global__ void __launch_bounds__(SORT_THREADS) sort_kernel(SortArgs a, int *status) {
    zn_pdl_release();
    if (blockIdx.x >= SORT_BLOCKS) {
        const int64_t blocks = gridDim.x - SORT_BLOCKS, from = zn_aligned_from(a.table, a.clear), vecs = (a.clear - from) / 4, to = from + 4 * vecs;
        const int64_t first = (int64_t)(blockIdx.x - SORT_BLOCKS) * SORT_THREADS + threadIdx.x;
        float4 *p = reinterpret_cast<float4 *>(a.table + from);
        for (int64_t i = first; i < vecs; i += blocks * SORT_THREADS) p[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (first < from) a.table[first] = 0.f;
        if (first < a.clear - to) a.table[to + first] = 0.f;
        return;
    }
    __shared__ int count[SORT_WARPS][RADIX];                 // first counts, then the places before a warp's first value of a digit
    __shared__ int total[SORT_BLOCKS][RADIX];
    __shared__ int base[RADIX], part[RADIX / 32];
    const int rank = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t stretch = ((a.rows + SORT_BLOCKS * SORT_WARPS - 1) / (SORT_BLOCKS * SORT_WARPS) + 31) / 32 * 32;
    const int64_t lo = min(a.rows, (rank * SORT_WARPS + warp) * stretch), hi = min(a.rows, lo + stretch);
    const int radix = 1 << a.bits;
    zn_cluster_arrive();                                     // all blocks have started
    zn_cluster_wait();
    for (int pass = 0; pass < a.passes; ++pass) {
        int32_t *src = a.buffer + (pass & 1 ? 0 : 2) * a.rows, *dst = a.buffer + (pass & 1 ? 2 : 0) * a.rows;
        const auto load = [&](int64_t i, uint32_t &key, int32_t &at) {
            if (pass == 0) {
                const int32_t t = __ldg(a.tokens + i);
                key = t < 0 || t >= a.vocab ? (uint32_t)a.vocab : (uint32_t)t;
                at = (int32_t)i;
            } else {
                key = (uint32_t)__ldcg(src + i);
                at = __ldcg(src + a.rows + i);
            }
        };
        for (int i = threadIdx.x; i < SORT_WARPS * RADIX; i += SORT_THREADS) (&count[0][0])[i] = 0;
        __syncthreads();
        for (int64_t i = lo + lane; i - lane < hi; i += 32) {
            const unsigned live = __ballot_sync(0xffffffffu, i < hi);
            if (i < hi) {
                uint32_t key;
                int32_t at;
                load(i, key, at);
                if (pass == 0 && __ldg(a.tokens + i) >= a.vocab) zn_bad_token(status);
                const int digit = (key >> (pass * a.bits)) & (radix - 1);
                const unsigned same = __match_any_sync(live, digit);
                if (lane == __ffs(same) - 1) count[warp][digit] += __popc(same);
            }
            __syncwarp();
        }
        __syncthreads();
        if (threadIdx.x < radix) {
            int sum = 0;
#pragma unroll 8
            for (int w = 0; w < SORT_WARPS; ++w) {
                const int n = count[w][threadIdx.x];
                count[w][threadIdx.x] = sum;
                sum += n;
            }
            for (int b = 0; b < SORT_BLOCKS; ++b) {
                uint32_t remote;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(zn_smem(&total[rank][threadIdx.x])), "r"(b));
                asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(remote), "r"(sum) : "memory");
            }
        }
        __syncwarp();
        zn_cluster_arrive();
        zn_cluster_wait();
        int before = 0, sum = 0, incl = 0;
        if (threadIdx.x < RADIX) {
            if (threadIdx.x < radix)
                for (int b = 0; b < SORT_BLOCKS; ++b) {
                    if (b == rank) before = sum;
                    sum += total[b][threadIdx.x];
                }
            incl = sum;
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const int n = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += n;
            }
            if (lane == 31) part[warp] = incl;
        }
        __syncthreads();
        if (threadIdx.x < radix) {
            for (int w = 0; w < warp; ++w) incl += part[w];
            base[threadIdx.x] = incl - sum + before;
        }
        __syncthreads();
        for (int64_t i = lo + lane; i - lane < hi; i += 32) {
            const unsigned live = __ballot_sync(0xffffffffu, i < hi);
            if (i < hi) {
                uint32_t key;
                int32_t at;
                load(i, key, at);
                const int digit = (key >> (pass * a.bits)) & (radix - 1);
                const unsigned same = __match_any_sync(live, digit);
                const int64_t place = (int64_t)base[digit] + count[warp][digit] + __popc(same & ((1u << lane) - 1u));
                __stcg(dst + place, (int32_t)key);
                __stcg(dst + a.rows + place, at);
                __syncwarp(live);
                if (lane == __ffs(same) - 1) count[warp][digit] += __popc(same);
            }
            __syncwarp();
        }
        zn_cluster_arrive();             // the next pass reads what all blocks wrote
        zn_cluster_wait();
    }
}

// ---- sums ---------------------------------------------------------------------------------------------

struct SumArgs {
    const float *grad;
    const int32_t *key, *at;      // sorted tokens and their positions
    float *table;
    float *head, *tail;           // per piece: the sum of a run that began before it, of one that goes on behind it
    int64_t rows, vocab, units;
    int piece;
    int64_t pieces;
    float scale;
    int accumulate;
};

template <bool VEC>
__device__ __forceinline__ void put_row(const SumArgs &a, int64_t token, int64_t c, typename Unit<VEC>::type sum) {
    using U = Unit<VEC>;
    auto *p = reinterpret_cast<typename U::type *>(a.table) + token * a.units + c;
    sum = U::mul(a.scale, sum);
    *p = a.accumulate ? U::add(*p, sum) : sum;
}

// A group of `wide` threads sums one piece of the sorted order, each thread one unit of the rows, eight rows on their way.
template <bool VEC>
__global__ void __launch_bounds__(TPB) run_sum_kernel(SumArgs a, int wide, int cuts) {
    using U = Unit<VEC>;
    using T = typename U::type;
    zn_pdl_release();
    zn_pdl_wait();
    const int64_t c = (int64_t)(blockIdx.x % cuts) * wide + threadIdx.x % wide;
    const int64_t piece = (int64_t)(blockIdx.x / cuts) * (TPB / wide) + threadIdx.x / wide;
    if (c >= a.units || piece >= a.pieces) return;
    const int64_t lo = piece * a.piece, hi = min(a.rows, lo + a.piece);
    const T *g = reinterpret_cast<const T *>(a.grad);
    bool continued = lo > 0 && __ldcg(a.key + lo - 1) == __ldcg(a.key + lo);
    int64_t token = __ldcg(a.key + lo);
    T sum = U::zero();
    for (int64_t i0 = lo; i0 < hi; i0 += 8) {
        int32_t key[8], at[8];
        T v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            key[j] = i0 + j < hi ? __ldcg(a.key + i0 + j) : (int32_t)a.vocab;
            at[j] = i0 + j < hi ? __ldcg(a.at + i0 + j) : 0;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = key[j] < a.vocab ? __ldcs(g + at[j] * a.units + c) : U::zero();
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (i0 + j >= hi) break;
            if (key[j] != token) {
                if (token < a.vocab) {
                    if (continued) reinterpret_cast<T *>(a.head)[piece * a.units + c] = sum;
                    else put_row<VEC>(a, token, c, sum);
                }
                continued = false;
                token = key[j];
                sum = U::zero();
            }
            sum = U::add(sum, v[j]);
        }
    }
    if (token >= a.vocab) return;
    if (continued) reinterpret_cast<T *>(a.head)[piece * a.units + c] = sum;
    else if (hi < a.rows && __ldcg(a.key + hi) == token) reinterpret_cast<T *>(a.tail)[piece * a.units + c] = sum;
    else put_row<VEC>(a, token, c, sum);
}

// One block per piece and cut.  Where a run begins in the piece and goes on behind it: its tail and the heads of the pieces
// that follow, added by groups of threads that take every so-many-th of them and then in the groups' order.
template <bool VEC>
__global__ void __launch_bounds__(TPB) run_join_kernel(SumArgs a, int wide, int cuts) {
    using U = Unit<VEC>;
    using T = typename U::type;
    __shared__ T sums[TPB];
    zn_pdl_wait();
    const int64_t piece = blockIdx.x / cuts, lo = piece * a.piece, hi = lo + a.piece;
    if (hi >= a.rows) return;
    const int32_t token = __ldcg(a.key + hi - 1);
    if (token >= a.vocab || __ldcg(a.key + hi) != token) return;
    if (lo > 0 && __ldcg(a.key + lo - 1) == token) return;              // began earlier
    int64_t heads = 0;                                                 // pieces that begin with the token
    for (;;) {
        const int64_t p = piece + 1 + heads + threadIdx.x;
        const int more = __syncthreads_count(p < a.pieces && __ldcg(a.key + p * a.piece) == token);
        heads += more;
        if (more < TPB) break;
    }
    const int64_t c = (int64_t)(blockIdx.x % cuts) * wide + threadIdx.x % wide;
    const int group = threadIdx.x / wide, groups = TPB / wide;
    T sum = U::zero();
    if (c < a.units) {
        const T *head = reinterpret_cast<const T *>(a.head) + (piece + 1) * a.units + c;
        int64_t i = group;
        for (; i + 7 * groups < heads; i += 8 * groups) {
            T v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = __ldcg(head + (i + j * groups) * a.units);
#pragma unroll
            for (int j = 0; j < 8; ++j) sum = U::add(sum, v[j]);
        }
        for (; i < heads; i += groups) sum = U::add(sum, __ldcg(head + i * a.units));
    }
    sums[threadIdx.x] = sum;
    __syncthreads();
    if (group == 0 && c < a.units) {
        T all = __ldcg(reinterpret_cast<const T *>(a.tail) + piece * a.units + c);
        for (int g = 0; g < groups; ++g) all = U::add(all, sums[g * wide + threadIdx.x]);
        put_row<VEC>(a, token, c, all);
    }
}

// Threads side by side on one row: the power of two that covers its units, `most` at most.
int width_of(int64_t units, int most) {
    int wide = 1;
    while (wide < most && wide < units) wide *= 2;
    return wide;
}
bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Rows of the sorted order per piece: as few as leave about a thousand threads per SM at work, eight at least.
int64_t piece_of(int64_t rows, int64_t units, int sms) {
    const int64_t piece = (rows * units / ((int64_t)sms * 1024) + 7) / 8 * 8;
    return piece < 8 ? 8 : piece;
}

}   // namespace

zn_token_plan zn_plan_embedding_forward(size_t rows, size_t dim, int sms) {
    zn_token_plan p;
    (void)sms;
    p.threads = TPB;
    const int64_t units = (int64_t)(dim % 4 == 0 ? dim / 4 : dim);
    const int wide = width_of(units, TPB);
    const int64_t cuts = (units + wide - 1) / wide, per = TPB / wide * (dim % 4 == 0 ? 4 : 8);
    p.share = (int)cuts;
    p.blocks = ((int64_t)rows + per - 1) / per * cuts;
    return p;
}

zn_status zn_k_embedding_forward(zn_ctx *ctx, const float *table, const int32_t *tokens, float *out, size_t rows, size_t vocab,
                                 size_t dim, float scale) {
    const bool vec = dim % 4 == 0 && aligned16(table) && aligned16(out);
    const int64_t units = (int64_t)(vec ? dim / 4 : dim);
    const int wide = width_of(units, TPB);
    const int64_t cuts = (units + wide - 1) / wide, per = TPB / wide * (vec ? 4 : 8), blocks = ((int64_t)rows + per - 1) / per * cuts;
    if (blocks > 0x7fffffff) return zn_fail(ctx, ZN_ERR_SHAPE, "embedding_forward: %zu x %zu values are too many for one launch", rows, dim);
    zn_launch_scope scope(ctx, ZN_PROF_ELEMENTWISE, (double)rows * dim, 8.0 * rows * dim);
    if (vec)
        embed_kernel<true, 4><<<(unsigned)blocks, TPB, 0, ctx->stream>>>(table, tokens, out, (int64_t)rows, (int64_t)vocab, units, wide, (int)cuts,
                                                                         scale, ctx->status_dev);
    else
        embed_kernel<false, 8><<<(unsigned)blocks, TPB, 0, ctx->stream>>>(table, tokens, out, (int64_t)rows, (int64_t)vocab, units, wide, (int)cuts,
                                                                          scale, ctx->status_dev);
    ZN_CUDA(ctx, cudaGetLastError());
    return ZN_OK;
}

zn_token_plan zn_plan_embedding_backward(size_t rows, size_t vocab, size_t dim, int sms) {
    zn_token_plan p;
    (void)vocab;
    p.threads = TPB;
    const int64_t units = (int64_t)(dim % 4 == 0 ? dim / 4 : dim);
    const int wide = width_of(units, TPB);
    const int64_t cuts = (units + wide - 1) / wide, piece = piece_of((int64_t)rows, units, sms), pieces = ((int64_t)rows + piece - 1) / piece;
    const int64_t per = TPB / wide;
    p.share = (int)cuts;
    p.blocks = (pieces + per - 1) / per * cuts;
    if (p.blocks < 1) p.blocks = 1;
    p.scratch_floats = 4 * ((rows + 3) / 4 * 4) + (size_t)(2 * pieces) * ((dim + 3) / 4 * 4);
    return p;
}

zn_status zn_k_embedding_backward(zn_ctx *ctx, const float *grad_out, const int32_t *tokens, float *grad_table, size_t rows,
                                  size_t vocab, size_t dim, float scale, bool accumulate) {
    if (rows == 0) {
        ZN_CUDA(ctx, cudaMemsetAsync(grad_table, 0, vocab * dim * sizeof(float), ctx->stream));
        return ZN_OK;
    }
    const zn_token_plan p = zn_plan_embedding_backward(rows, vocab, dim, ctx->sm_count);
    ZN_TRY(zn_scratch_reserve(ctx, p.scratch_floats));
    // the sort; two blocks to an SM, those that do not sort clear the table
    SortArgs s{tokens, reinterpret_cast<int32_t *>(ctx->scratch), grad_table, (int64_t)rows, (int64_t)vocab, (int64_t)(vocab * dim), 0, 0};
    int key_bits = 1;
    while (((int64_t)vocab >> key_bits) != 0) ++key_bits;
    s.passes = (key_bits + 7) / 8;
    s.bits = (key_bits + s.passes - 1) / s.passes;
    int64_t clear_blocks = 0;
    if (!accumulate) {
        clear_blocks = (s.clear / 4 + 4 * SORT_THREADS - 1) / (4 * SORT_THREADS);
        const int64_t most = (int64_t)(2 * ctx->sm_count - SORT_BLOCKS);
        clear_blocks = (clear_blocks < most ? clear_blocks + SORT_BLOCKS - 1 : most) / SORT_BLOCKS * SORT_BLOCKS;
        if (clear_blocks < SORT_BLOCKS) clear_blocks = SORT_BLOCKS;
    }
    // 16-byte units where every row allows them
    const bool vec = dim % 4 == 0 && aligned16(grad_out) && aligned16(grad_table);
    SumArgs a{};
    a.units = (int64_t)(vec ? dim / 4 : dim);
    a.piece = (int)piece_of((int64_t)rows, (int64_t)(dim % 4 == 0 ? dim / 4 : dim), ctx->sm_count);
    a.pieces = ((int64_t)rows + a.piece - 1) / a.piece;
    const int64_t row_pad = ((int64_t)rows + 3) / 4 * 4, dim_pad = ((int64_t)dim + 3) / 4 * 4;
    int32_t *sorted = s.buffer + ((s.passes - 1) & 1 ? 2 : 0) * (int64_t)rows;
    a.grad = grad_out; a.key = sorted; a.at = sorted + rows; a.table = grad_table;
    a.head = ctx->scratch + 4 * row_pad; a.tail = a.head + a.pieces * dim_pad;
    a.rows = (int64_t)rows; a.vocab = (int64_t)vocab; a.scale = scale; a.accumulate = accumulate ? 1 : 0;
    const int wide = width_of(a.units, TPB), join_wide = width_of(a.units, 64);
    const int64_t cuts = (a.units + wide - 1) / wide, join_cuts = (a.units + join_wide - 1) / join_wide;
    const int64_t sum_blocks = (a.pieces + TPB / wide - 1) / (TPB / wide) * cuts, join_blocks = a.pieces * join_cuts;
    if (sum_blocks > 0x7fffffff || join_blocks > 0x7fffffff)
        return zn_fail(ctx, ZN_ERR_SHAPE, "embedding_backward: %zu x %zu values are too many for one launch", rows, dim);
    zn_launch_scope scope(ctx, ZN_PROF_ELEMENTWISE, 2.0 * rows * dim, 4.0 * rows * dim + 4.0 * (accumulate ? 2 * rows : vocab) * dim, 3);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(SORT_BLOCKS + clear_blocks));
    cfg.blockDim = dim3(SORT_THREADS);
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = SORT_BLOCKS;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    ZN_CUDA(ctx, cudaLaunchKernelEx(&cfg, sort_kernel, s, ctx->status_dev));
    if (vec) {
        ZN_CUDA(ctx, zn_launch_pdl(run_sum_kernel<true>, dim3((unsigned)sum_blocks), dim3(TPB), 0, ctx->stream, a, wide, (int)cuts));
        ZN_CUDA(ctx, zn_launch_pdl(run_join_kernel<true>, dim3((unsigned)join_blocks), dim3(TPB), 0, ctx->stream, a, join_wide, (int)join_cuts));
    } else {
        ZN_CUDA(ctx, zn_launch_pdl(run_sum_kernel<false>, dim3((unsigned)sum_blocks), dim3(TPB), 0, ctx->stream, a, wide, (int)cuts));
        ZN_CUDA(ctx, zn_launch_pdl(run_join_kernel<false>, dim3((unsigned)join_blocks), dim3(TPB), 0, ctx->stream, a, join_wide, (int)join_cuts));
    }
    return ZN_OK;
}
