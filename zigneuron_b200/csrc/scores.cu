// Scores of given tokens under softmax(x / T): log-probability, entropy, the largest alternatives, and the gradient of
// the first two.
#include "zn_token.cuh"

namespace {

constexpr int TPB = 256;

// A logit and its column as one number that orders by value, then by lowest column: larger is better.  0 is "none".
__device__ __forceinline__ unsigned long long rank_key(float x, int64_t c) {
    if (x == 0.f) x = 0.f;                                    // -0 and 0 are equal
    const uint32_t b = __float_as_uint(x);
    const uint32_t u = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return x == -INFINITY ? 0ull : ((unsigned long long)u << 32) | (uint32_t)(0xffffffffu - (uint32_t)c);
}

// The k largest keys seen by a block.  Keys above the bar go into a list; when it is nearly full it is sorted and
// cut to k, and the bar rises to the k-th.  The result does not depend on the order in which keys arrive: keys are
// distinct.  `count` and `bar` are read by all threads between barriers only.
constexpr int LIST = 1024;
struct TopList {
    unsigned long long key[LIST];
    unsigned long long bar;            // only keys above it can still be among the k largest
    int count;
};

// Sorts the first n keys, largest first (bitonic network over the next power of two, filled up with zeros).
__device__ void sort_list(TopList &t, int n) {
    int size = 32;
    while (size < n) size *= 2;
    for (int i = n + threadIdx.x; i < size; i += TPB) t.key[i] = 0;
    for (int run = 2; run <= size; run *= 2)
        for (int half = run / 2; half > 0; half /= 2) {
            __syncthreads();
            for (int i = threadIdx.x; i < size / 2; i += TPB) {
                const int lo = 2 * half * (i / half) + i % half, hi = lo + half;
                const unsigned long long a = t.key[lo], b = t.key[hi];
                if ((a < b) == ((lo & run) == 0)) { t.key[lo] = b; t.key[hi] = a; }
            }
        }
    __syncthreads();
}

// Cuts the list to its k largest keys, sorted.
__device__ void cut_list(TopList &t, int k) {
    const int n = t.count;
    sort_list(t, n);
    if (threadIdx.x == 0) {
        t.count = n < k ? n : k;
        if (n >= k) t.bar = t.key[k - 1];
    }
    __syncthreads();
}

// Offers one tile of keys, N per thread (0 = none).  Usually all that reach the bar fit behind the list; where they do not
// (a sorted row, say), the tile is taken back and offered again in steps that always fit.
template <int N>
__device__ void offer(TopList &t, const unsigned long long (&key)[N], int k) {
    const int before = t.count;
    const unsigned long long bar = t.bar;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (key[i] > bar) {
            const int at = atomicAdd(&t.count, 1);
            if (at < LIST) t.key[at] = key[i];
        }
    __syncthreads();
    if (t.count <= LIST) {
        if (t.count > LIST / 2) cut_list(t, k);
        return;
    }
    __syncthreads();
    if (threadIdx.x == 0) t.count = before;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (t.count > LIST - TPB) cut_list(t, k);
        const unsigned long long now = t.bar;
        __syncthreads();
        if (key[i] > now) t.key[atomicAdd(&t.count, 1)] = key[i];
        __syncthreads();
    }
}

// One row, or one piece of it where rows alone would leave SMs idle (then the block that finishes a row last joins the
// pieces, in their order).  The row is read once: 16 values a thread at a time, as 16-byte loads from the first aligned
// one on; the statistics stay in registers and the few values that reach the bar go to the list.
constexpr int TILE = TPB * 16;
constexpr int MAX_PIECES = 64;

__global__ void __launch_bounds__(TPB, 4) scores_kernel(zn_scores_args a, int pieces, int64_t piece_len, float *scratch, unsigned int *arrivals,
                                                        int *status) {
    __shared__ zn_softmax part[TPB / 32];
    __shared__ TopList list;
    __shared__ zn_softmax piece_stats[MAX_PIECES];
    __shared__ bool last;
    const int64_t r = blockIdx.x / pieces;
    const int piece = (int)(blockIdx.x % pieces);
    const float *x = a.logits + r * a.ld;
    const int64_t lo = piece * piece_len, hi = min(a.vocab, lo + piece_len);
    const float c = 1.4426950408889634f / a.temperature;
    const int k = a.top_k;
    zn_softmax st{-INFINITY, 0.f, 0.f};
    if (threadIdx.x == 0) {
        list.count = 0;
        list.bar = 0;
    }
    __syncthreads();
    bool first = true;
    // the tile that holds the unaligned ends of the piece comes on top of the aligned ones
    const int64_t from = lo + zn_aligned_from(x + lo, hi - lo), vecs = (hi - from) / 4, to = from + 4 * vecs;
    const int64_t tiles = (vecs + TPB * 4 - 1) / (TPB * 4);
    for (int64_t t = 0; t <= tiles; ++t) {
        float v[16];
        int64_t at[4];
        if (t < tiles) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t i = (t * 4 + j) * TPB + threadIdx.x;
                at[j] = from + 4 * i;
                float4 f = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                if (i < vecs) f = __ldcs(reinterpret_cast<const float4 *>(x + at[j]));
                v[4 * j] = f.x; v[4 * j + 1] = f.y; v[4 * j + 2] = f.z; v[4 * j + 3] = f.w;
            }
        } else {
            if (from == lo && to == hi) break;
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = -INFINITY;
            const int64_t i = threadIdx.x < 4 ? lo + threadIdx.x : to + (threadIdx.x - 4);
            at[0] = i;
            at[1] = at[2] = at[3] = 0;
            if (threadIdx.x < 8 && (threadIdx.x < 4 ? i < from : i < hi)) v[0] = x[i];
        }
        zn_softmax_add<16, true>(st, v, c);
        if (k == 0) continue;
        unsigned long long bar = list.bar;
        if (first) {
            // the k-th largest of the threads' own largest is a bar that at least k values reach
            unsigned long long mine = 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const unsigned long long o = rank_key(v[i], at[i / 4] + i % 4);
                if (v[i] > -INFINITY && o > mine) mine = o;
            }
            list.key[threadIdx.x] = mine;
            __syncthreads();
            sort_list(list, TPB);
            if (threadIdx.x == 0 && list.key[k - 1] != 0) list.bar = list.key[k - 1] - 1;
            __syncthreads();
            bar = list.bar;
            first = false;
        }
        const uint32_t bar_value = (uint32_t)(bar >> 32);
        const float bar_x = bar == 0 ? -INFINITY : __uint_as_float((bar_value & 0x80000000u) ? bar_value & 0x7fffffffu : ~bar_value);
        unsigned long long key[16];
        bool any = false;
#pragma unroll
        for (int i = 0; i < 16; ++i) any = any || v[i] >= bar_x;
        if (__syncthreads_or(any)) {
#pragma unroll
            for (int i = 0; i < 16; ++i) key[i] = v[i] > -INFINITY ? rank_key(v[i], at[i / 4] + i % 4) : 0ull;
            offer(list, key, k);
        }
    }
    st = zn_softmax_block<TPB, true>(st, c, part, [] { __syncthreads(); });
    if (k > 0) cut_list(list, k);
    int kept = list.count;
    if (pieces > 1) {
        // a piece's record: m, s, w, count, then its keys
        const int64_t record = 4 + 2 * k;
        float *mine = scratch + (r * pieces + piece) * record;
        unsigned long long *keys = reinterpret_cast<unsigned long long *>(mine + 4);
        if (threadIdx.x == 0) {
            mine[0] = st.m; mine[1] = st.s; mine[2] = st.w; mine[3] = __int_as_float(kept);
        }
        for (int i = threadIdx.x; i < k; i += TPB) keys[i] = i < kept ? list.key[i] : 0ull;
        __threadfence();
        __syncthreads();
        if (threadIdx.x == 0) last = atomicAdd(&arrivals[r], 1u) == (unsigned)pieces - 1;
        __syncthreads();
        if (!last) return;
        __threadfence();
        if (threadIdx.x == 0) {
            arrivals[r] = 0u;
            list.count = 0;
            list.bar = 0;
        }
        __syncthreads();
        const int share = k > 0 ? (k + pieces - 1) / pieces - 1 : 0;
        if (threadIdx.x < pieces) {
            const float *rec = scratch + (r * pieces + threadIdx.x) * record;
            piece_stats[threadIdx.x] = {__ldcg(rec), __ldcg(rec + 1), __ldcg(rec + 2)};
            if (k > 0) list.key[threadIdx.x] = __ldcg(reinterpret_cast<const unsigned long long *>(rec + 4) + share);
        }
        __syncthreads();
        st = zn_softmax_join<true>(pieces, c, [&](int i) { return piece_stats[i]; });
        // every piece has share + 1 keys at or above the lowest of these, so k in all
        unsigned long long bar = list.key[0];
        for (int p = 1; p < pieces; ++p) bar = min(bar, list.key[p]);
        __syncthreads();
        if (k > 0) {
            if (threadIdx.x == 0 && bar != 0) list.bar = bar - 1;
            __syncthreads();
            for (int64_t i0 = 0; i0 < (int64_t)pieces * k; i0 += TPB * 4) {
                unsigned long long key[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int64_t i = i0 + j * TPB + threadIdx.x;
                    key[j] = i < (int64_t)pieces * k
                                 ? __ldcg(reinterpret_cast<const unsigned long long *>(scratch + (r * pieces + i / k) * record + 4) + i % k)
                                 : 0ull;
                }
                offer(list, key, k);
            }
            cut_list(list, k);
            kept = list.count;
        }
    }
    const float nan = zn_nan(), inv_t = 1.f / a.temperature, ls = logf(st.s);
    const bool bad = !(st.s >= 0.f), empty = !bad && st.m == -INFINITY;
    if (threadIdx.x == 0) {
        if (a.stats) {
            a.stats[2 * r] = bad ? nan : st.m;
            a.stats[2 * r + 1] = bad ? nan : empty ? -INFINITY : ls;
        }
        if (a.entropy) a.entropy[r] = bad ? nan : empty ? 0.f : ls - st.w * inv_t / st.s;
        if (a.logprob) {
            const int64_t t = a.tokens[r];
            float lp = 0.f;
            if (t >= a.vocab) { zn_bad_token(status); lp = nan; }
            else if (bad) lp = nan;
            else if (t >= 0) lp = empty ? -INFINITY : (x[t] - st.m) * inv_t - ls;
            a.logprob[r] = lp;
        }
    }
    for (int j = threadIdx.x; j < k; j += TPB) {
        const unsigned long long o = j < kept && !bad ? list.key[j] : 0ull;
        const int64_t col = (int64_t)(0xffffffffu - (uint32_t)o);
        a.top_tokens[r * k + j] = o ? (int32_t)col : -1;
        a.top_logprobs[r * k + j] = bad ? nan : o ? (x[col] - st.m) * inv_t - ls : -INFINITY;
    }
}

// Gradient: every value by itself, one read and one write of the block.  A block takes 4096 columns of a row, stores 16
// bytes at a time and loads as wide where both rows stand alike.
__global__ void __launch_bounds__(TPB) scores_grad_kernel(zn_scores_grad_args a, int pieces, int *status) {
    const int64_t r = blockIdx.x / pieces;
    const int64_t lo = (blockIdx.x % pieces) * (int64_t)TILE, hi = min(a.vocab, lo + TILE);
    const float *x = a.logits + r * a.ld;
    float *g = a.grad + r * a.ld_grad;
    int64_t t = a.grad_logprob ? a.tokens[r] : -1;
    if (t >= a.vocab) {
        if (threadIdx.x == 0 && lo == 0) zn_bad_token(status);
        t = -1;
    }
    const float c = 1.4426950408889634f / a.temperature, inv_t = 1.f / a.temperature;
    float gl = t >= 0 ? a.grad_logprob[r] : 0.f, gh = a.grad_entropy ? a.grad_entropy[r] : 0.f;
    const float h = a.entropy ? a.entropy[r] : 0.f, m = a.stats[2 * r], ls = a.stats[2 * r + 1];
    const bool none = (gl == 0.f && gh == 0.f) || m == -INFINITY;
    const float inv_s = expf(-ls);
    gl *= inv_t;
    gh *= inv_t;
    const auto value = [&](float v, int64_t col) {
        const float d = v - m, p = zn_exp2(d * c) * inv_s;
        // where p is zero its logarithm may be -inf: any finite number does there
        float f = gl;
        if (gh != 0.f) f = fmaf(gh, fmaxf(d * inv_t, -300.f) - ls + h, gl);
        return none ? 0.f : fmaf(-p, f, col == t ? gl : 0.f);
    };
    const int64_t from = lo + zn_aligned_from(g + lo, hi - lo), vecs = (hi - from) / 4, to = from + 4 * vecs;
    const bool alike = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(g)) & 15) == 0;
    float4 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int64_t i = j * TPB + threadIdx.x;
        if (i >= vecs || none) continue;
        const float *p = x + from + 4 * i;
        if (alike) v[j] = __ldcs(reinterpret_cast<const float4 *>(p));
        else v[j] = make_float4(p[0], p[1], p[2], p[3]);
    }
    float ends = 0.f;
    const int64_t end = threadIdx.x < 4 ? lo + threadIdx.x : to + (threadIdx.x - 4);
    const bool has_end = threadIdx.x < 8 && (threadIdx.x < 4 ? end < from : end < hi);
    if (has_end) ends = x[end];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int64_t i = j * TPB + threadIdx.x, col = from + 4 * i;
        if (i >= vecs) continue;
        float4 o;
        o.x = value(v[j].x, col);
        o.y = value(v[j].y, col + 1);
        o.z = value(v[j].z, col + 2);
        o.w = value(v[j].w, col + 3);
        __stcs(reinterpret_cast<float4 *>(g + col), o);
    }
    if (has_end) g[end] = value(ends, end);
}

}   // namespace

// Rows alone fill the GPU from two blocks per SM on; fewer are cut into pieces of whole tiles.
zn_token_plan zn_plan_token_logprobs(size_t rows, size_t vocab, size_t top_k, int sms) {
    zn_token_plan p;
    p.threads = TPB;
    const int64_t tiles = (int64_t)((vocab + TILE - 1) / TILE);
    int64_t pieces = rows > 0 && (int64_t)rows < 2 * sms ? (2 * sms + (int64_t)rows - 1) / (int64_t)rows : 1;
    if (pieces > tiles) pieces = tiles;
    if (pieces > MAX_PIECES) pieces = MAX_PIECES;
    const int64_t per = (tiles + pieces - 1) / pieces;
    pieces = (tiles + per - 1) / per;
    p.share = (int)pieces;
    p.blocks = (int64_t)rows * pieces;
    if (pieces > 1) p.scratch_floats = (size_t)p.blocks * (4 + 2 * top_k);
    return p;
}

zn_status zn_k_token_logprobs(zn_ctx *ctx, const zn_scores_args &a) {
    const zn_token_plan p = zn_plan_token_logprobs((size_t)a.rows, (size_t)a.vocab, (size_t)a.top_k, ctx->sm_count);
    const int64_t tiles = (a.vocab + TILE - 1) / TILE;
    unsigned int *arrivals = nullptr;
    if (p.share > 1) {                 // at most 2 x SMs rows then: fewer than the lane's counters
        ZN_TRY(zn_scratch_reserve(ctx, p.scratch_floats));
        ZN_TRY(zn_lane_counters(ctx, &arrivals));
    }
    zn_launch_scope scope(ctx, ZN_PROF_LOSS, 5.0 * a.rows * a.vocab, 4.0 * a.rows * a.vocab);
    scores_kernel<<<(unsigned)p.blocks, p.threads, 0, ctx->stream>>>(a, p.share, (tiles + p.share - 1) / p.share * TILE, ctx->scratch, arrivals,
                                                                     ctx->status_dev);
    ZN_CUDA(ctx, cudaGetLastError());
    return ZN_OK;
}

zn_token_plan zn_plan_token_logprobs_backward(size_t rows, size_t vocab, int sms) {
    zn_token_plan p;
    (void)sms;
    p.threads = TPB;
    p.share = (int)((vocab + TILE - 1) / TILE);
    p.blocks = (int64_t)rows * p.share;
    return p;
}

zn_status zn_k_token_logprobs_backward(zn_ctx *ctx, const zn_scores_grad_args &a) {
    const zn_token_plan p = zn_plan_token_logprobs_backward((size_t)a.rows, (size_t)a.vocab, ctx->sm_count);
    zn_launch_scope scope(ctx, ZN_PROF_LOSS, 7.0 * a.rows * a.vocab, 8.0 * a.rows * a.vocab);
    scores_grad_kernel<<<(unsigned)p.blocks, p.threads, 0, ctx->stream>>>(a, p.share, ctx->status_dev);
    ZN_CUDA(ctx, cudaGetLastError());
    return ZN_OK;
}
