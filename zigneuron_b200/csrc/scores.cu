// Scores of given tokens under softmax(x / T): log-probability, entropy, the largest alternatives, and the gradient of
// the first two.
#include "zn_token.cuh"

namespace {

constexpr int GRAD_TPB = 256;

// A logit and its column as one number that orders by value, then by lowest column: larger is better.  0 is "none".
__device__ __forceinline__ unsigned long long rank_key(float x, int64_t c) {
    if (x == 0.f) x = 0.f;                                    // -0 and 0 are equal
    const uint32_t b = __float_as_uint(x);
    const uint32_t u = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return x == -INFINITY ? 0ull : ((unsigned long long)u << 32) | (uint32_t)(0xffffffffu - (uint32_t)c);
}

// The logit of a key, which is not "none".
__device__ __forceinline__ float key_logit(unsigned long long key) {
    const uint32_t u = (uint32_t)(key >> 32);
    return __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u);
}

// The k largest keys seen by a block.  Keys above the bar go into a list; when it is half full it is sorted and cut to k,
// and the bar rises to the k-th.  The result does not depend on the order in which keys arrive: keys are distinct.
// `count` and `bar` are read by all threads between barriers only.
constexpr int LIST = 1024;
struct TopList {
    unsigned long long key[LIST];
    unsigned long long bar;            // only keys above it can still be among the k largest
    int count;
};

// Sorts the first n keys, largest first: a short list by counting, for each key, those above it; a long one by a bitonic
// network over the next power of two, filled up with zeros.
template <int TPB>
__device__ void sort_list(TopList &t, int n) {
    __syncthreads();
    if (n <= TPB) {
        const unsigned long long mine = threadIdx.x < n ? t.key[threadIdx.x] : 0ull;
        int place = 0;
        if (threadIdx.x < n) {
#pragma unroll 8
            for (int i = 0; i < n; ++i) place += t.key[i] > mine;
        }
        __syncthreads();
        if (threadIdx.x < n) t.key[place] = mine;
        __syncthreads();
        return;
    }
    int size = 2 * TPB;
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
template <int TPB>
__device__ void cut_list(TopList &t, int k) {
    const int n = t.count;
    sort_list<TPB>(t, n);
    if (threadIdx.x == 0) {
        t.count = n < k ? n : k;
        if (n >= k) t.bar = t.key[k - 1];
    }
    __syncthreads();
}

// Puts a key above the bar on the list, if it has room; the count goes on where it has not.
__device__ __forceinline__ void put_key(TopList &t, unsigned long long key, unsigned long long bar) {
    if (key <= bar) return;
    const int at = atomicAdd(&t.count, 1);
    if (at < LIST) t.key[at] = key;
}

// One step of the slow way, taken where a list has run over (a sorted row, say): at most one key a thread, and the list is
// cut whenever another step might not fit.
template <int TPB>
__device__ __forceinline__ void put_step(TopList &t, int k, unsigned long long key) {
    if (t.count > LIST - TPB) cut_list<TPB>(t, k);
    const unsigned long long bar = t.bar;
    __syncthreads();
    put_key(t, key, bar);
    __syncthreads();
}

// One row, or one piece of it where rows alone would leave SMs idle (then the block that finishes a row last joins the
// pieces, in their order).  The row is read once: 16 values a thread at a time, as 16-byte loads from the first aligned
// one on; the statistics stay in registers and the few values that reach the bar go to the list.  The list is looked after
// when the number of tiles has doubled, not tile by tile: about k values pass the bar in between, and barriers are what
// such a loop can least afford.
constexpr int MAX_PIECES = 64;

// Six blocks of 256 threads to an SM: rows at different places hide each other's barriers and loads better than a tile
// fetched ahead does (4096 rows of 50,001, five alternatives: 155 us; with the next tile in registers and four blocks 161).
template <int TPB>
__global__ void __launch_bounds__(TPB, 1536 / TPB) scores_kernel(zn_scores_args a, int pieces, int64_t piece_len, float *scratch, unsigned int *arrivals,
                                                        int *status) {
    __shared__ zn_softmax part[TPB / 32];
    __shared__ TopList list;
    __shared__ __align__(16) float largest[TPB];
    __shared__ zn_softmax piece_stats[MAX_PIECES];
    __shared__ bool last;
    const int64_t r = blockIdx.x / pieces;
    const int piece = (int)(blockIdx.x % pieces);
    const float *x = a.logits + r * a.ld;
    const int lo = (int)(piece * piece_len), hi = (int)min(a.vocab, lo + piece_len);
    const float c = 1.4426950408889634f / a.temperature;
    const int k = a.top_k;
    zn_softmax st{-INFINITY, 0.f, 0.f};
    int64_t token = -1;
    float given = 0.f;                   // the logit of the row's token, asked for early
    if (threadIdx.x == 0) {
        if (a.logprob) token = a.tokens[r];
        if (token >= 0 && token < a.vocab) given = x[token];
        list.count = 0;
        list.bar = 0;
    }
    __syncthreads();
    const int from = lo + (int)zn_aligned_from(x + lo, hi - lo), vecs = (hi - from) / 4, to = from + 4 * vecs;
    {
        // up to six values around the aligned part
        const int at = threadIdx.x < 4 ? lo + threadIdx.x : to + threadIdx.x - 4;
        const bool there = threadIdx.x < 8 && (threadIdx.x < 4 ? at < from : at < hi);
        const float v[1] = {there ? x[at] : -INFINITY};
        zn_softmax_add<1, true>(st, v, v[0], c);
        if (k > 0 && v[0] > -INFINITY) put_key(list, rank_key(v[0], at), 0ull);
    }
    unsigned long long bar = 0;
    float bar_x = -INFINITY;
    const auto read_bar = [&]() {
        bar = list.bar;
        bar_x = bar == 0 ? -INFINITY : key_logit(bar);
    };
    const float4 *p = reinterpret_cast<const float4 *>(x + from) + threadIdx.x;
    const float4 none = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    int held = 0, since = 0, check = 0;  // the list's length at the last look, the first tile after it, the end of the next
    for (int v0 = 0; v0 < vecs; v0 += TPB * 4) {
        float v[16];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float4 f = v0 + j * TPB + (int)threadIdx.x < vecs ? __ldcs(p + v0 + j * TPB) : none;
            v[4 * j] = f.x; v[4 * j + 1] = f.y; v[4 * j + 2] = f.z; v[4 * j + 3] = f.w;
        }
        const float top = zn_largest(v);
        zn_softmax_add<16, true>(st, v, top, c);
        if (k == 0) continue;
        const auto key_of = [&](const float (&v)[16], int v0, int i) {
            float u = v[0];
#pragma unroll
            for (int j = 1; j < 16; ++j) u = i == j ? v[j] : u;
            return u > -INFINITY ? rank_key(u, from + 4 * (v0 + (int)threadIdx.x) + i / 4 * (4 * TPB) + i % 4) : 0ull;
        };
        if (v0 == 0) {
            // A bar for the first tile: the k-th largest of the largest values of groups of threads, four to a group or (for
            // a large k) each by itself.  At least k values reach it, and few more do.
            const int width = k <= TPB / 8 ? 4 : 1, groups = TPB / width;
            float mine = top;
            for (int o = width / 2; o > 0; o /= 2) mine = fmaxf(mine, __shfl_xor_sync(0xffffffffu, mine, o));
            if (threadIdx.x % width == 0) largest[threadIdx.x / width] = mine;
            __syncthreads();
            held = list.count;                       // the values around the aligned part
            if (threadIdx.x < groups) {
                mine = largest[threadIdx.x];
                int above = 0, reach = 0;
                for (int i = 0; i < groups; i += 4) {
                    const float4 f = *reinterpret_cast<const float4 *>(largest + i);
                    above += (f.x > mine) + (f.y > mine) + (f.z > mine) + (f.w > mine);
                    reach += (f.x >= mine) + (f.y >= mine) + (f.z >= mine) + (f.w >= mine);
                }
                // equal ones write the same; below k values in all, nothing is barred
                if (above < k && k <= reach && mine > -INFINITY) list.bar = rank_key(mine, 0xffffffffll);
            }
            __syncthreads();
            read_bar();
        }
        const int col0 = from + 4 * (v0 + (int)threadIdx.x);
        if (v0 > 0) {
            if (top >= bar_x) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (v[i] >= bar_x && v[i] > -INFINITY) put_key(list, rank_key(v[i], col0 + i / 4 * (4 * TPB) + i % 4), bar);
            }
        } else {
            // most of the first tile's come at once: room for all of a warp's
            uint32_t reach = 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) reach |= v[i] >= bar_x && v[i] > -INFINITY ? 1u << i : 0u;
            int before = __popc(reach);
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const int n = __shfl_up_sync(0xffffffffu, before, o);
                if ((threadIdx.x & 31) >= o) before += n;
            }
            int at = 0;
            if ((threadIdx.x & 31) == 31) at = atomicAdd(&list.count, before);
            at = __shfl_sync(0xffffffffu, at, 31) + before - __popc(reach);
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (reach >> i & 1) {
                    if (at < LIST) list.key[at] = rank_key(v[i], col0 + i / 4 * (4 * TPB) + i % 4);
                    ++at;
                }
        }
        if (v0 + TPB * 4 < check && v0 + TPB * 4 < vecs) continue;
        __syncthreads();
        if (list.count > LIST) {
            // not all had room: the tiles since the last look once more, the slow way
            __syncthreads();
            if (threadIdx.x == 0) list.count = held;
            __syncthreads();
#pragma unroll 1
            for (int u0 = since; u0 <= v0; u0 += TPB * 4) {
                float u[16];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float4 f = u0 + j * TPB + (int)threadIdx.x < vecs ? p[u0 + j * TPB] : none;
                    u[4 * j] = f.x; u[4 * j + 1] = f.y; u[4 * j + 2] = f.z; u[4 * j + 3] = f.w;
                }
#pragma unroll 1
                for (int i = 0; i < 16; ++i) put_step<TPB>(list, k, key_of(u, u0, i));
            }
        }
        cut_list<TPB>(list, k);
        read_bar();
        held = list.count;
        __syncthreads();
        since = v0 + TPB * 4;
        check = 2 * since;
    }
    st = zn_softmax_block<TPB, true>(st, c, part, [] { __syncthreads(); });
    if (k > 0 && vecs <= 0) cut_list<TPB>(list, k);
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
        bar = list.key[0];
        for (int i = 1; i < pieces; ++i) bar = min(bar, list.key[i]);
        __syncthreads();
        if (k > 0) {
            if (threadIdx.x == 0 && bar != 0) list.bar = bar - 1;
            __syncthreads();
            const auto key_at = [&](int i) {
                return i < pieces * k ? __ldcg(reinterpret_cast<const unsigned long long *>(scratch + (r * pieces + i / k) * record + 4) + i % k) : 0ull;
            };
            bar = list.bar;
            for (int i0 = threadIdx.x; i0 < pieces * k; i0 += 4 * TPB) {
                unsigned long long key[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) key[j] = key_at(i0 + j * TPB);
#pragma unroll
                for (int j = 0; j < 4; ++j) put_key(list, key[j], bar);
            }
            __syncthreads();
            if (list.count > LIST) {
                __syncthreads();
                if (threadIdx.x == 0) list.count = 0;
                __syncthreads();
                for (int i = threadIdx.x; i - (int)threadIdx.x < pieces * k; i += TPB) put_step<TPB>(list, k, key_at(i));
            }
            cut_list<TPB>(list, k);
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
        if (a.entropy) a.entropy[r] = bad ? nan : empty ? 0.f : ls - st.w * 0.6931471805599453f / st.s;
        if (a.logprob) {
            float lp = 0.f;
            if (token >= a.vocab) { zn_bad_token(status); lp = nan; }
            else if (bad) lp = nan;
            else if (token >= 0) lp = empty ? -INFINITY : (given - st.m) * inv_t - ls;
            a.logprob[r] = lp;
        }
    }
    for (int j = threadIdx.x; j < k; j += TPB) {
        const unsigned long long o = j < kept && !bad ? list.key[j] : 0ull;
        const int64_t col = (int64_t)(0xffffffffu - (uint32_t)o);
        a.top_tokens[r * k + j] = o ? (int32_t)col : -1;
        a.top_logprobs[r * k + j] = bad ? nan : o ? (key_logit(o) - st.m) * inv_t - ls : -INFINITY;
    }
}

// Gradient: every value by itself, one read and one write of the block, bound by HBM (2048 x 131,072: 350 us, 6.1 TB/s, 0.94
// of a copy).  A block takes 4096 columns of a row, stores 16 bytes at a time and loads as wide where both rows stand alike.
constexpr int GRAD_TILE = GRAD_TPB * 16;
__global__ void __launch_bounds__(GRAD_TPB) scores_grad_kernel(zn_scores_grad_args a, int pieces, int *status) {
    const int64_t r = blockIdx.x / pieces;
    const int64_t lo = (blockIdx.x % pieces) * (int64_t)GRAD_TILE, hi = min(a.vocab, lo + GRAD_TILE);
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
        const int64_t i = j * GRAD_TPB + threadIdx.x;
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
        const int64_t i = j * GRAD_TPB + threadIdx.x, col = from + 4 * i;
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

// Threads per row by the vocabulary: a short row is over before many threads have met, so more rows at once do better
// (8192 rows, ten alternatives, against 256 threads: vocabulary 1500 41 against 68 us, 6000 70 against 97).
// Rows alone fill the GPU from two blocks of 256 threads per SM on; fewer are cut into pieces of whole tiles.
zn_token_plan zn_plan_token_logprobs(size_t rows, size_t vocab, size_t top_k, int sms) {
    zn_token_plan p;
    p.threads = vocab <= 2048 ? 64 : vocab <= 8192 ? 128 : 256;
    const int64_t tile = p.threads * 16, tiles = ((int64_t)vocab + tile - 1) / tile;
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
    const int64_t tile = p.threads * 16, tiles = (a.vocab + tile - 1) / tile;
    unsigned int *arrivals = nullptr;
    if (p.share > 1) {                 // fewer than 2 x SMs rows then: fewer than the lane's counters
        ZN_TRY(zn_scratch_reserve(ctx, p.scratch_floats));
        ZN_TRY(zn_lane_counters(ctx, &arrivals));
    }
    zn_launch_scope scope(ctx, ZN_PROF_LOSS, 5.0 * a.rows * a.vocab, 4.0 * a.rows * a.vocab);
    const auto kernel = p.threads == 64 ? scores_kernel<64> : p.threads == 128 ? scores_kernel<128> : scores_kernel<256>;
    kernel<<<(unsigned)p.blocks, p.threads, 0, ctx->stream>>>(a, p.share, (tiles + p.share - 1) / p.share * tile, ctx->scratch, arrivals,
                                                              ctx->status_dev);
    ZN_CUDA(ctx, cudaGetLastError());
    return ZN_OK;
}

zn_token_plan zn_plan_token_logprobs_backward(size_t rows, size_t vocab, int sms) {
    zn_token_plan p;
    (void)sms;
    p.threads = GRAD_TPB;
    p.share = (int)((vocab + GRAD_TILE - 1) / GRAD_TILE);
    p.blocks = (int64_t)rows * p.share;
    return p;
}

zn_status zn_k_token_logprobs_backward(zn_ctx *ctx, const zn_scores_grad_args &a) {
    const zn_token_plan p = zn_plan_token_logprobs_backward((size_t)a.rows, (size_t)a.vocab, ctx->sm_count);
    if (p.blocks > 0x7fffffff) return zn_fail(ctx, ZN_ERR_SHAPE, "token_logprobs_backward: too many values for one launch");
    zn_launch_scope scope(ctx, ZN_PROF_LOSS, 7.0 * a.rows * a.vocab, 8.0 * a.rows * a.vocab);
    scores_grad_kernel<<<(unsigned)p.blocks, p.threads, 0, ctx->stream>>>(a, p.share, ctx->status_dev);
    ZN_CUDA(ctx, cudaGetLastError());
    return ZN_OK;
}
