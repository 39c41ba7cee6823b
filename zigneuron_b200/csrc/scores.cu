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

__global__ void scores_kernel(zn_scores_args a, int *status) {
    __shared__ float part[TPB / 32];
    __shared__ unsigned long long best[TPB / 32];
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const float *x = a.logits + r * a.ld;
        float mx = -INFINITY, bad = 0.f;
        for (int64_t c = threadIdx.x; c < a.vocab; c += TPB) {
            const float v = x[c];
            if (!(v < INFINITY)) bad = 1.f;
            mx = fmaxf(mx, v);
        }
        mx = zn_block_max<TPB>(mx, part);
        bad = zn_block_max<TPB>(bad, part);
        const bool empty = mx == -INFINITY && bad == 0.f;
        float s = 0.f, sz = 0.f;
        for (int64_t c = threadIdx.x; c < a.vocab; c += TPB) {
            const float z = (x[c] - mx) / a.temperature, e = expf(z);
            s += e;
            if (e > 0.f) sz += e * z;
        }
        s = zn_block_sum<TPB>(s, part);
        sz = zn_block_sum<TPB>(sz, part);
        const float nan = __int_as_float(0x7fffffff), ls = logf(s);
        if (threadIdx.x == 0) {
            if (a.stats) {
                a.stats[2 * r] = bad ? nan : mx;
                a.stats[2 * r + 1] = bad ? nan : empty ? -INFINITY : ls;
            }
            if (a.entropy) a.entropy[r] = bad ? nan : empty ? 0.f : ls - sz / s;
            if (a.logprob) {
                const int64_t t = a.tokens[r];
                float lp = 0.f;
                if (t >= a.vocab) { zn_bad_token(status); lp = nan; }
                else if (bad) lp = nan;
                else if (t >= 0) lp = empty ? -INFINITY : (x[t] - mx) / a.temperature - ls;
                a.logprob[r] = lp;
            }
        }
        unsigned long long before = ~0ull;
        for (int j = 0; j < a.top_k; ++j) {
            unsigned long long k = 0;
            if (!bad)
                for (int64_t c = threadIdx.x; c < a.vocab; c += TPB) {
                    const unsigned long long o = rank_key(x[c], c);
                    if (o < before && o > k) k = o;
                }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const unsigned long long other = __shfl_xor_sync(0xffffffffu, k, o);
                if (other > k) k = other;
            }
            __syncthreads();
            if ((threadIdx.x & 31) == 0) best[threadIdx.x >> 5] = k;
            __syncthreads();
            for (int i = 0; i < TPB / 32; ++i)
                if (best[i] > k) k = best[i];
            before = k;
            if (threadIdx.x == 0) {
                const int64_t c = (int64_t)(0xffffffffu - (uint32_t)k);
                a.top_tokens[r * a.top_k + j] = k ? (int32_t)c : -1;
                a.top_logprobs[r * a.top_k + j] = bad ? nan : k ? (x[c] - mx) / a.temperature - ls : -INFINITY;
            }
        }
    }
}

__global__ void scores_grad_kernel(zn_scores_grad_args a, int *status) {
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const float *x = a.logits + r * a.ld;
        float *g = a.grad + r * a.ld_grad;
        int64_t t = a.grad_logprob ? a.tokens[r] : -1;
        if (t >= a.vocab) {
            if (threadIdx.x == 0) zn_bad_token(status);
            t = -1;
        }
        const float gl = t >= 0 ? a.grad_logprob[r] : 0.f, gh = a.grad_entropy ? a.grad_entropy[r] : 0.f;
        const float h = a.entropy ? a.entropy[r] : 0.f, mx = a.stats[2 * r], ls = a.stats[2 * r + 1];
        const bool none = (gl == 0.f && gh == 0.f) || mx == -INFINITY;
        for (int64_t c = threadIdx.x; c < a.vocab; c += TPB) {
            float v = 0.f;
            if (!none) {
                const float lp = (x[c] - mx) / a.temperature - ls, p = expf(lp);
                v = (c == t ? gl : 0.f) - p * gl;
                if (p > 0.f) v -= p * (lp + h) * gh;
                v = __fdiv_rn(v, a.temperature);
            }
            g[c] = v;
        }
    }
}

}   // namespace

zn_token_plan zn_plan_token_logprobs(size_t rows, size_t vocab, size_t top_k, int sms) {
    zn_token_plan p;
    (void)vocab; (void)top_k;
    p.threads = TPB;
    p.blocks = (int64_t)rows < (int64_t)sms * 8 ? (int64_t)rows : (int64_t)sms * 8;
    return p;
}

zn_status zn_k_token_logprobs(zn_ctx *ctx, const zn_scores_args &a) {
    const zn_token_plan p = zn_plan_token_logprobs((size_t)a.rows, (size_t)a.vocab, (size_t)a.top_k, ctx->sm_count);
    zn_launch_scope scope(ctx, ZN_PROF_LOSS, 5.0 * a.rows * a.vocab, 4.0 * a.rows * a.vocab);
    scores_kernel<<<(unsigned)p.blocks, p.threads, 0, ctx->stream>>>(a, ctx->status_dev);
    ZN_CUDA(ctx, cudaGetLastError());
    return ZN_OK;
}

zn_token_plan zn_plan_token_logprobs_backward(size_t rows, size_t vocab, int sms) {
    return zn_plan_token_logprobs(rows, vocab, 0, sms);
}

zn_status zn_k_token_logprobs_backward(zn_ctx *ctx, const zn_scores_grad_args &a) {
    const zn_token_plan p = zn_plan_token_logprobs_backward((size_t)a.rows, (size_t)a.vocab, ctx->sm_count);
    zn_launch_scope scope(ctx, ZN_PROF_LOSS, 7.0 * a.rows * a.vocab, 8.0 * a.rows * a.vocab);
    scores_grad_kernel<<<(unsigned)p.blocks, p.threads, 0, ctx->stream>>>(a, ctx->status_dev);
    ZN_CUDA(ctx, cudaGetLastError());
    return ZN_OK;
}
