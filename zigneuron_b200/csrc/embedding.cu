// Embedding lookup with scaling and its gradient.
#include "zn_token.cuh"

namespace {

constexpr int TPB = 256;

__global__ void embed_kernel(const float *__restrict__ table, const int32_t *__restrict__ tokens, float *__restrict__ out,
                             int64_t rows, int64_t vocab, int64_t dim, float scale, int *status) {
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const int64_t t = tokens[r];
        if (t >= vocab && threadIdx.x == 0) zn_bad_token(status);
        for (int64_t c = threadIdx.x; c < dim; c += TPB) out[r * dim + c] = (t >= 0 && t < vocab) ? scale * table[t * dim + c] : 0.f;
    }
}

// Place of every position in the order by (token, position): the number of positions before it in that order.
// Positions without a token come last.
__global__ void rank_kernel(const int32_t *__restrict__ tokens, int64_t rows, int64_t vocab, int32_t *__restrict__ order, int *status) {
    const int64_t r = (int64_t)blockIdx.x * TPB + threadIdx.x;
    if (r >= rows) return;
    if (tokens[r] >= vocab) zn_bad_token(status);
    const uint32_t mine = tokens[r] >= vocab ? 0xffffffffu : (uint32_t)tokens[r];
    int64_t place = 0;
    for (int64_t i = 0; i < rows; ++i) {
        const uint32_t other = tokens[i] >= vocab ? 0xffffffffu : (uint32_t)tokens[i];
        const bool both_none = mine >= 0x80000000u && other >= 0x80000000u;
        if (both_none ? i < r : (other < mine || (other == mine && i < r))) ++place;
    }
    order[place] = (int32_t)r;
}

// One block per place that starts a token's run: adds the run's rows in order of position.
__global__ void run_sum_kernel(const float *__restrict__ grad_out, const int32_t *__restrict__ tokens, const int32_t *__restrict__ order,
                               float *__restrict__ grad_table, int64_t rows, int64_t vocab, int64_t dim, float scale, int accumulate) {
    const int64_t i = blockIdx.x;
    const int64_t t = tokens[order[i]];
    if (t < 0 || t >= vocab || (i > 0 && tokens[order[i - 1]] == t)) return;
    for (int64_t c = threadIdx.x; c < dim; c += TPB) {
        float s = 0.f;
        for (int64_t j = i; j < rows && tokens[order[j]] == t; ++j) s += grad_out[(int64_t)order[j] * dim + c];
        float *g = grad_table + t * dim + c;
        *g = accumulate ? *g + scale * s : scale * s;
    }
}

}   // namespace

zn_token_plan zn_plan_embedding_forward(size_t rows, size_t dim, int sms) {
    zn_token_plan p;
    (void)dim;
    p.threads = TPB;
    p.blocks = (int64_t)rows < (int64_t)sms * 8 ? (int64_t)rows : (int64_t)sms * 8;
    return p;
}

zn_status zn_k_embedding_forward(zn_ctx *ctx, const float *table, const int32_t *tokens, float *out, size_t rows, size_t vocab,
                                 size_t dim, float scale) {
    const zn_token_plan p = zn_plan_embedding_forward(rows, dim, ctx->sm_count);
    zn_launch_scope scope(ctx, ZN_PROF_ELEMENTWISE, (double)rows * dim, 8.0 * rows * dim);
    embed_kernel<<<(unsigned)p.blocks, p.threads, 0, ctx->stream>>>(table, tokens, out, (int64_t)rows, (int64_t)vocab, (int64_t)dim, scale,
                                                                    ctx->status_dev);
    ZN_CUDA(ctx, cudaGetLastError());
    return ZN_OK;
}

zn_token_plan zn_plan_embedding_backward(size_t rows, size_t vocab, size_t dim, int sms) {
    zn_token_plan p;
    (void)vocab; (void)dim; (void)sms;
    p.threads = TPB;
    p.blocks = (int64_t)rows;
    p.scratch_floats = rows;
    return p;
}

zn_status zn_k_embedding_backward(zn_ctx *ctx, const float *grad_out, const int32_t *tokens, float *grad_table, size_t rows,
                                  size_t vocab, size_t dim, float scale, bool accumulate) {
    const zn_token_plan p = zn_plan_embedding_backward(rows, vocab, dim, ctx->sm_count);
    if (!accumulate) ZN_CUDA(ctx, cudaMemsetAsync(grad_table, 0, vocab * dim * sizeof(float), ctx->stream));
    if (rows == 0) return ZN_OK;
    ZN_TRY(zn_scratch_reserve(ctx, p.scratch_floats));
    int32_t *order = reinterpret_cast<int32_t *>(ctx->scratch);
    zn_launch_scope scope(ctx, ZN_PROF_ELEMENTWISE, 2.0 * rows * dim, 4.0 * rows * dim + 4.0 * vocab * dim, 2);
    rank_kernel<<<(unsigned)((rows + TPB - 1) / TPB), TPB, 0, ctx->stream>>>(tokens, (int64_t)rows, (int64_t)vocab, order, ctx->status_dev);
    run_sum_kernel<<<(unsigned)p.blocks, p.threads, 0, ctx->stream>>>(grad_out, tokens, order, grad_table, (int64_t)rows, (int64_t)vocab,
                                                                      (int64_t)dim, scale, accumulate ? 1 : 0);
    ZN_CUDA(ctx, cudaGetLastError());
    return ZN_OK;
}
