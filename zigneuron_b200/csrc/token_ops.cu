// Entry points of the token-model operators: argument checks, staging of host operands, and the call of the launcher.
// The kernels are in embedding.cu (lookup and its gradient), scores.cu (token log-probabilities), distill.cu
// (distillation loss) and quant4.cu (4-bit weights).
#include "zn_internal.h"

namespace {

constexpr size_t MAX_DIM = 0x7fffffff;      // rows, vocabularies and widths are 32-bit; their products are not
constexpr size_t MAX_CELLS = (size_t)1 << 44;

zn_status check_sizes(zn_ctx *ctx, const char *op, size_t a, size_t b, size_t c) {
    if (a > MAX_DIM || b > MAX_DIM || c > MAX_DIM) return zn_fail(ctx, ZN_ERR_SHAPE, "%s: a dimension is above 2^31 - 1", op);
    if (a * b > MAX_CELLS || a * c > MAX_CELLS || b * c > MAX_CELLS) return zn_fail(ctx, ZN_ERR_SHAPE, "%s: a block of more than 2^44 values", op);
    return ZN_OK;
}

// Columns of a row of logits are counted in 32 bits, some of them past its end.
constexpr size_t MAX_PITCH = (size_t)1 << 30;
zn_status check_logits(zn_ctx *ctx, const char *op, size_t rows, size_t vocab, size_t ld) {
    if (vocab == 0) return zn_fail(ctx, ZN_ERR_SHAPE, "%s: empty vocabulary", op);
    if (ld < vocab) return zn_fail(ctx, ZN_ERR_SHAPE, "%s: the row pitch %zu is below the vocabulary %zu", op, ld, vocab);
    if (ld > MAX_PITCH) return zn_fail(ctx, ZN_ERR_SHAPE, "%s: rows more than 2^30 values apart", op);
    return check_sizes(ctx, op, rows, ld, 1);
}

zn_status check_group(zn_ctx *ctx, const char *op, size_t group) {
    if (group != 32 && group != 64 && group != 128)
        return zn_fail(ctx, ZN_ERR_INVALID_VALUE, "%s: groups of %zu weights (32, 64 or 128 are taken)", op, group);
    return ZN_OK;
}

zn_status check_temperature(zn_ctx *ctx, const char *op, float t) {
    if (!(t >= 1e-4f && t <= 1e4f)) return zn_fail(ctx, ZN_ERR_INVALID_VALUE, "%s: temperature %g outside 1e-4..1e4", op, t);
    return ZN_OK;
}

// One call's operands: `rows` rows of `width` values, `pitch` values apart; every value is four bytes wide.
struct Call {
    enum Kind { IN, OUT, INOUT };
    struct Arg { const void *p; size_t rows, width, pitch; Kind kind; size_t align; void *dev; };

    zn_ctx *ctx;
    const char *op;
    Arg args[ZN_STAGE_SLOTS];
    int count = 0;
    int in_place_a = -1, in_place_b = -1;       // this pair may be one block

    Call(zn_ctx *c, const char *name) : ctx(c), op(name) {}
    int add(const void *p, size_t rows, size_t width, size_t pitch, Kind kind, size_t align = 4) {
        args[count] = {p, rows, width, pitch, kind, align, nullptr};
        return count++;
    }
    template <typename T> T *dev(int i) const { return i < 0 ? nullptr : static_cast<T *>(args[i].dev); }
    static size_t extent(const Arg &a) { return a.rows ? (a.rows - 1) * a.pitch + a.width : 0; }

    // Checks the pointers and copies host inputs in.
    zn_status bind() {
        int owner[ZN_STAGE_SLOTS];
        for (int i = 0; i < count; ++i) {
            Arg &a = args[i];
            owner[i] = a.p ? zn_ptr_device(a.p) : -1;
            if (!a.p) continue;
            if (owner[i] >= 0 && owner[i] != ctx->device)
                return zn_fail(ctx, ZN_ERR_INVALID_DEVICE, "%s: operand lives on device %d, the context on device %d", op, owner[i], ctx->device);
            if (reinterpret_cast<uintptr_t>(a.p) % (owner[i] >= 0 ? a.align : 4) != 0)
                return zn_fail(ctx, ZN_ERR_INVALID_VALUE, "%s: operand %d is not aligned", op, i);
        }
        for (int i = 0; i < count; ++i)
            for (int j = 0; j < count; ++j) {
                if (i == j || !args[i].p || !args[j].p || args[i].kind == IN) continue;
                const char *x = (const char *)args[i].p, *y = (const char *)args[j].p;
                if (x >= y + 4 * extent(args[j]) || y >= x + 4 * extent(args[i])) continue;
                const bool pair = (i == in_place_a && j == in_place_b) || (i == in_place_b && j == in_place_a);
                if (!(pair && x == y && args[i].pitch == args[j].pitch))
                    return zn_fail(ctx, ZN_ERR_INVALID_VALUE, "%s: an output overlaps another operand", op);
            }
        ZN_CUDA(ctx, cudaSetDevice(ctx->device));
        for (int i = 0; i < count; ++i) {
            Arg &a = args[i];
            if (!a.p) continue;
            if (owner[i] >= 0) { a.dev = const_cast<void *>(a.p); continue; }
            ZN_TRY(zn_stage_reserve(ctx, i, extent(a)));
            a.dev = ctx->stage[i];
            staged[i] = true;
            if (a.kind != OUT) ZN_CUDA(ctx, copy(a.dev, a.p, a, cudaMemcpyHostToDevice));
        }
        return ZN_OK;
    }
    // Copies host outputs back; waits when any operand lived on the host.
    zn_status done() {
        bool any = false;
        for (int i = 0; i < count; ++i) {
            any = any || staged[i];
            if (staged[i] && args[i].kind != IN) ZN_CUDA(ctx, copy(const_cast<void *>(args[i].p), args[i].dev, args[i], cudaMemcpyDeviceToHost));
        }
        if (!any) return ZN_OK;
        ZN_CUDA(ctx, cudaStreamSynchronize(ctx->stream));
        return zn_check_device_status(ctx);
    }

private:
    bool staged[ZN_STAGE_SLOTS] = {};
    // the columns between width and pitch belong to the caller: they are not copied
    cudaError_t copy(void *dst, const void *src, const Arg &a, cudaMemcpyKind kind) {
        if (a.pitch == a.width || a.rows == 1) return cudaMemcpyAsync(dst, src, 4 * extent(a), kind, ctx->stream);
        return cudaMemcpy2DAsync(dst, 4 * a.pitch, src, 4 * a.pitch, 4 * a.width, a.rows, kind, ctx->stream);
    }
};

}   // namespace

extern "C" zn_status zn_embedding_forward(zn_ctx *ctx, const float *table, const int32_t *tokens, float *out, size_t rows,
                                          size_t vocab, size_t dim, float scale) {
    if (!ctx) return ZN_ERR_NOT_INITIALIZED;
    if (vocab == 0 || dim == 0) return zn_fail(ctx, ZN_ERR_SHAPE, "embedding_forward: empty table");
    ZN_TRY(check_sizes(ctx, "embedding_forward", rows, vocab, dim));
    if (rows == 0) return ZN_OK;
    if (!table || !tokens || !out) return zn_fail(ctx, ZN_ERR_INVALID_VALUE, "embedding_forward: null operand");
    Call call(ctx, "embedding_forward");
    const int t = call.add(table, vocab, dim, dim, Call::IN), id = call.add(tokens, 1, rows, rows, Call::IN);
    const int o = call.add(out, rows, dim, dim, Call::OUT);
    ZN_TRY(call.bind());
    ZN_TRY(zn_k_embedding_forward(ctx, call.dev<float>(t), call.dev<int32_t>(id), call.dev<float>(o), rows, vocab, dim, scale));
    return call.done();
}

extern "C" zn_status zn_embedding_backward(zn_ctx *ctx, const float *grad_out, const int32_t *tokens, float *grad_table,
                                           size_t rows, size_t vocab, size_t dim, float scale, int32_t accumulate) {
    if (!ctx) return ZN_ERR_NOT_INITIALIZED;
    if (vocab == 0 || dim == 0) return zn_fail(ctx, ZN_ERR_SHAPE, "embedding_backward: empty table");
    ZN_TRY(check_sizes(ctx, "embedding_backward", rows, vocab, dim));
    if (rows == 0 && accumulate) return ZN_OK;
    if (((!grad_out || !tokens) && rows > 0) || !grad_table) return zn_fail(ctx, ZN_ERR_INVALID_VALUE, "embedding_backward: null operand");
    Call call(ctx, "embedding_backward");
    const int g = call.add(rows ? grad_out : nullptr, rows, dim, dim, Call::IN), id = call.add(rows ? tokens : nullptr, 1, rows, rows, Call::IN);
    const int t = call.add(grad_table, vocab, dim, dim, accumulate ? Call::INOUT : Call::OUT);
    ZN_TRY(call.bind());
    ZN_TRY(zn_k_embedding_backward(ctx, call.dev<float>(g), call.dev<int32_t>(id), call.dev<float>(t), rows, vocab, dim, scale, accumulate != 0));
    return call.done();
}

extern "C" zn_status zn_token_logprobs(zn_ctx *ctx, const float *logits, size_t ld, const int32_t *tokens, size_t rows,
                                       size_t vocab, float temperature, size_t top_k, float *logprob, float *entropy,
                                       float *row_stats, int32_t *top_tokens, float *top_logprobs) {
    const char *op = "token_logprobs";
    if (!ctx) return ZN_ERR_NOT_INITIALIZED;
    ZN_TRY(check_logits(ctx, op, rows, vocab, ld));
    ZN_TRY(check_temperature(ctx, op, temperature));
    if (top_k > ZN_TOP_MAX) return zn_fail(ctx, ZN_ERR_INVALID_VALUE, "%s: %zu alternatives, at most %d are taken", op, top_k, (int)ZN_TOP_MAX);
    if (rows == 0) return ZN_OK;
    if (!logits) return zn_fail(ctx, ZN_ERR_INVALID_VALUE, "%s: null operand", op);
    if (!tokens != !logprob) return zn_fail(ctx, ZN_ERR_INVALID_VALUE, "%s: tokens and logprob go together", op);
    if (!top_tokens != (top_k == 0) || !top_logprobs != (top_k == 0))
        return zn_fail(ctx, ZN_ERR_INVALID_VALUE, "%s: top_tokens, top_logprobs and top_k > 0 go together", op);
    if (!logprob && !entropy && !row_stats && top_k == 0) return zn_fail(ctx, ZN_ERR_INVALID_VALUE, "%s: no output asked for", op);
    Call call(ctx, op);
    const int x = call.add(logits, rows, vocab, ld, Call::IN), id = call.add(tokens, 1, rows, rows, Call::IN);
    const int lp = call.add(logprob, 1, rows, rows, Call::OUT), h = call.add(entropy, 1, rows, rows, Call::OUT);
    const int st = call.add(row_stats, rows, 2, 2, Call::OUT), tt = call.add(top_tokens, rows, top_k, top_k, Call::OUT);
    const int tl = call.add(top_logprobs, rows, top_k, top_k, Call::OUT);
    ZN_TRY(call.bind());
    zn_scores_args a{call.dev<float>(x), (int64_t)ld, call.dev<int32_t>(id), (int64_t)rows, (int64_t)vocab, temperature, (int)top_k,
                     call.dev<float>(lp), call.dev<float>(h), call.dev<float>(st), call.dev<int32_t>(tt), call.dev<float>(tl)};
    ZN_TRY(zn_k_token_logprobs(ctx, a));
    return call.done();
}

extern "C" zn_status zn_token_logprobs_backward(zn_ctx *ctx, const float *logits, size_t ld, const int32_t *tokens,
                                                const float *row_stats, const float *entropy, const float *grad_logprob,
                                                const float *grad_entropy, float *grad_logits, size_t ld_grad, size_t rows,
                                                size_t vocab, float temperature) {
    const char *op = "token_logprobs_backward";
    if (!ctx) return ZN_ERR_NOT_INITIALIZED;
    ZN_TRY(check_logits(ctx, op, rows, vocab, ld));
    ZN_TRY(check_logits(ctx, op, rows, vocab, ld_grad));
    ZN_TRY(check_temperature(ctx, op, temperature));
    if (rows == 0) return ZN_OK;
    if (!logits || !row_stats || !grad_logits) return zn_fail(ctx, ZN_ERR_INVALID_VALUE, "%s: null operand", op);
    if (!grad_logprob && !grad_entropy) return zn_fail(ctx, ZN_ERR_INVALID_VALUE, "%s: grad_logprob and grad_entropy are both null", op);
    if (grad_logprob && !tokens) return zn_fail(ctx, ZN_ERR_INVALID_VALUE, "%s: grad_logprob needs the tokens", op);
    if (grad_entropy && !entropy) return zn_fail(ctx, ZN_ERR_INVALID_VALUE, "%s: grad_entropy needs the entropy", op);
    Call call(ctx, op);
    const int x = call.add(logits, rows, vocab, ld, Call::IN);
    const int id = call.add(grad_logprob ? tokens : nullptr, 1, rows, rows, Call::IN);
    const int st = call.add(row_stats, rows, 2, 2, Call::IN);
    const int h = call.add(grad_entropy ? entropy : nullptr, 1, rows, rows, Call::IN);
    const int gl = call.add(grad_logprob, 1, rows, rows, Call::IN), gh = call.add(grad_entropy, 1, rows, rows, Call::IN);
    const int g = call.add(grad_logits, rows, vocab, ld_grad, Call::OUT);
    call.in_place_a = x;
    call.in_place_b = g;
    ZN_TRY(call.bind());
    zn_scores_grad_args a{call.dev<float>(x), (int64_t)ld, call.dev<int32_t>(id), call.dev<float>(st), call.dev<float>(h),
                          call.dev<float>(gl), call.dev<float>(gh), call.dev<float>(g), (int64_t)ld_grad, (int64_t)rows, (int64_t)vocab, temperature};
    ZN_TRY(zn_k_token_logprobs_backward(ctx, a));
    return call.done();
}

extern "C" zn_status zn_distill_loss(zn_ctx *ctx, const float *logits, size_t ld, const int32_t *teacher_tokens,
                                     const float *teacher_logits, size_t rows, size_t vocab, size_t k, float temperature,
                                     const float *row_weights, float *row_loss, float *grad_logits, size_t ld_grad) {
    const char *op = "distill_loss";
    if (!ctx) return ZN_ERR_NOT_INITIALIZED;
    ZN_TRY(check_logits(ctx, op, rows, vocab, ld));
    if (grad_logits) ZN_TRY(check_logits(ctx, op, rows, vocab, ld_grad));
    if (k == 0 || k > ZN_TEACHER_MAX) return zn_fail(ctx, ZN_ERR_SHAPE, "%s: teacher lists of %zu entries (1..%d are taken)", op, k, (int)ZN_TEACHER_MAX);
    ZN_TRY(check_sizes(ctx, op, rows, k, 1));
    ZN_TRY(check_temperature(ctx, op, temperature));
    if (rows == 0) return ZN_OK;
    if (!logits || !teacher_tokens || !teacher_logits) return zn_fail(ctx, ZN_ERR_INVALID_VALUE, "%s: null operand", op);
    if (!row_loss && !grad_logits) return zn_fail(ctx, ZN_ERR_INVALID_VALUE, "%s: no output asked for", op);
    Call call(ctx, op);
    const int x = call.add(logits, rows, vocab, ld, Call::IN);
    const int id = call.add(teacher_tokens, rows, k, k, Call::IN), u = call.add(teacher_logits, rows, k, k, Call::IN);
    const int w = call.add(row_weights, 1, rows, rows, Call::IN), l = call.add(row_loss, 1, rows, rows, Call::OUT);
    const int g = call.add(grad_logits, rows, vocab, ld_grad, Call::OUT);
    call.in_place_a = x;
    call.in_place_b = g;
    ZN_TRY(call.bind());
    zn_distill_args a{call.dev<float>(x), (int64_t)ld, call.dev<int32_t>(id), call.dev<float>(u), (int64_t)rows, (int64_t)vocab, (int)k,
                      temperature, call.dev<float>(w), call.dev<float>(l), call.dev<float>(g), (int64_t)ld_grad};
    ZN_TRY(zn_k_distill(ctx, a));
    return call.done();
}

extern "C" zn_status zn_quantize4(zn_ctx *ctx, const float *w, uint32_t *packed, float *scales, size_t n, size_t k, size_t group) {
    const char *op = "quantize4";
    if (!ctx) return ZN_ERR_NOT_INITIALIZED;
    if (n == 0 || k == 0) return zn_fail(ctx, ZN_ERR_SHAPE, "%s: zero dimension", op);
    ZN_TRY(check_sizes(ctx, op, n, k, 1));
    ZN_TRY(check_group(ctx, op, group));
    if (!w || !packed || !scales) return zn_fail(ctx, ZN_ERR_INVALID_VALUE, "%s: null operand", op);
    const size_t words = (k + 127) / 128 * 16, groups = (k + group - 1) / group;
    Call call(ctx, op);
    const int wi = call.add(w, k, n, n, Call::IN), p = call.add(packed, n, words, words, Call::OUT, 16);
    const int s = call.add(scales, n, groups, groups, Call::OUT);
    ZN_TRY(call.bind());
    ZN_TRY(zn_k_quantize4(ctx, call.dev<float>(wi), call.dev<uint32_t>(p), call.dev<float>(s), n, k, group));
    return call.done();
}

extern "C" zn_status zn_matmul4_bias_act(zn_ctx *ctx, const float *x, const uint32_t *packed, const float *scales,
                                         const float *bias, float *y, size_t rows, size_t n, size_t k, size_t group,
                                         zn_activation act) {
    const char *op = "matmul4_bias_act";
    if (!ctx) return ZN_ERR_NOT_INITIALIZED;
    if (n == 0 || k == 0) return zn_fail(ctx, ZN_ERR_SHAPE, "%s: zero dimension", op);
    ZN_TRY(check_sizes(ctx, op, rows, n, k));
    ZN_TRY(check_group(ctx, op, group));
    if ((int)act < ZN_ACT_RELU || (int)act > ZN_ACT_ELU) return zn_fail(ctx, ZN_ERR_INVALID_VALUE, "%s: unknown activation %d", op, (int)act);
    if (rows == 0) return ZN_OK;
    if (!x || !packed || !scales || !y) return zn_fail(ctx, ZN_ERR_INVALID_VALUE, "%s: null operand", op);
    const size_t words = (k + 127) / 128 * 16, groups = (k + group - 1) / group;
    Call call(ctx, op);
    const int xi = call.add(x, rows, k, k, Call::IN), p = call.add(packed, n, words, words, Call::IN, 16);
    const int s = call.add(scales, n, groups, groups, Call::IN), b = call.add(bias, 1, n, n, Call::IN);
    const int o = call.add(y, rows, n, n, Call::OUT);
    ZN_TRY(call.bind());
    // softmax needs whole rows: the product writes the biased pre-activations, a row kernel follows
    const int fused = act == ZN_ACT_SOFTMAX ? (int)ZN_ACT_LINEAR : (int)act;
    ZN_TRY(zn_k_matmul4(ctx, call.dev<float>(xi), call.dev<uint32_t>(p), call.dev<float>(s), call.dev<float>(b), call.dev<float>(o), rows, n, k,
                        group, fused));
    if (act == ZN_ACT_SOFTMAX)
        ZN_TRY(zn_k_softmax_rows(ctx, call.dev<float>(o), false, (int64_t)n, nullptr, false, 0, call.dev<float>(o), (int64_t)n, (int64_t)rows,
                                 (int64_t)n, ctx->precision == ZN_FP32_EXACT));
    return call.done();
}

extern "C" zn_status zn_debug_token_plan(int32_t op, size_t a, size_t b, size_t c, int32_t sms, int64_t out[5]) {
    if (!out || sms <= 0 || op < 0 || op > 6) return ZN_ERR_INVALID_VALUE;
    if (a > MAX_DIM || b > MAX_DIM || c > MAX_DIM) return ZN_ERR_SHAPE;
    zn_token_plan p;
    switch (op) {
    case 0:
        if (b == 0 || c == 0) return ZN_ERR_SHAPE;
        ZN_TRY(check_sizes(nullptr, "", a, b, c));
        p = zn_plan_embedding_forward(a, c, sms);
        break;
    case 1:
        if (b == 0 || c == 0) return ZN_ERR_SHAPE;
        ZN_TRY(check_sizes(nullptr, "", a, b, c));
        p = zn_plan_embedding_backward(a, b, c, sms);
        break;
    case 2:
        ZN_TRY(check_logits(nullptr, "", a, b, b));
        if (c > ZN_TOP_MAX) return ZN_ERR_INVALID_VALUE;
        p = zn_plan_token_logprobs(a, b, c, sms);
        break;
    case 3:
        ZN_TRY(check_logits(nullptr, "", a, b, b));
        p = zn_plan_token_logprobs_backward(a, b, sms);
        break;
    case 4:
        ZN_TRY(check_logits(nullptr, "", a, b, b));
        if (c == 0 || c > ZN_TEACHER_MAX) return ZN_ERR_SHAPE;
        ZN_TRY(check_sizes(nullptr, "", a, c, 1));
        p = zn_plan_distill(a, b, c, sms);
        break;
    case 5:
        if (a == 0 || b == 0) return ZN_ERR_SHAPE;
        ZN_TRY(check_sizes(nullptr, "", a, b, 1));
        ZN_TRY(check_group(nullptr, "", c));
        p = zn_plan_quantize4(a, b, sms);
        break;
    default:
        if (b == 0 || c == 0) return ZN_ERR_SHAPE;
        ZN_TRY(check_sizes(nullptr, "", a, b, c));
        p = zn_plan_matmul4(a, b, c, sms);
    }
    out[0] = a == 0 ? 0 : p.blocks;
    out[1] = p.threads;
    out[2] = p.share;
    out[3] = (int64_t)p.smem;
    out[4] = (int64_t)p.scratch_floats;
    return ZN_OK;
}
