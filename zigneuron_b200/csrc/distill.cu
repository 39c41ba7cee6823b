// Distillation from a teacher's top logits: loss and gradient of a row in one block.
#include "zn_token.cuh"

namespace {

constexpr int TPB = 256;

__global__ void distill_kernel(zn_distill_args a, int *status) {
    __shared__ float part[TPB / 32];
    __shared__ float q[ZN_TEACHER_MAX], xt[ZN_TEACHER_MAX];
    __shared__ int32_t id[ZN_TEACHER_MAX];
    const float nan = __int_as_float(0x7fffffff), inv_t = 1.f / a.temperature;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const float *x = a.logits + r * a.ld;
        float *g = a.grad ? a.grad + r * a.ld_grad : nullptr;
        const float w = a.weights ? a.weights[r] : 1.f;
        __syncthreads();
        // the teacher's entries: softmax(u / T)
        float um = -INFINITY, wrong = 0.f, ubad = 0.f;
        for (int j = threadIdx.x; j < a.k; j += TPB) {
            const int32_t t = a.ids[r * a.k + j];
            const float u = a.teacher[r * a.k + j];
            const bool entry = t >= 0 && u != -INFINITY;
            if (entry && t >= a.vocab) { wrong = 1.f; zn_bad_token(status); }
            if (entry && !(u < INFINITY)) ubad = 1.f;
            id[j] = entry && t < a.vocab ? t : -1;
            q[j] = u;
            xt[j] = id[j] >= 0 ? x[t] : 0.f;
            if (entry) um = fmaxf(um, u);
        }
        um = zn_block_max<TPB>(um, part);
        wrong = zn_block_max<TPB>(wrong, part);
        ubad = zn_block_max<TPB>(ubad, part);
        if (w == 0.f || (um == -INFINITY && ubad == 0.f) || wrong != 0.f) {
            if (g)
                for (int64_t c = threadIdx.x; c < a.vocab; c += TPB) g[c] = 0.f;
            if (a.loss && threadIdx.x == 0) a.loss[r] = w != 0.f && wrong != 0.f ? nan : 0.f;
            continue;
        }
        float mass = 0.f;
        for (int j = threadIdx.x; j < a.k; j += TPB)
            if (id[j] >= 0) mass += expf((q[j] - um) * inv_t);
        mass = zn_block_sum<TPB>(mass, part);
        // the student's statistics
        float mx = -INFINITY, bad = ubad;
        for (int64_t c = threadIdx.x; c < a.vocab; c += TPB) {
            const float v = x[c];
            if (!(v < INFINITY)) bad = 1.f;
            mx = fmaxf(mx, v);
        }
        mx = zn_block_max<TPB>(mx, part);
        bad = zn_block_max<TPB>(bad, part);
        const bool empty = mx == -INFINITY;
        float s = 0.f;
        for (int64_t c = threadIdx.x; c < a.vocab; c += TPB) s += expf((x[c] - mx) * inv_t);
        s = zn_block_sum<TPB>(s, part);
        const float ls = logf(s), lm = logf(mass);
        float loss = 0.f;
        for (int j = threadIdx.x; j < a.k; j += TPB) {
            if (id[j] < 0) continue;
            const float lq = (q[j] - um) * inv_t - lm, lp = empty ? -INFINITY : (xt[j] - mx) * inv_t - ls, qj = expf(lq);
            if (qj > 0.f) loss += qj * (lq - lp);
            q[j] = qj;
        }
        loss = zn_block_sum<TPB>(loss, part);
        if (a.loss && threadIdx.x == 0) a.loss[r] = bad != 0.f ? nan : w * a.temperature * a.temperature * loss;
        if (!g) continue;
        const float wt = w * a.temperature, inv_s = 1.f / s;
        for (int64_t c = threadIdx.x; c < a.vocab; c += TPB)
            g[c] = bad != 0.f ? nan : empty ? 0.f : wt * (expf((x[c] - mx) * inv_t) * inv_s);
        __syncthreads();
        if (bad != 0.f) continue;
        // the listed tokens: the first place of an id takes the q of all its places
        for (int j = threadIdx.x; j < a.k; j += TPB) {
            if (id[j] < 0) continue;
            float sum = 0.f;
            bool first = true;
            for (int i = 0; i < a.k; ++i)
                if (id[i] == id[j]) {
                    if (i < j) first = false;
                    sum += q[i];
                }
            if (first) g[id[j]] = wt * ((empty ? 0.f : expf((xt[j] - mx) * inv_t) * inv_s) - sum);
        }
    }
}

}   // namespace

zn_token_plan zn_plan_distill(size_t rows, size_t vocab, size_t k, int sms) {
    zn_token_plan p;
    (void)vocab; (void)k;
    p.threads = TPB;
    p.blocks = (int64_t)rows < (int64_t)sms * 8 ? (int64_t)rows : (int64_t)sms * 8;
    return p;
}

zn_status zn_k_distill(zn_ctx *ctx, const zn_distill_args &a) {
    const zn_token_plan p = zn_plan_distill((size_t)a.rows, (size_t)a.vocab, (size_t)a.k, ctx->sm_count);
    zn_launch_scope scope(ctx, ZN_PROF_LOSS, 6.0 * a.rows * a.vocab, (a.grad ? 8.0 : 4.0) * a.rows * a.vocab);
    distill_kernel<<<(unsigned)p.blocks, p.threads, 0, ctx->stream>>>(a, ctx->status_dev);
    ZN_CUDA(ctx, cudaGetLastError());
    return ZN_OK;
}
