// 4-bit weights in scaled groups: quantisation, and the product for few rows.
#include "zn_token.cuh"
#include "zn_act.cuh"

namespace {

constexpr int TPB = 256;

__device__ __forceinline__ float apply_act(int act, float x) {
    switch (act) {
    case ZN_ACT_RELU: return x > 0.f ? x : 0.f;
    case ZN_ACT_SIGMOID:
        if (x >= 0.f) return 1.f / (1.f + expf(-x));
        else { const float e = expf(x); return e / (1.f + e); }
    case ZN_ACT_TANH: return tanhf(x);
    case ZN_ACT_GELU: return zn_gelu_fwd(x);
    case ZN_ACT_LEAKY_RELU: return zn_leaky_fwd(x);
    case ZN_ACT_ELU: return zn_elu_fwd(x);
    default: return x;
    }
}

// Place of word w (codes 8 w .. 8 w + 7 of a column) in the packed row.
__device__ __forceinline__ int64_t word_place(int64_t w) { return (w & ~15ll) + (w & 3) * 4 + ((w & 15) >> 2); }

// One thread per (group, column); neighbouring threads take neighbouring columns, so the reads of w are whole lines.
__global__ void quantize_kernel(const float *__restrict__ w, uint32_t *__restrict__ packed, float *__restrict__ scales, int64_t n, int64_t k,
                                int64_t group) {
    const int64_t words = (k + 127) / 128 * 16, groups = (k + group - 1) / group, padded = words * 8 / group;
    const int64_t total = n * padded;
    for (int64_t at = (int64_t)blockIdx.x * TPB + threadIdx.x; at < total; at += (int64_t)gridDim.x * TPB) {
        const int64_t j = at % n, g = at / n;
        const int64_t lo = g * group, hi = min(k, lo + group);
        float top = 0.f;
        bool bad = false;
        for (int64_t i = lo; i < hi; ++i) {
            const float v = w[i * n + j];
            if (!(fabsf(v) < INFINITY)) bad = true;
            top = fmaxf(top, fabsf(v));
        }
        const float scale = __fdiv_rn(top, 7.f);
        if (g < groups) scales[j * groups + g] = bad ? __int_as_float(0x7fffffff) : scale;
        for (int64_t i = lo; i < lo + group; i += 8) {
            uint32_t word = 0;
            for (int b = 0; b < 8; ++b) {
                int code = 8;
                if (i + b < hi && !bad && scale > 0.f) {
                    const float q = rintf(__fdiv_rn(w[(i + b) * n + j], scale));
                    code = 8 + (int)fminf(7.f, fmaxf(-7.f, q));
                }
                word |= (uint32_t)code << (4 * b);
            }
            packed[j * words + word_place(i / 8)] = word;
        }
    }
}

// One warp per output.
__global__ void matmul4_kernel(const float *__restrict__ x, const uint32_t *__restrict__ packed, const float *__restrict__ scales,
                               const float *__restrict__ bias, float *__restrict__ y, int64_t rows, int64_t n, int64_t k, int64_t group, int act) {
    const int64_t words = (k + 127) / 128 * 16, groups = (k + group - 1) / group;
    const int lane = threadIdx.x & 31;
    const int64_t total = rows * n;
    for (int64_t o = ((int64_t)blockIdx.x * TPB + threadIdx.x) >> 5; o < total; o += ((int64_t)gridDim.x * TPB) >> 5) {
        const int64_t r = o / n, j = o % n;
        float s = 0.f;
        for (int64_t i = lane; i < k; i += 32) {
            const uint32_t code = (packed[j * words + word_place(i / 8)] >> (4 * (i & 7))) & 15u;
            s += x[r * k + i] * ((float)((int)code - 8) * scales[j * groups + i / group]);
        }
        s = zn_warp_sum(s);
        if (lane == 0) y[o] = apply_act(act, s + (bias ? bias[j] : 0.f));
    }
}

}   // namespace

zn_token_plan zn_plan_quantize4(size_t n, size_t k, int sms) {
    zn_token_plan p;
    p.threads = TPB;
    const int64_t want = (int64_t)((n * ((k + 127) / 128) + TPB - 1) / TPB);
    p.blocks = want < (int64_t)sms * 8 ? want : (int64_t)sms * 8;
    return p;
}

zn_status zn_k_quantize4(zn_ctx *ctx, const float *w, uint32_t *packed, float *scales, size_t n, size_t k, size_t group) {
    const zn_token_plan p = zn_plan_quantize4(n, k, ctx->sm_count);
    zn_launch_scope scope(ctx, ZN_PROF_CONVERT, 0, 4.5 * n * k);
    quantize_kernel<<<(unsigned)p.blocks, p.threads, 0, ctx->stream>>>(w, packed, scales, (int64_t)n, (int64_t)k, (int64_t)group);
    ZN_CUDA(ctx, cudaGetLastError());
    return ZN_OK;
}

zn_token_plan zn_plan_matmul4(size_t rows, size_t n, size_t k, int sms) {
    zn_token_plan p;
    (void)k;
    p.threads = TPB;
    const int64_t want = (int64_t)((rows * n + TPB / 32 - 1) / (TPB / 32));
    p.blocks = want < (int64_t)sms * 8 ? want : (int64_t)sms * 8;
    return p;
}

zn_status zn_k_matmul4(zn_ctx *ctx, const float *x, const uint32_t *packed, const float *scales, const float *bias, float *y,
                       size_t rows, size_t n, size_t k, size_t group, int act) {
    const zn_token_plan p = zn_plan_matmul4(rows, n, k, ctx->sm_count);
    zn_launch_scope scope(ctx, ZN_PROF_GEMM_SIMT, 2.0 * rows * n * k, 0.5 * n * k);
    matmul4_kernel<<<(unsigned)p.blocks, p.threads, 0, ctx->stream>>>(x, packed, scales, bias, y, (int64_t)rows, (int64_t)n, (int64_t)k,
                                                                      (int64_t)group, act);
    ZN_CUDA(ctx, cudaGetLastError());
    return ZN_OK;
}
