// 4-bit weights in scaled groups: quantisation, and the product for few rows.
//
// The product is bound by the bytes of the weights, so a weight must not cost many instructions.  It goes through the
// tensor cores in their warp form (a tile of 16 columns of w by 8 columns of x: the shape of few rows), with codes turned
// into bf16 two at a time: a code in the low bits of the bf16 number 128 is 128 + code exactly, and code - 8 after one
// subtraction.  x keeps all its 24 bits as the sum of three bf16 numbers, which take three columns of the tile; a product
// of two bf16 numbers is exact in f32, so the only roundings are those of the f32 sums.  A group's sum is scaled once.
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

// x as the product reads it.  For each 32 weights and each eight columns of the tile (column 3 r + part of row r): the 16
// bytes that every lane of a warp feeds to two tensor-core steps.  Lane 4 g + t holds column g at the weights
// 8 t + {0, 4, 1, 5, 2, 6, 3, 7}, the order in which masks take the codes out of a word.
__global__ void split_kernel(const float *__restrict__ x, uint4 *__restrict__ out, int rows, int64_t k, int64_t total, int tiles) {
    zn_pdl_release();
    for (int64_t at = (int64_t)blockIdx.x * TPB + threadIdx.x; at < total; at += (int64_t)gridDim.x * TPB) {
        const int lane = (int)(at & 31), t = lane & 3;
        const int64_t tile = at >> 5;
        const int column = (int)(tile % tiles) * 8 + (lane >> 2), row = column / 3, part = column % 3;
        const int64_t k0 = tile / tiles * 32 + 8 * t;
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int64_t kk = k0 + (i >> 1) + (i & 1) * 4;
            const float v = row < rows && kk < k ? x[row * k + kk] : 0.f;
            // cut, not rounded: each part takes the next eight bits, and what is left is exact
            uint32_t bits = __float_as_uint(v);
            if (!(fabsf(v) < INFINITY)) {
                bits = part > 0 ? 0u : isnan(v) ? 0x7fc00000u : bits;
            } else if (part > 0) {
                float rest = v - __uint_as_float(bits & 0xffff0000u);
                if (part > 1) rest -= __uint_as_float(__float_as_uint(rest) & 0xffff0000u);
                bits = __float_as_uint(rest);
            }
            if (i & 1) w[i >> 1] |= bits & 0xffff0000u;
            else w[i >> 1] = bits >> 16;
        }
        out[at] = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// Two codes of a word, `s` and `s` + 4, less 8 as a pair of bf16.
__device__ __forceinline__ uint32_t code_pair(uint32_t word, int s) {
    const uint32_t raw = ((word >> (4 * s)) & 0x000f000fu) | 0x43004300u;
    const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&raw), __nv_bfloat162(__float2bfloat16(136.f), __float2bfloat16(136.f)));
    return *reinterpret_cast<const uint32_t *>(&v);
}
__device__ __forceinline__ void mma_16x8(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

struct Product {
    const uint4 *x, *w;
    const float *scales, *bias;
    float *y;
    int64_t n, blocks, groups;        // blocks of 128 weights, groups per column
    int rows, group_log, wide, act;
};

// Eight warps: `wide` of them side by side over the columns of w, TALL tiles of 16 each, the others along k.  A lane reads
// 16 bytes of a column at a time (128 weights by four lanes), the next ones before it works on these.
template <int TILES, int TALL>
__global__ void __launch_bounds__(TPB) matmul4_kernel(Product a) {
    extern __shared__ float sums[];                        // [warp][16 TALL][8 TILES + 1]
    zn_pdl_release();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int side = warp % a.wide, depth = TPB / 32 / a.wide;
    const int64_t first = ((int64_t)blockIdx.x * a.wide + side) * (16 * TALL);
    const uint4 *w[TALL][2];
    const float *sc[TALL][2];
#pragma unroll
    for (int j = 0; j < TALL; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int64_t row = min(a.n - 1, first + 16 * j + 8 * h + g);      // past the last column: read it again, drop the result
            w[j][h] = a.w + row * a.blocks * 4 + t;
            sc[j][h] = a.scales + row * a.groups;
        }
    float total[TALL][TILES][4], sum[TALL][TILES][4];
#pragma unroll
    for (int j = 0; j < TALL; ++j)
#pragma unroll
        for (int q = 0; q < TILES; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) total[j][q][e] = sum[j][q][e] = 0.f;
    int64_t b = warp / a.wide;
    uint4 next[TALL][2];
#pragma unroll
    for (int j = 0; j < TALL; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) next[j][h] = b < a.blocks ? __ldcs(w[j][h] + b * 4) : make_uint4(0, 0, 0, 0);
    zn_pdl_wait();                                          // x comes from the kernel before
    for (; b < a.blocks; b += depth) {
        uint4 now[TALL][2];
#pragma unroll
        for (int j = 0; j < TALL; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                now[j][h] = next[j][h];
                if (b + depth < a.blocks) next[j][h] = __ldcs(w[j][h] + (b + depth) * 4);
            }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint4 xb[TILES];
#pragma unroll
            for (int q = 0; q < TILES; ++q) xb[q] = __ldg(a.x + ((b * 4 + i) * TILES + q) * 32 + lane);
#pragma unroll
            for (int j = 0; j < TALL; ++j) {
                const uint32_t lo = i == 0 ? now[j][0].x : i == 1 ? now[j][0].y : i == 2 ? now[j][0].z : now[j][0].w;
                const uint32_t hi = i == 0 ? now[j][1].x : i == 1 ? now[j][1].y : i == 2 ? now[j][1].z : now[j][1].w;
                const uint32_t l0 = code_pair(lo, 0), l1 = code_pair(lo, 1), l2 = code_pair(lo, 2), l3 = code_pair(lo, 3);
                const uint32_t h0 = code_pair(hi, 0), h1 = code_pair(hi, 1), h2 = code_pair(hi, 2), h3 = code_pair(hi, 3);
#pragma unroll
                for (int q = 0; q < TILES; ++q) {
                    mma_16x8(sum[j][q], l0, h0, l1, h1, xb[q].x, xb[q].y);
                    mma_16x8(sum[j][q], l2, h2, l3, h3, xb[q].z, xb[q].w);
                }
            }
            if ((((i + 1) << 5) & ((1 << a.group_log) - 1)) == 0) {       // a group ends here
                const int64_t group = (b * 128 + i * 32) >> a.group_log;
#pragma unroll
                for (int j = 0; j < TALL; ++j) {
                    const float s0 = group < a.groups ? __ldg(sc[j][0] + group) : 0.f, s1 = group < a.groups ? __ldg(sc[j][1] + group) : 0.f;
#pragma unroll
                    for (int q = 0; q < TILES; ++q) {
                        total[j][q][0] = fmaf(s0, sum[j][q][0], total[j][q][0]);
                        total[j][q][1] = fmaf(s0, sum[j][q][1], total[j][q][1]);
                        total[j][q][2] = fmaf(s1, sum[j][q][2], total[j][q][2]);
                        total[j][q][3] = fmaf(s1, sum[j][q][3], total[j][q][3]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) sum[j][q][e] = 0.f;
                    }
                }
            }
        }
    }
    constexpr int PITCH = 8 * TILES + 1;
    float *mine = sums + warp * (16 * TALL) * PITCH;
#pragma unroll
    for (int j = 0; j < TALL; ++j)
#pragma unroll
        for (int q = 0; q < TILES; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) mine[(16 * j + 8 * (e >> 1) + g) * PITCH + 8 * q + 2 * t + (e & 1)] = total[j][q][e];
    __syncthreads();
    // the parts of x and the warps along k, in a fixed order, the smallest parts first
    const int columns = 16 * TALL * a.wide;
    for (int i = threadIdx.x; i < columns * a.rows; i += TPB) {
        const int col = i % columns, row = i / columns;
        const int64_t at = (int64_t)blockIdx.x * columns + col;
        if (at >= a.n) continue;
        float part[3] = {0.f, 0.f, 0.f};
        for (int d = 0; d < depth; ++d) {
            const float *p = sums + ((d * a.wide + col / (16 * TALL)) * (16 * TALL) + col % (16 * TALL)) * PITCH + 3 * row;
#pragma unroll
            for (int e = 0; e < 3; ++e) part[e] += p[e];
        }
        const float v = part[0] + (part[1] + part[2]);
        a.y[(int64_t)row * a.n + at] = apply_act(a.act, a.bias ? v + __ldg(a.bias + at) : v);
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

namespace {

constexpr int ROWS_AT_ONCE = 16;

// Tiles of 16 columns per warp and warps side by side: what reads x least often while two blocks per SM remain.
struct Shape {
    int tiles, tall, wide;
    int64_t blocks;
    size_t smem, split;
};
Shape shape_of(int64_t rows, int64_t n, int64_t k, int sms) {
    Shape s;
    s.tiles = (int)((3 * (rows < ROWS_AT_ONCE ? rows : ROWS_AT_ONCE) + 7) / 8);
    if (s.tiles < 1) s.tiles = 1;
    s.tall = n >= (int64_t)64 * sms ? 2 : 1;
    s.wide = 1;
    while (s.wide < 4 && n >= (int64_t)16 * s.tall * s.wide * 2 * 2 * sms) s.wide *= 2;
    const int64_t columns = (int64_t)16 * s.tall * s.wide;
    s.blocks = (n + columns - 1) / columns;
    s.smem = (size_t)(TPB / 32) * 16 * s.tall * (8 * s.tiles + 1) * sizeof(float);
    s.split = (size_t)((k + 127) / 128) * 4 * s.tiles * 32 * 4;        // floats of scratch
    return s;
}

template <int TILES>
zn_status launch(zn_ctx *ctx, const Product &p, const Shape &s) {
    const auto kernel = s.tall == 2 ? matmul4_kernel<TILES, 2> : matmul4_kernel<TILES, 1>;
    if (s.smem > 48 * 1024) ZN_CUDA(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)s.smem));
    ZN_CUDA(ctx, zn_launch_pdl(kernel, dim3((unsigned)s.blocks), dim3(TPB), s.smem, ctx->stream, p));
    return ZN_OK;
}

}   // namespace

zn_token_plan zn_plan_matmul4(size_t rows, size_t n, size_t k, int sms) {
    const Shape s = shape_of((int64_t)rows, (int64_t)n, (int64_t)k, sms);
    zn_token_plan p;
    p.threads = TPB;
    p.blocks = s.blocks;
    p.smem = s.smem;
    p.scratch_floats = s.split;
    return p;
}

zn_status zn_k_matmul4(zn_ctx *ctx, const float *x, const uint32_t *packed, const float *scales, const float *bias, float *y,
                       size_t rows, size_t n, size_t k, size_t group, int act) {
    for (size_t r = 0; r < rows; r += ROWS_AT_ONCE) {
        const size_t now = rows - r < ROWS_AT_ONCE ? rows - r : (size_t)ROWS_AT_ONCE;
        const Shape s = shape_of((int64_t)now, (int64_t)n, (int64_t)k, ctx->sm_count);
        ZN_TRY(zn_scratch_reserve(ctx, s.split));
        uint4 *split = reinterpret_cast<uint4 *>(ctx->scratch);
        zn_launch_scope scope(ctx, ZN_PROF_GEMM_TC, 2.0 * now * n * k, 0.5 * n * k + 4.0 * n * k / group + 4.0 * now * (n + k), 2);
        const int64_t total = (int64_t)(s.split / 4);
        int64_t blocks = (total + TPB - 1) / TPB;
        if (blocks > ctx->sm_count * 8) blocks = ctx->sm_count * 8;
        split_kernel<<<(unsigned)blocks, TPB, 0, ctx->stream>>>(x + r * k, split, (int)now, (int64_t)k, total, s.tiles);
        ZN_CUDA(ctx, cudaGetLastError());
        Product p{split, reinterpret_cast<const uint4 *>(packed), scales, bias, y + r * n, (int64_t)n, (int64_t)((k + 127) / 128),
                  (int64_t)((k + group - 1) / group), (int)now, group == 32 ? 5 : group == 64 ? 6 : 7, s.wide, act};
        switch (s.tiles) {
        case 1: ZN_TRY(launch<1>(ctx, p, s)); break;
        case 2: ZN_TRY(launch<2>(ctx, p, s)); break;
        case 3: ZN_TRY(launch<3>(ctx, p, s)); break;
        case 4: ZN_TRY(launch<4>(ctx, p, s)); break;
        case 5: ZN_TRY(launch<5>(ctx, p, s)); break;
        default: ZN_TRY(launch<6>(ctx, p, s));
        }
    }
    return ZN_OK;
}
