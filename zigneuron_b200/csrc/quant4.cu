// 4-bit weights in scaled groups: quantisation, and the product for few rows.
//
// The product is bound by the bytes of the weights, so a weight must not cost many instructions.  It goes through the
// tensor cores in their warp form (a tile of 16 columns of w by 8 columns of x: the shape of few rows), with codes turned
// into bf16 two at a time: a code in the low bits of the bf16 number 128 is 128 + code exactly, and code - 8 after one
// subtraction.  x keeps all its 24 bits as the sum of three bf16 numbers, which take three columns of the tile; a product
// of two bf16 numbers is exact in f32, so the only roundings are those of the f32 sums.  A group's sum is scaled once.
//
// Measured, 65,536 x 8192 weights in groups of 128 (288 MB, 44 us of HBM): one row 76 us, bound by the codes' conversion (51 %
// of the integer pipe's cycles; without it 58 us); eight rows 107 us, bound by the matrix steps (three parts of eight rows:
// 24 columns; without the conversion still 101 us).  4096 x 4096, one row: 10.2 us, latency.
#include <cuda.h>

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

// A block takes 32 columns and 128 weights of each: a warp reads 16 rows of w as whole lines, the groups' largest values meet
// in shared memory, and so do the words, which leave as 64 bytes per column.  Measured, 16,384 x 8192 in groups of
// 128: 228 us, bound by the divisions, against 582 with one thread per group (its words went out four bytes at a time).
constexpr int QUANT_COLUMNS = 32, QUANT_ROWS = 16;
__global__ void __launch_bounds__(TPB) quantize_kernel(const float *__restrict__ w, uint32_t *__restrict__ packed, float *__restrict__ scales,
                                                       int64_t n, int64_t k, int group, int64_t column_blocks) {
    __shared__ float most[TPB / 32][QUANT_COLUMNS];
    __shared__ __align__(16) uint32_t word[QUANT_COLUMNS][20];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t block = blockIdx.x / column_blocks, first = blockIdx.x % column_blocks * QUANT_COLUMNS, j = first + lane;
    const int64_t i0 = block * 128 + warp * QUANT_ROWS, blocks = (k + 127) / 128, groups = (k + group - 1) / group;
    float v[QUANT_ROWS], top = 0.f;
#pragma unroll
    for (int i = 0; i < QUANT_ROWS; ++i) v[i] = j < n && i0 + i < k ? __ldcs(w + (i0 + i) * n + j) : 0.f;
#pragma unroll
    for (int i = 0; i < QUANT_ROWS; ++i) top = fabsf(v[i]) < INFINITY ? fmaxf(top, fabsf(v[i])) : INFINITY;      // NaN counts as infinity
    most[warp][lane] = top;
    __syncthreads();
    const int warps = group / QUANT_ROWS, lead = warp / warps * warps;       // of this warp's group
    for (int i = 0; i < warps; ++i) top = fmaxf(top, most[lead + i][lane]);
    const bool bad = top == INFINITY;
    const float scale = __fdiv_rn(top, 7.f);
    const int64_t g = i0 / group;
    if (warp == lead && j < n && g < groups) scales[j * groups + g] = bad ? zn_nan() : scale;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        uint32_t codes = 0;
#pragma unroll
        for (int b = 0; b < 8; ++b) {
            int code = 8;
            if (!bad && scale > 0.f) code = 8 + (int)fminf(7.f, fmaxf(-7.f, rintf(__fdiv_rn(v[8 * h + b], scale))));
            codes |= (uint32_t)code << (4 * b);
        }
        const int at = 2 * warp + h;
        word[lane][(at & 3) * 4 + (at >> 2)] = codes;
    }
    __syncthreads();
    const int column = threadIdx.x >> 2, part = threadIdx.x & 3;
    if (threadIdx.x < 4 * QUANT_COLUMNS && first + column < n)
        reinterpret_cast<uint4 *>(packed)[((first + column) * blocks + block) * 4 + part] = *reinterpret_cast<const uint4 *>(&word[column][4 * part]);
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
    uint32_t raw;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(raw) : "r"(word >> (4 * s)), "r"(0x000f000fu), "r"(0x43004300u));      // (w & mask) | 128, 128
    asm("sub.bf16x2 %0, %0, %1;" : "+r"(raw) : "r"(0x43084308u));                                                        // less 136, 136
    return raw;
}
__device__ __forceinline__ void mma_16x8(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, bool first) {
    const float c0 = first ? 0.f : d[0], c1 = first ? 0.f : d[1], c2 = first ? 0.f : d[2], c3 = first ? 0.f : d[3];
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}

struct Product {
    const uint4 *x;
    const float *scales, *bias;
    float *y, *partial;               // two places of COLUMNS x rows sums per block
    unsigned int *arrivals;
    int64_t n, groups;                // groups per column
    int blocks, rows, act;            // blocks of 128 weights per column
    int split, stages, tiles;         // blocks of a cluster that share k; stages of the whole k; column tiles
};

constexpr int COLUMNS = 128;          // of w per tile
constexpr int SIDE = 4, TALL = 2;     // warps side by side over them, and tiles of 16 of each

// What a place of the ring holds: DEPTH blocks of 128 weights of every column, and of x, and the scales.
template <int TILES, int WARPS> struct Layout {
    static constexpr int DEPTH = WARPS / SIDE, W = DEPTH * COLUMNS * 64, X = DEPTH * 4 * TILES * 512, S = DEPTH * COLUMNS * 16, STAGE = W + X + S;
    static constexpr int PITCH = 8 * TILES + 1, SUMS = WARPS * 16 * TALL * PITCH * 4;
    static constexpr int RING = (225 * 1024 - SUMS) / STAGE < 6 ? (225 * 1024 - SUMS) / STAGE : 6;
};

// Two warps keep a ring of stages filled (a tensor copy of the weights, a plain one of x, scales word by word, since a row of
// them need not stand on 16 bytes); the others work on it, SIDE of
// them side by side over the columns, each of DEPTH such rows on its own block of 128 weights.
//
// Where there are too few tiles for the GPU, a cluster shares one, each block a stretch of k, and the sums meet through
// distributed shared memory.  Where there are more, the stages of all tiles in a row are cut into equal stretches, one per
// block, which goes through its own without emptying the ring; a tile at a cut leaves partial sums, and the block that
// finishes it last adds them in their order.
template <int TILES, int WARPS, int GROUP_LOG>
__global__ void __launch_bounds__(WARPS * 32 + 64) matmul4_kernel(const __grid_constant__ CUtensorMap map, Product a, int *status) {
    using L = Layout<TILES, WARPS>;
    extern __shared__ __align__(128) unsigned char ring[];
    __shared__ uint64_t full[L::RING], free_[L::RING];
    __shared__ bool joins;
    float *sums = reinterpret_cast<float *>(ring + L::RING * L::STAGE);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = blockIdx.x % a.split;
    // this block's stages, counted over all tiles: tile * stages + stage
    const int64_t units = (int64_t)a.tiles * a.stages;
    const int64_t begin = a.split > 1 ? (int64_t)(blockIdx.x / a.split) * a.stages + a.stages * rank / a.split : units * blockIdx.x / gridDim.x;
    const int64_t end = a.split > 1 ? (int64_t)(blockIdx.x / a.split) * a.stages + a.stages * (rank + 1) / a.split : units * (blockIdx.x + 1) / gridDim.x;
    if (threadIdx.x == 0) {
        for (int i = 0; i < L::RING; ++i) {
            zn_bar_init(&full[i], 33);
            zn_bar_init(&free_[i], WARPS);
        }
        zn_bar_init_done();
    }
    __syncthreads();
    zn_pdl_release();
    // output i of a tile, column by column of a row
    const auto finish = [&](int tile, int i, float v) {
        const int64_t at = (int64_t)tile * COLUMNS + i % COLUMNS;
        if (at < a.n) a.y[(int64_t)(i / COLUMNS) * a.n + at] = apply_act(a.act, a.bias ? v + __ldg(a.bias + at) : v);
    };
    if (warp == WARPS) {
        if (lane == 0) {
            const auto x_bytes = [&](int s) { return (uint32_t)(min(L::DEPTH, a.blocks - s * L::DEPTH) * (4 * TILES * 512)); };
            const auto load_w = [&](int tile, int s, int place) {
                zn_bar_expect(&full[place], L::W + x_bytes(s));
                asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                             ::"r"(zn_smem(ring + place * L::STAGE)), "l"(&map), "r"(0), "r"(tile * COLUMNS), "r"(s * L::DEPTH), "r"(zn_smem(&full[place]))
                             : "memory");
            };
            const auto load_x = [&](int s, int place) {
                zn_bulk_load(ring + place * L::STAGE + L::W, a.x + (int64_t)s * L::DEPTH * 4 * TILES * 32, x_bytes(s), &full[place]);
            };
            // the weights are there already; x comes from the kernel before, which may still run
            const int ahead = (int)min((int64_t)L::RING, end - begin);
            int tile = (int)(begin / a.stages), stage = (int)(begin % a.stages);
            const auto forward = [&]() {
                if (++stage == a.stages) {
                    stage = 0;
                    ++tile;
                }
            };
            for (int i = 0; i < ahead; ++i, forward()) load_w(tile, stage, i);
            zn_pdl_wait();
            for (int i = 0; i < ahead; ++i) load_x((int)((begin + i) % a.stages), i);
            int place = ahead % L::RING, turn = ahead / L::RING;
            for (int64_t u = begin + ahead; u < end; ++u, forward()) {
                zn_bar_wait(&free_[place], (turn - 1) & 1, status, 31);
                load_w(tile, stage, place);
                load_x(stage, place);
                if (++place == L::RING) {
                    place = 0;
                    ++turn;
                }
            }
        }
        __syncwarp();
    } else if (warp == WARPS + 1) {
        // neighbouring lanes take neighbouring groups of a column, `per` of them in a stage, then the next columns
        constexpr int DEPTH_LOG = L::DEPTH == 4 ? 2 : 1;
        constexpr int per_log = DEPTH_LOG + 7 - GROUP_LOG;
        const int group0 = lane & ((1 << per_log) - 1), hop = 32 >> per_log;
        int place = 0, turn = 0, tile = (int)(begin / a.stages), stage = (int)(begin % a.stages);
        for (int64_t u = begin; u < end; ++u) {
            if (turn > 0) zn_bar_wait(&free_[place], (turn - 1) & 1, status, 33);
            float *to = reinterpret_cast<float *>(ring + place * L::STAGE + L::W + L::X) + lane;
            const int64_t group = ((int64_t)stage << per_log) + group0;
            int64_t col = (int64_t)tile * COLUMNS + (lane >> per_log);
            const float *from = a.scales + col * a.groups + group;
            for (int i = 0; i < COLUMNS / 32 << per_log; ++i) {
                const bool there = col < a.n && group < a.groups;
                zn_async_word(to, there ? from : a.scales, there);
                to += 32;
                col += hop;
                from += hop * a.groups;
            }
            zn_async_words_arrive(&full[place]);
            if (++place == L::RING) {
                place = 0;
                ++turn;
            }
            if (++stage == a.stages) {
                stage = 0;
                ++tile;
            }
        }
    } else {
        const int side = warp % SIDE, depth = warp / SIDE, g = lane >> 2, t = lane & 3;
        int place = 0, phase = 0;
        for (int64_t u = begin; u < end;) {
            const int tile = (int)(u / a.stages), first = (int)(u % a.stages), last = (int)min((int64_t)a.stages, first + (end - u));
            u += last - first;
            float total[TALL][TILES][4], sum[TALL][TILES][4];
#pragma unroll
            for (int j = 0; j < TALL; ++j)
#pragma unroll
                for (int q = 0; q < TILES; ++q)
#pragma unroll
                    for (int e = 0; e < 4; ++e) total[j][q][e] = 0.f;
            for (int s = first; s < last; ++s) {
                const int b = s * L::DEPTH + depth;
                zn_bar_wait(&full[place], phase, status, 32);
                if (b < a.blocks) {
                    const unsigned char *w = ring + place * L::STAGE + depth * (COLUMNS * 64) + (side * 16 * TALL + g) * 64 + t * 16;
                    const uint4 *x = reinterpret_cast<const uint4 *>(ring + place * L::STAGE + L::W + depth * (4 * TILES * 512)) + lane;
                    constexpr int log = 7 - GROUP_LOG, per = L::DEPTH << log;
                    // of this lane's four columns of w, 8 h + g of each tile of 16
                    const float *scale = reinterpret_cast<const float *>(ring + place * L::STAGE + L::W + L::X) + (side * 16 * TALL + g) * per + (depth << log);
                    uint4 word[TALL * 2];
#pragma unroll
                    for (int h = 0; h < TALL * 2; ++h) word[h] = *reinterpret_cast<const uint4 *>(w + h * 8 * 64);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint4 xb[TILES];
#pragma unroll
                        for (int q = 0; q < TILES; ++q) xb[q] = x[(i * TILES + q) * 32];
#pragma unroll
                        for (int j = 0; j < TALL; ++j) {
                            const uint4 &wl = word[2 * j], &wh = word[2 * j + 1];
                            const uint32_t lo = i == 0 ? wl.x : i == 1 ? wl.y : i == 2 ? wl.z : wl.w;
                            const uint32_t hi = i == 0 ? wh.x : i == 1 ? wh.y : i == 2 ? wh.z : wh.w;
                            const uint32_t l0 = code_pair(lo, 0), l1 = code_pair(lo, 1), l2 = code_pair(lo, 2), l3 = code_pair(lo, 3);
                            const uint32_t h0 = code_pair(hi, 0), h1 = code_pair(hi, 1), h2 = code_pair(hi, 2), h3 = code_pair(hi, 3);
#pragma unroll
                            for (int q = 0; q < TILES; ++q) mma_16x8(sum[j][q], l0, h0, l1, h1, xb[q].x, xb[q].y, ((i << 5) & ((1 << GROUP_LOG) - 1)) == 0);
#pragma unroll
                            for (int q = 0; q < TILES; ++q) mma_16x8(sum[j][q], l2, h2, l3, h3, xb[q].z, xb[q].w, false);
                        }
                        if ((((i + 1) << 5) & ((1 << GROUP_LOG) - 1)) == 0) {       // a group ends here
                            const int group = (i << 5) >> GROUP_LOG;
#pragma unroll
                            for (int j = 0; j < TALL; ++j) {
                                const float s0 = scale[16 * j * per + group], s1 = scale[(16 * j + 8) * per + group];
#pragma unroll
                                for (int q = 0; q < TILES; ++q) {
                                    total[j][q][0] = fmaf(s0, sum[j][q][0], total[j][q][0]);
                                    total[j][q][1] = fmaf(s0, sum[j][q][1], total[j][q][1]);
                                    total[j][q][2] = fmaf(s1, sum[j][q][2], total[j][q][2]);
                                    total[j][q][3] = fmaf(s1, sum[j][q][3], total[j][q][3]);
                                }
                            }
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) zn_bar_arrive(&free_[place]);
                if (++place == L::RING) {
                    place = 0;
                    phase ^= 1;
                }
            }
            float *mine = sums + warp * (16 * TALL) * L::PITCH;
#pragma unroll
            for (int j = 0; j < TALL; ++j)
#pragma unroll
                for (int q = 0; q < TILES; ++q)
#pragma unroll
                    for (int e = 0; e < 4; ++e) mine[(16 * j + 8 * (e >> 1) + g) * L::PITCH + 8 * q + 2 * t + (e & 1)] = total[j][q][e];
            zn_part_sync(WARPS * 32);
            // the warps along k and the parts of x, in a fixed order, the smallest parts first
            for (int i = threadIdx.x; i < COLUMNS * a.rows; i += WARPS * 32) {
                const int col = i % COLUMNS, row = i / COLUMNS;
                float part[3] = {0.f, 0.f, 0.f};
#pragma unroll
                for (int d = 0; d < L::DEPTH; ++d) {
                    const float *p = sums + ((d * SIDE + col / (16 * TALL)) * (16 * TALL) + col % (16 * TALL)) * L::PITCH + 3 * row;
#pragma unroll
                    for (int e = 0; e < 3; ++e) part[e] += p[e];
                }
                const float v = part[0] + (part[1] + part[2]);
                if (a.split > 1) reinterpret_cast<float *>(ring)[i] = v;       // nothing else is to come: the ring is done with
                else if (last - first == a.stages) finish(tile, i, v);
                else a.partial[(2 * (int64_t)blockIdx.x + (first == 0)) * (COLUMNS * a.rows) + i] = v;
            }
            if (a.split == 1 && last - first < a.stages) {
                // the blocks that share the tile: the first one left its sums at its second place, the others at their first
                const int64_t t0 = (int64_t)tile * a.stages, t1 = t0 + a.stages - 1;
                const int from = (int)(((t0 + 1) * gridDim.x - 1) / units), to = (int)(((t1 + 1) * gridDim.x - 1) / units);
                __threadfence();
                zn_part_sync(WARPS * 32);
                if (threadIdx.x == 0) {
                    joins = atomicAdd(&a.arrivals[from], 1u) == (unsigned)(to - from);
                    if (joins) a.arrivals[from] = 0u;
                }
                zn_part_sync(WARPS * 32);
                if (joins) {
                    __threadfence();
                    for (int i = threadIdx.x; i < COLUMNS * a.rows; i += WARPS * 32) {
                        float v = 0.f;
                        for (int b = from; b <= to; ++b) v += __ldcg(a.partial + (2 * (int64_t)b + (b == from)) * (COLUMNS * a.rows) + i);
                        finish(tile, i, v);
                    }
                }
            }
            zn_part_sync(WARPS * 32);
        }
    }
    if (a.split == 1) return;
    __syncwarp();
    zn_cluster_arrive();
    zn_cluster_wait();
    // each block of the cluster finishes its share of the tile, the stretches of k in their order
    const int outputs = COLUMNS * a.rows, lo = outputs * rank / a.split, hi = outputs * (rank + 1) / a.split, tile = blockIdx.x / a.split;
    for (int i = lo + threadIdx.x; i < hi; i += WARPS * 32 + 64) {
        float v = 0.f;
        for (int b = 0; b < a.split; ++b) {
            uint32_t remote;
            float p;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(zn_smem(ring + 4 * i)), "r"(b));
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(p) : "r"(remote) : "memory");
            v += p;
        }
        finish(tile, i, v);
    }
    __syncwarp();
    zn_cluster_arrive();             // until here the other blocks read this one's sums
    zn_cluster_wait();
}

}   // namespace

zn_token_plan zn_plan_quantize4(size_t n, size_t k, int sms) {
    zn_token_plan p;
    (void)sms;
    p.threads = TPB;
    p.blocks = (int64_t)((n + QUANT_COLUMNS - 1) / QUANT_COLUMNS * ((k + 127) / 128));
    return p;
}

zn_status zn_k_quantize4(zn_ctx *ctx, const float *w, uint32_t *packed, float *scales, size_t n, size_t k, size_t group) {
    const zn_token_plan p = zn_plan_quantize4(n, k, ctx->sm_count);
    if (p.blocks > 0x7fffffff) return zn_fail(ctx, ZN_ERR_SHAPE, "quantize4: %zu x %zu weights are too many for one launch", n, k);
    zn_launch_scope scope(ctx, ZN_PROF_CONVERT, 0, 4.5 * n * k);
    quantize_kernel<<<(unsigned)p.blocks, p.threads, 0, ctx->stream>>>(w, packed, scales, (int64_t)n, (int64_t)k, (int)group,
                                                                       (int64_t)((n + QUANT_COLUMNS - 1) / QUANT_COLUMNS));
    ZN_CUDA(ctx, cudaGetLastError());
    return ZN_OK;
}

namespace {

constexpr int ROWS_AT_ONCE = 16;

struct Shape {
    int tiles_x, warps, blocks, stages, tiles, split;
    int64_t grid;
    size_t smem, split_floats, scratch;
};
// Up to eight rows sixteen warps share the work; more rows need the registers of eight.
Shape shape_of(int64_t rows, int64_t n, int64_t k, int sms) {
    Shape s;
    s.tiles_x = (int)((3 * (rows < ROWS_AT_ONCE ? rows : ROWS_AT_ONCE) + 7) / 8);
    if (s.tiles_x < 1) s.tiles_x = 1;
    s.warps = s.tiles_x <= 3 ? 16 : 8;
    const int depth = s.warps / SIDE;
    s.blocks = (int)((k + 127) / 128);
    s.stages = (s.blocks + depth - 1) / depth;
    s.tiles = (int)((n + COLUMNS - 1) / COLUMNS);
    s.split = 1;
    while (s.split < 8 && s.tiles * s.split * 2 <= sms && s.split * 2 <= s.stages) s.split *= 2;
    s.grid = s.split > 1 ? (int64_t)s.tiles * s.split : s.tiles * (int64_t)s.stages < sms ? s.tiles * (int64_t)s.stages : sms;
    s.split_floats = (size_t)s.blocks * 4 * s.tiles_x * 32 * 4;
    s.scratch = s.split_floats + (s.split == 1 ? (size_t)s.grid * 2 * COLUMNS * (size_t)(rows < ROWS_AT_ONCE ? rows : ROWS_AT_ONCE) : 0);
    const auto smem = [](auto l) { return (size_t)(decltype(l)::RING * decltype(l)::STAGE + decltype(l)::SUMS); };
    switch (s.tiles_x) {
    case 1: s.smem = smem(Layout<1, 16>()); break;
    case 2: s.smem = smem(Layout<2, 16>()); break;
    case 3: s.smem = smem(Layout<3, 16>()); break;
    case 4: s.smem = smem(Layout<4, 8>()); break;
    case 5: s.smem = smem(Layout<5, 8>()); break;
    default: s.smem = smem(Layout<6, 8>());
    }
    return s;
}

typedef CUresult (*EncodeTiled)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The packed weights as words of a block, columns, blocks: a copy brings whole blocks of many columns, column by column.
zn_status weight_map(zn_ctx *ctx, CUtensorMap *map, const uint32_t *packed, int64_t n, int blocks, int depth) {
    const EncodeTiled encode = reinterpret_cast<EncodeTiled>(zn_tensor_map_encoder());
    if (!encode) return zn_fail(ctx, ZN_ERR_NOT_INITIALIZED, "cuTensorMapEncodeTiled is not available from the driver");
    const cuuint64_t dims[3] = {16, (cuuint64_t)n, (cuuint64_t)blocks}, strides[2] = {(cuuint64_t)blocks * 64, 64};
    const cuuint32_t box[3] = {16, COLUMNS, (cuuint32_t)depth}, ones[3] = {1, 1, 1};
    const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, const_cast<uint32_t *>(packed), dims, strides, box, ones,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return zn_fail(ctx, ZN_ERR_CUDA, "cuTensorMapEncodeTiled failed with %d", (int)r);
    return ZN_OK;
}

template <int TILES, int WARPS>
zn_status launch(zn_ctx *ctx, const CUtensorMap &map, const Product &p, const Shape &s, size_t group) {
    const auto kernel = group == 32 ? matmul4_kernel<TILES, WARPS, 5> : group == 64 ? matmul4_kernel<TILES, WARPS, 6> : matmul4_kernel<TILES, WARPS, 7>;
    ZN_CUDA(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)s.smem));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)s.grid);
    cfg.blockDim = dim3(WARPS * 32 + 64);
    cfg.dynamicSmemBytes = s.smem;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)s.split;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    ZN_CUDA(ctx, cudaLaunchKernelEx(&cfg, kernel, map, p, ctx->status_dev));
    return ZN_OK;
}

}   // namespace

zn_token_plan zn_plan_matmul4(size_t rows, size_t n, size_t k, int sms) {
    const Shape s = shape_of((int64_t)rows, (int64_t)n, (int64_t)k, sms);
    zn_token_plan p;
    p.threads = s.warps * 32 + 64;
    p.blocks = s.grid;
    p.share = s.split;
    p.smem = s.smem;
    p.scratch_floats = s.scratch;
    return p;
}

zn_status zn_k_matmul4(zn_ctx *ctx, const float *x, const uint32_t *packed, const float *scales, const float *bias, float *y,
                       size_t rows, size_t n, size_t k, size_t group, int act) {
    for (size_t r = 0; r < rows; r += ROWS_AT_ONCE) {
        const size_t now = rows - r < ROWS_AT_ONCE ? rows - r : (size_t)ROWS_AT_ONCE;
        const Shape s = shape_of((int64_t)now, (int64_t)n, (int64_t)k, ctx->sm_count);
        ZN_TRY(zn_scratch_reserve(ctx, s.scratch));
        unsigned int *arrivals = nullptr;
        if (s.split == 1) ZN_TRY(zn_lane_counters(ctx, &arrivals));      // one per block: fewer than the lane has
        CUtensorMap map;
        ZN_TRY(weight_map(ctx, &map, packed, (int64_t)n, s.blocks, s.warps / SIDE));
        uint4 *split = reinterpret_cast<uint4 *>(ctx->scratch);
        zn_launch_scope scope(ctx, ZN_PROF_GEMM_TC, 2.0 * now * n * k, 0.5 * n * k + 4.0 * n * k / group + 4.0 * now * (n + k), 2);
        const int64_t total = (int64_t)(s.split_floats / 4);
        int64_t blocks = (total + TPB - 1) / TPB;
        if (blocks > ctx->sm_count * 8) blocks = ctx->sm_count * 8;
        split_kernel<<<(unsigned)blocks, TPB, 0, ctx->stream>>>(x + r * k, split, (int)now, (int64_t)k, total, s.tiles_x);
        ZN_CUDA(ctx, cudaGetLastError());
        const Product p{split, scales, bias, y + r * n, ctx->scratch + s.split_floats, arrivals, (int64_t)n, (int64_t)((k + group - 1) / group), s.blocks, (int)now,
                        act, s.split, s.stages, s.tiles};
        switch (s.tiles_x) {
        case 1: ZN_TRY((launch<1, 16>(ctx, map, p, s, group))); break;
        case 2: ZN_TRY((launch<2, 16>(ctx, map, p, s, group))); break;
        case 3: ZN_TRY((launch<3, 16>(ctx, map, p, s, group))); break;
        case 4: ZN_TRY((launch<4, 8>(ctx, map, p, s, group))); break;
        case 5: ZN_TRY((launch<5, 8>(ctx, map, p, s, group))); break;
        default: ZN_TRY((launch<6, 8>(ctx, map, p, s, group)));
        }
    }
    return ZN_OK;
}
