// Embedding lookup with scaling and its gradient.
//
// The gradient is a sum of rows per token.  The positions are sorted by token first (a stable radix sort, so that a
// token's rows are added in the order of their positions), then fixed pieces of the sorted order are summed, however the
// tokens are distributed: one token in every position costs the same as all different ones.  A token whose run crosses
// pieces leaves partial sums, which a last kernel adds in their order.  Nothing is added by atomics.
//
// Both are bound by HBM.  Measured: 32,768 rows of 2048 looked up 73 us (5.0 TB/s of the distinct rows and the output); the
// whole gradient of a 50,001 x 1024 table from 16,384 rows 67 us (4.1 TB/s of rows read once and table written once), of
// which sort and first part of the clearing 21, sums and the rest of it 35, joins 10.
#include "zn_token.cuh"

namespace {

constexpr int TPB = 256;

template <bool VEC> struct Unit;
template <> struct Unit<true> {
    using type = float4;
    static __device__ __forceinline__ float4 zero() { return make_float4(0.f, 0.f, 0.f, 0.f); }
    static __device__ __forceinline__ float4 add(float4 a, float4 b) { return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w); }
    static __device__ __forceinline__ float4 mul(float s, float4 a) { return make_float4(s * a.x, s * a.y, s * a.z, s * a.w); }
    static __device__ __forceinline__ float4 from_above(float4 a, int o) {
        return make_float4(__shfl_down_sync(0xffffffffu, a.x, o), __shfl_down_sync(0xffffffffu, a.y, o), __shfl_down_sync(0xffffffffu, a.z, o),
                           __shfl_down_sync(0xffffffffu, a.w, o));
    }
};
template <> struct Unit<false> {
    using type = float;
    static __device__ __forceinline__ float zero() { return 0.f; }
    static __device__ __forceinline__ float add(float a, float b) { return a + b; }
    static __device__ __forceinline__ float mul(float s, float a) { return s * a; }
    static __device__ __forceinline__ float from_above(float a, int o) { return __shfl_down_sync(0xffffffffu, a, o); }
};

// A block takes `wide` units of 16 bytes of TPB / wide * ROWS rows; a thread has ROWS loads on their way.
template <int ROWS>
__global__ void __launch_bounds__(TPB) embed_kernel(const float *__restrict__ table, const int32_t *__restrict__ tokens, float *__restrict__ out,
                                                    int64_t rows, int64_t vocab, int64_t units, int wide, int cuts, float scale, int *status) {
    using U = Unit<true>;
    using T = float4;
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

// The form for rows that do not stand on 16 bytes: the output as one run of values, four of them a thread with one store,
// from whichever rows they fall in.
__global__ void __launch_bounds__(TPB) embed_flat_kernel(const float *__restrict__ table, const int32_t *__restrict__ tokens, float *__restrict__ out,
                                                         int64_t rows, int64_t vocab, int64_t dim, float scale, int *status) {
    constexpr int QUADS = 4;
    const int64_t total = rows * dim, lead = zn_aligned_from(out, total);
    const int64_t first = (int64_t)blockIdx.x * (TPB * QUADS * 4) - (4 - lead) % 4 + 4 * (int64_t)threadIdx.x;      // 16-byte places from here on
    float v[QUADS][4];
#pragma unroll
    for (int q = 0; q < QUADS; ++q) {
        const int64_t at = first + q * TPB * 4;
        int64_t r = at <= 0 ? 0 : total <= 0x7fffffff ? (int64_t)((uint32_t)at / (uint32_t)dim) : at / dim, c = (at <= 0 ? 0 : at) - r * dim;
        int64_t t = at < total ? __ldg(tokens + r) : -1;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[q][e] = 0.f;
            if (at + e < 0 || at + e >= total) continue;
            if (c == dim) {
                c = 0;
                t = __ldg(tokens + ++r);
            }
            if (t >= vocab && c == 0) zn_bad_token(status);
            if (t >= 0 && t < vocab) v[q][e] = scale * __ldg(table + t * dim + c);
            ++c;
        }
    }
#pragma unroll
    for (int q = 0; q < QUADS; ++q) {
        const int64_t at = first + q * TPB * 4;
        if (at >= 0 && at + 4 <= total) *reinterpret_cast<float4 *>(out + at) = make_float4(v[q][0], v[q][1], v[q][2], v[q][3]);
        else
            for (int e = 0; e < 4; ++e)
                if (at + e >= 0 && at + e < total) out[at + e] = v[q][e];
    }
}

// ---- sort ---------------------------------------------------------------------------------------------

constexpr int SORT_THREADS = 1024, SORT_WARPS = SORT_THREADS / 32, SORT_BLOCKS = 8, RADIX = 256;
constexpr int BATCH = 8;             // values of a lane on their way at once

struct SortArgs {
    const int32_t *tokens;
    int2 *buffer;                 // twice `rows` pairs of key and position
    float *table;                 // its first `clear` values are set to zero by the blocks that do not sort
    int64_t rows, vocab, clear;
    int passes, bits;
    int sorters;
};

// Sets this block's share (block `me` of `blocks`) of a run of values to zero.
__device__ __forceinline__ void clear_share(float *p, int64_t n, int64_t me, int64_t blocks) {
    const int64_t from = zn_aligned_from(p, n), vecs = (n - from) / 4, to = from + 4 * vecs, first = me * blockDim.x + threadIdx.x;
    float4 *q = reinterpret_cast<float4 *>(p + from);
    for (int64_t i = first; i < vecs; i += blocks * blockDim.x) q[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (first < from) p[first] = 0.f;
    if (first < n - to) p[to + first] = 0.f;
}

// Few positions: the place of each in the order by (token, position) is the number of positions before it, counted by a
// warp against all tokens in shared memory.  One launch without barriers between blocks, but work that grows with the
// square.  Measured, the whole gradient of 512-wide rows, counted against sorted: 777 positions 12.3 and 18.6 us, 2048 12.9
// and 20.6, 4096 20.2 and 22.7, 8192 39.0 and 26.8.
constexpr int COUNT_MOST = 4096, COUNT_THREADS = 512;
__global__ void __launch_bounds__(COUNT_THREADS) count_kernel(SortArgs a, int *status) {
    __shared__ __align__(16) uint32_t key[COUNT_MOST];
    zn_pdl_release();
    if (blockIdx.x >= a.sorters) {
        clear_share(a.table, a.clear, blockIdx.x - a.sorters, gridDim.x - a.sorters);
        return;
    }
    const int n = (int)a.rows, padded = (n + 127) / 128 * 128, lane = threadIdx.x & 31;
    for (int i = threadIdx.x; i < padded; i += COUNT_THREADS) {
        const int32_t t = i < n ? __ldg(a.tokens + i) : -1;
        if (t >= a.vocab && blockIdx.x == 0) zn_bad_token(status);
        key[i] = i >= n ? 0xffffffffu : t < 0 || t >= a.vocab ? (uint32_t)a.vocab : (uint32_t)t;
    }
    __syncthreads();
    for (int r = blockIdx.x * (COUNT_THREADS / 32) + (threadIdx.x >> 5); r < n; r += a.sorters * (COUNT_THREADS / 32)) {
        const uint32_t mine = key[r];
        int before = 0;
        for (int i = 4 * lane; i < padded; i += 128) {
            const uint4 k = *reinterpret_cast<const uint4 *>(key + i);
            before += (k.x < mine || (k.x == mine && i < r)) + (k.y < mine || (k.y == mine && i + 1 < r)) +
                      (k.z < mine || (k.z == mine && i + 2 < r)) + (k.w < mine || (k.w == mine && i + 3 < r));
        }
        before = __reduce_add_sync(0xffffffffu, before);
        if (lane == 0) {
            __stcg(a.buffer + before, make_int2((int)mine, r));
        }
    }
}

// One cluster of eight blocks sorts the positions by token, `bits` of it at a time, the lowest first; a position without a
// token counts as token `vocab` and comes last.  Every warp owns a stretch of the positions and keeps its own counts, so
// places follow from sums alone and equal tokens keep their order.  The other blocks of the launch clear the table
// meanwhile.  16,384 positions of 16 bits take 14 us, 65,536 of 17 bits 45: bound by the scattered stores of eight SMs and two
// cluster barriers a pass, and hidden behind the clearing where there is one.
__global__ void __launch_bounds__(SORT_THREADS) sort_kernel(SortArgs a, int *status) {
    zn_pdl_release();
    if (blockIdx.x >= SORT_BLOCKS) {
        clear_share(a.table, a.clear, blockIdx.x - SORT_BLOCKS, gridDim.x - SORT_BLOCKS);
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
        int2 *src = a.buffer + (pass & 1 ? 0 : a.rows), *dst = a.buffer + (pass & 1 ? a.rows : 0);
        const auto load = [&](int64_t i, uint32_t &key, int32_t &at) {
            if (pass == 0) {
                const int32_t t = __ldg(a.tokens + i);
                key = t < 0 || t >= a.vocab ? (uint32_t)a.vocab : (uint32_t)t;
                at = (int32_t)i;
            } else {
                const int2 v = __ldcg(src + i);
                key = (uint32_t)v.x;
                at = v.y;
            }
        };
        for (int i = threadIdx.x; i < SORT_WARPS * RADIX; i += SORT_THREADS) (&count[0][0])[i] = 0;
        __syncthreads();
        uint32_t key[BATCH];
        int32_t at[BATCH], place[BATCH];
        const auto load_batch = [&](int64_t i0) {
#pragma unroll
            for (int j = 0; j < BATCH; ++j)
                if (i0 + 32 * j < hi) load(i0 + 32 * j, key[j], at[j]);
        };
        const auto digit_of = [&](uint32_t k) { return (int)(k >> (pass * a.bits)) & (radix - 1); };
        // Places of a batch among the warp's values of the same digit, and on with the counts.  Lanes of the same digit find
        // each other by one vote per bit.
        const auto count_batch = [&](int64_t i0) {
#pragma unroll
            for (int j = 0; j < BATCH; ++j) {
                const bool here = i0 + 32 * j < hi;
                const int digit = here ? digit_of(key[j]) : 0;
                unsigned same = __ballot_sync(0xffffffffu, here);
                if (same == 0) break;
                for (int b = 0; b < a.bits; ++b) {
                    const unsigned ones = __ballot_sync(0xffffffffu, digit >> b & 1);
                    same &= digit >> b & 1 ? ones : ~ones;
                }
                if (here) place[j] = count[warp][digit] + __popc(same & ((1u << lane) - 1u));
                __syncwarp();
                if (here && lane == __ffs(same) - 1) count[warp][digit] += __popc(same);
                __syncwarp();
            }
        };
        for (int64_t i0 = lo + lane; i0 - lane < hi; i0 += 32 * BATCH) {
            load_batch(i0);
            if (pass == 0)
                for (int j = 0; j < BATCH; ++j)
                    if (i0 + 32 * j < hi && __ldg(a.tokens + i0 + 32 * j) >= a.vocab) zn_bad_token(status);
            count_batch(i0);
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
        // a stretch of one batch still has its keys and places; of a longer one they are formed again
        const bool held = stretch <= 32 * BATCH;
        for (int64_t i0 = lo + lane; i0 - lane < hi; i0 += 32 * BATCH) {
            if (!held) {
                load_batch(i0);
                count_batch(i0);
            }
#pragma unroll
            for (int j = 0; j < BATCH; ++j)
                if (i0 + 32 * j < hi) {
                    const int digit = digit_of(key[j]);
                    const int64_t to = (int64_t)base[digit] + (held ? count[warp][digit] : 0) + place[j];
                    __stcg(dst + to, make_int2((int)key[j], at[j]));
                }
        }
        zn_cluster_arrive();             // the next pass reads what all blocks wrote
        zn_cluster_wait();
    }
}

// ---- sums ---------------------------------------------------------------------------------------------

struct SumArgs {
    const float *grad;
    const int2 *sorted;           // tokens in their order, each with its position
    float *table;
    float *head, *tail;           // per piece: the sum of a run that began before it, of one that goes on behind it
    int64_t rows, vocab, units;
    int piece;
    int64_t pieces;
    float scale;
    int accumulate;
    int64_t clear_from, vocab_rows;   // table rows from here on have still to be cleared, but for those that get a sum
};

// The first place of the sorted order whose token is at least `token`, by one warp: 32 probes at a time.
__device__ int64_t first_at_least(const int2 *sorted, int64_t n, int64_t token) {
    int64_t lo = 0, hi = n;                           // the answer lies in [lo, hi]
    const int lane = threadIdx.x & 31;
    while (lo < hi) {
        const int64_t step = (hi - lo + 31) / 32, at = lo + step * lane;
        const unsigned below = __ballot_sync(0xffffffffu, at < hi && __ldcg(&sorted[at].x) < token);
        const int last = 31 - __clz(below);           // probes are in order: the ones below come first
        if (below == 0) return lo;
        const int64_t next = lo + step * (last + 1);
        lo = lo + step * last + 1;
        hi = min(hi, next);
    }
    return lo;
}

// Clears a share of the rows from a.clear_from on that have no token: a block takes CLEAR_ROWS at a time and marks those
// with one in shared memory first.
constexpr int CLEAR_ROWS = 32;
__device__ void clear_rows(const SumArgs &a, int64_t width, int64_t me, int64_t blocks) {
    __shared__ uint32_t mark[CLEAR_ROWS / 32];
    __shared__ int64_t range[2];
    for (int64_t row = a.clear_from + me * CLEAR_ROWS; row < a.vocab_rows; row += blocks * CLEAR_ROWS) {
        const int64_t end = min(a.vocab_rows, row + CLEAR_ROWS);
        __syncthreads();
        if (threadIdx.x < CLEAR_ROWS / 32) mark[threadIdx.x] = 0;
        if (threadIdx.x < 64) {
            const int64_t at = first_at_least(a.sorted, a.rows, threadIdx.x < 32 ? row : end);
            if ((threadIdx.x & 31) == 0) range[threadIdx.x >> 5] = at;
        }
        __syncthreads();
        for (int64_t i = range[0] + threadIdx.x; i < range[1]; i += TPB) {
            const int t = (int)(__ldcg(&a.sorted[i].x) - row);
            atomicOr(&mark[t >> 5], 1u << (t & 31));
        }
        __syncthreads();
        for (int64_t r = row + (threadIdx.x >> 5); r < end; r += TPB / 32) {
            if (mark[(r - row) >> 5] >> ((r - row) & 31) & 1) continue;
            float *p = a.table + r * width;
            const int64_t from = zn_aligned_from(p, width), vecs = (width - from) / 4, to = from + 4 * vecs, lane = threadIdx.x & 31;
            for (int64_t i = lane; i < vecs; i += 32) reinterpret_cast<float4 *>(p + from)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (lane < from) p[lane] = 0.f;
            if (lane < width - to) p[to + lane] = 0.f;
        }
    }
}

// A group of `wide` threads sums one piece of the sorted order, each thread one unit of the rows, eight rows on their way,
// and with them what the table holds at the rows that get their sum here.
template <bool VEC, bool ADD>
__device__ __forceinline__ void sum_piece(const SumArgs &a, int wide, int cuts) {
    using U = Unit<VEC>;
    using T = typename U::type;
    const int64_t c = (int64_t)(blockIdx.x % cuts) * wide + threadIdx.x % wide;
    const int64_t piece = (int64_t)(blockIdx.x / cuts) * (TPB / wide) + threadIdx.x / wide;
    if (c >= a.units || piece >= a.pieces) return;
    const int64_t lo = piece * a.piece, hi = min(a.rows, lo + a.piece);
    const T *g = reinterpret_cast<const T *>(a.grad);
    T *table = reinterpret_cast<T *>(a.table);
    const int32_t ahead = lo > 0 ? __ldcg(&a.sorted[lo - 1].x) : -1, behind = hi < a.rows ? __ldcg(&a.sorted[hi].x) : -1;
    bool continued = false, begun = false;
    T sum = U::zero();
    for (int64_t i0 = lo; i0 < hi; i0 += 8) {
        int32_t key[9], at[8];
        T v[8], old[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int2 s = i0 + j < hi ? __ldcg(a.sorted + i0 + j) : make_int2(-1, 0);
            key[j] = s.x;
            at[j] = s.y;
        }
        key[8] = i0 + 8 < hi ? __ldcg(&a.sorted[i0 + 8].x) : -1;
        // -1 and the count of tokens stand for none: nothing is read or written there
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const bool live = key[j] >= 0 && key[j] < a.vocab;
            v[j] = live ? __ldcs(g + at[j] * a.units + c) : U::zero();
            old[j] = ADD && live && key[j + 1] != key[j] ? table[key[j] * a.units + c] : U::zero();
        }
        if (!begun) {
            continued = key[0] == ahead;
            begun = true;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (key[j] < 0 || key[j] >= a.vocab) continue;
            sum = U::add(sum, v[j]);
            if (key[j + 1] == key[j]) continue;                      // the run goes on in this piece
            const bool last = i0 + j + 1 == hi;
            if (continued) reinterpret_cast<T *>(a.head)[piece * a.units + c] = sum;
            else if (last && behind == key[j]) reinterpret_cast<T *>(a.tail)[piece * a.units + c] = sum;
            else table[key[j] * a.units + c] = ADD ? U::add(old[j], U::mul(a.scale, sum)) : U::mul(a.scale, sum);
            continued = false;
            sum = U::zero();
        }
    }
}

template <bool VEC, bool ADD>
__global__ void __launch_bounds__(TPB, !VEC ? 4 : ADD ? 2 : 3) run_sum_kernel(SumArgs a, int wide, int cuts) {
    zn_pdl_release();
    zn_pdl_wait();
    // every block clears a share; half of them before their sums and half after, so that both go on at any time
    const bool clears = a.clear_from < a.vocab_rows, early = (blockIdx.x & 1) != 0;
    if (clears && early) clear_rows(a, a.units * (VEC ? 4 : 1), blockIdx.x, gridDim.x);
    sum_piece<VEC, ADD>(a, wide, cuts);
    if (clears && !early) clear_rows(a, a.units * (VEC ? 4 : 1), blockIdx.x, gridDim.x);
}

// A warp per piece, for up to 32 units of the rows.  Where a run begins in the piece and goes on behind it: its tail and
// the heads of the pieces that follow.  Narrow rows are taken by several groups of lanes, each every so-many-th head; a
// long run is left to all warps of the block in the same way.  The groups' sums are added in a fixed order.  (One warp for
// runs of up to 64 heads: 89 us for the gradient above instead of 70.)
constexpr int JOIN_LONG = 8;
template <bool VEC>
__global__ void __launch_bounds__(TPB) run_join_kernel(SumArgs a, int wide, int cuts) {
    using U = Unit<VEC>;
    using T = typename U::type;
    constexpr int WARPS = TPB / 32;
    __shared__ T sums[WARPS][32];
    __shared__ int64_t later[WARPS];
    zn_pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, side = lane % wide;
    const int64_t c = (int64_t)(blockIdx.x % cuts) * wide + side, piece0 = (int64_t)(blockIdx.x / cuts) * WARPS;
    const bool live = c < a.units;
    // the heads behind `piece`, from the `first`-th on, every `stride`-th; then over the warp's groups
    const auto add_heads = [&](int64_t piece, int64_t heads, int first, int stride) {
        T sum = U::zero();
        if (live) {
            const T *head = reinterpret_cast<const T *>(a.head) + (piece + 1) * a.units + c;
            for (int64_t i = first; i < heads; i += 8 * stride) {
                T v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = i + j * stride < heads ? __ldcg(head + (i + j * stride) * a.units) : U::zero();
#pragma unroll
                for (int j = 0; j < 8; ++j) sum = U::add(sum, v[j]);
            }
        }
        for (int o = 16; o >= wide; o /= 2) sum = U::add(sum, U::from_above(sum, o));
        return sum;
    };
    const auto put = [&](int64_t piece, T tail, T old, T sum) {
        const int64_t token = __ldcg(&a.sorted[(piece + 1) * a.piece - 1].x);
        if (lane < wide && live) reinterpret_cast<T *>(a.table)[token * a.units + c] = U::add(old, U::mul(a.scale, U::add(tail, sum)));
    };
    const auto old_of = [&](int64_t token) { return live && a.accumulate ? reinterpret_cast<const T *>(a.table)[token * a.units + c] : U::zero(); };
    const auto tail_of = [&](int64_t piece) { return live ? __ldcg(reinterpret_cast<const T *>(a.tail) + piece * a.units + c) : U::zero(); };
    if (lane == 0) later[warp] = 0;
    const int64_t piece = piece0 + warp, lo = piece * a.piece, hi = lo + a.piece;
    if (hi < a.rows) {
        const int32_t token = __ldcg(&a.sorted[hi - 1].x), behind = __ldcg(&a.sorted[hi].x), ahead = lo > 0 ? __ldcg(&a.sorted[lo - 1].x) : -1;
        if (token < a.vocab && behind == token && ahead != token) {
            int64_t heads = 0;                                               // pieces that begin with the token
            for (;;) {
                const int64_t p = piece + 1 + heads + lane;
                const int more = __popc(__ballot_sync(0xffffffffu, p < a.pieces && __ldcg(&a.sorted[p * a.piece].x) == token));
                heads += more;
                if (more < 32) break;
            }
            if (heads < JOIN_LONG) put(piece, tail_of(piece), old_of(token), add_heads(piece, heads, lane / wide, 32 / wide));
            else if (lane == 0) later[warp] = heads;
        }
    }
    __syncthreads();
    for (int w = 0; w < WARPS; ++w) {
        const int64_t heads = later[w];
        if (heads == 0) continue;
        sums[warp][lane] = add_heads(piece0 + w, heads, warp * (32 / wide) + lane / wide, WARPS * (32 / wide));
        __syncthreads();
        if (warp == 0) {
            T all = sums[0][lane];
            for (int i = 1; i < WARPS; ++i) all = U::add(all, sums[i][lane]);
            put(piece0 + w, tail_of(piece0 + w), old_of(__ldcg(&a.sorted[(piece0 + w + 1) * a.piece - 1].x)), all);
        }
        __syncthreads();
    }
}

// Threads side by side on one row: the power of two that covers its units, `most` at most.
int width_of(int64_t units, int most) {
    int wide = 1;
    while (wide < most && wide < units) wide *= 2;
    return wide;
}
// Values of the table cleared beside the sort, and beside the counting: about what those launches leave time for.  (All of
// it beside the sort: 77 us for the gradient above instead of 70.)
constexpr size_t CLEAR_FIRST = (size_t)24 << 20, CLEAR_FIRST_COUNT = (size_t)4 << 20;
bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Rows of the sorted order per piece: so many that about two thousand threads per SM have one, eight at least.
constexpr int64_t MOST_IN_PIECE = 1 << 20;
int64_t piece_of(int64_t rows, int64_t units, int sms) {
    const int64_t piece = (rows * units / ((int64_t)sms * 2048) + 7) / 8 * 8;
    return piece < 8 ? 8 : piece < MOST_IN_PIECE ? piece : MOST_IN_PIECE;
}

}   // namespace

zn_token_plan zn_plan_embedding_forward(size_t rows, size_t dim, int sms) {
    zn_token_plan p;
    (void)sms;
    p.threads = TPB;
    if (dim % 4 == 0) {
        const int wide = width_of((int64_t)dim / 4, TPB);
        const int64_t per = TPB / wide * 4;
        p.share = (int)((dim / 4 + wide - 1) / wide);
        p.blocks = ((int64_t)rows + per - 1) / per * p.share;
    } else {
        p.blocks = (int64_t)((rows * dim + 3 + TPB * 16 - 1) / (TPB * 16));
    }
    return p;
}

zn_status zn_k_embedding_forward(zn_ctx *ctx, const float *table, const int32_t *tokens, float *out, size_t rows, size_t vocab,
                                 size_t dim, float scale) {
    const bool vec = dim % 4 == 0 && aligned16(table) && aligned16(out);
    const zn_token_plan p = zn_plan_embedding_forward(rows, dim, ctx->sm_count);
    const int64_t flat = (int64_t)((rows * dim + 3 + TPB * 16 - 1) / (TPB * 16)), blocks = vec ? p.blocks : flat;
    if (blocks > 0x7fffffff) return zn_fail(ctx, ZN_ERR_SHAPE, "embedding_forward: %zu x %zu values are too many for one launch", rows, dim);
    zn_launch_scope scope(ctx, ZN_PROF_ELEMENTWISE, (double)rows * dim, 8.0 * rows * dim);
    if (vec)
        embed_kernel<4><<<(unsigned)blocks, TPB, 0, ctx->stream>>>(table, tokens, out, (int64_t)rows, (int64_t)vocab, (int64_t)dim / 4,
                                                                   width_of((int64_t)dim / 4, TPB), p.share, scale, ctx->status_dev);
    else
        embed_flat_kernel<<<(unsigned)blocks, TPB, 0, ctx->stream>>>(table, tokens, out, (int64_t)rows, (int64_t)vocab, (int64_t)dim, scale,
                                                                     ctx->status_dev);
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
    const bool count = rows <= COUNT_MOST;
    SortArgs s{tokens, reinterpret_cast<int2 *>(ctx->scratch), grad_table, (int64_t)rows, (int64_t)vocab, 0, 0, 0, 0};
    int key_bits = 1;
    while (((int64_t)vocab >> key_bits) != 0) ++key_bits;
    s.passes = count ? 1 : (key_bits + 7) / 8;
    s.bits = (key_bits + s.passes - 1) / s.passes;
    // The table is cleared in two parts: beside the sort what can be written meanwhile (about CLEAR_FIRST values), whatever
    // those rows will hold; beside the sums the rest, where it is known which rows get one.
    const int64_t first_rows = accumulate ? 0 : (int64_t)(vocab * dim <= (count ? CLEAR_FIRST_COUNT : CLEAR_FIRST) ? vocab : (count ? CLEAR_FIRST_COUNT : CLEAR_FIRST) / dim);
    s.clear = first_rows * (int64_t)dim;
    // 16-byte units where every row allows them
    const bool vec = dim % 4 == 0 && aligned16(grad_out) && aligned16(grad_table);
    SumArgs a{};
    a.units = (int64_t)(vec ? dim / 4 : dim);
    a.piece = (int)piece_of((int64_t)rows, (int64_t)(dim % 4 == 0 ? dim / 4 : dim), ctx->sm_count);
    a.pieces = ((int64_t)rows + a.piece - 1) / a.piece;
    const int64_t row_pad = ((int64_t)rows + 3) / 4 * 4, dim_pad = ((int64_t)dim + 3) / 4 * 4;
    a.grad = grad_out; a.sorted = s.buffer + (!count && (s.passes - 1) & 1 ? (int64_t)rows : 0); a.table = grad_table;
    a.head = ctx->scratch + 4 * row_pad; a.tail = a.head + a.pieces * dim_pad;
    a.rows = (int64_t)rows; a.vocab = (int64_t)vocab; a.scale = scale; a.accumulate = accumulate ? 1 : 0;
    const int wide = width_of(a.units, TPB), join_wide = width_of(a.units, 32);
    const int64_t cuts = (a.units + wide - 1) / wide, join_cuts = (a.units + join_wide - 1) / join_wide;
    const int64_t sum_blocks = (a.pieces + TPB / wide - 1) / (TPB / wide) * cuts, join_blocks = (a.pieces + TPB / 32 - 1) / (TPB / 32) * join_cuts;
    if (sum_blocks > 0x7fff0000 || join_blocks > 0x7fffffff)
        return zn_fail(ctx, ZN_ERR_SHAPE, "embedding_backward: %zu x %zu values are too many for one launch", rows, dim);
    a.clear_from = accumulate ? (int64_t)vocab : first_rows;
    a.vocab_rows = (int64_t)vocab;
    // where there are fewer sums than that, more blocks come for the clearing alone
    int64_t late = accumulate ? 0 : ((int64_t)vocab - first_rows + CLEAR_ROWS - 1) / CLEAR_ROWS;
    if (late > 4 * ctx->sm_count) late = 4 * ctx->sm_count;
    zn_launch_scope scope(ctx, ZN_PROF_ELEMENTWISE, 2.0 * rows * dim, 4.0 * rows * dim + 4.0 * (accumulate ? 2 * rows : vocab) * dim, 3);
    const auto blocks_to_clear = [&](int threads, int64_t most) {
        const int64_t want = (s.clear / 4 + 4 * threads - 1) / (4 * threads);
        return want < most ? want : most;
    };
    if (count) {
        const int64_t want = ((int64_t)rows + COUNT_THREADS / 32 - 1) / (COUNT_THREADS / 32);
        s.sorters = (int)(want < 2 * ctx->sm_count ? want : 2 * ctx->sm_count);
        const int64_t blocks = s.sorters + blocks_to_clear(COUNT_THREADS, 4 * ctx->sm_count);
        count_kernel<<<(unsigned)blocks, COUNT_THREADS, 0, ctx->stream>>>(s, ctx->status_dev);
        ZN_CUDA(ctx, cudaGetLastError());
    } else {
        const int64_t clear_blocks = (blocks_to_clear(SORT_THREADS, 2 * ctx->sm_count - SORT_BLOCKS) + SORT_BLOCKS - 1) / SORT_BLOCKS * SORT_BLOCKS;
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
    }
    const dim3 sums((unsigned)(sum_blocks > late ? sum_blocks : late)), joins((unsigned)join_blocks), block(TPB);
    if (vec) {
        ZN_CUDA(ctx, zn_launch_pdl(accumulate ? run_sum_kernel<true, true> : run_sum_kernel<true, false>, sums, block, 0, ctx->stream, a, wide, (int)cuts));
        ZN_CUDA(ctx, zn_launch_pdl(run_join_kernel<true>, joins, block, 0, ctx->stream, a, join_wide, (int)join_cuts));
    } else {
        ZN_CUDA(ctx, zn_launch_pdl(accumulate ? run_sum_kernel<false, true> : run_sum_kernel<false, false>, sums, block, 0, ctx->stream, a, wide, (int)cuts));
        ZN_CUDA(ctx, zn_launch_pdl(run_join_kernel<false>, joins, block, 0, ctx->stream, a, join_wide, (int)join_cuts));
    }
    return ZN_OK;
}
