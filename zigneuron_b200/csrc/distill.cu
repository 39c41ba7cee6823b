// Distillation from a teacher's top logits: loss and gradient of a row in one pass over it.
//
// The row is read from HBM once and the gradient written once.  A cluster of blocks holds a row, each block a slice of it,
// and goes from row to row.  In a block a ring of buffers keeps the next rows on their way (bulk copies) while one is
// worked on.  Each thread takes its values of the slice to registers and turns them into exponentials against its own
// maximum, so that one exponential per value does for the sums and the gradient both; every warp sends its maximum and
// sum to all blocks of the row through distributed shared memory; the gradient, a product per value, goes back to the
// buffer, and from there out by a bulk copy.  What is slow and small -- the teacher's entries, the listed tokens, the
// loss -- is left to helper warps.
//
// Bound by HBM: 4096 rows of 131,072 take 744 us (5.8 TB/s of read and write, 0.88 of a copy; clusters of eight leave 20 of
// 148 SMs without work), 1024 of 32,000 48 us.  What held it back on the way: the row read twice 2658 us, blocks that load,
// wait and store by themselves 1230, a barrier of the whole cluster per row 1183, each value's exponential formed twice 1011,
// the teacher's entries read when their place was free 897.
#include "zn_token.cuh"

namespace {

constexpr int MAX_SHARE = 8, MAX_RING = 3, MAX_WARPS = 16;
constexpr int HELD = 36;                         // values of a slice that a thread holds in registers

struct Shared {
    float part[MAX_WARPS][2];                    // maximum and sum of every warp
    float slice[2][MAX_SHARE][2];                // and of every block of the row; rows take turns
    float ends[MAX_RING][8];                     // the values before and behind the aligned part of the slice
    float weight[MAX_RING], loss_q[MAX_RING];    // sum q log q of the row in this place of the ring
    int state[MAX_RING];                         // what the teacher's entries leave of it
    float m[MAX_RING], s[MAX_RING];              // what the row comes to
    int verdict[MAX_RING], copy_out[MAX_RING];   // the gradient stands in the ring and goes out by a copy
    uint64_t full[MAX_RING], done[MAX_RING], free_[MAX_RING], met[2];
};
enum { FILL_GRADIENT = 0, FILL_ZERO = 1, FILL_NAN = 2, FILL_EMPTY = 3 };
enum { ROW_FINE = 0, ROW_NONE = 1, ROW_WRONG = 2, ROW_NAN = 3 };     // nothing to learn; id past the vocabulary; NaN among the logits

// A lane's share of 128 of the teacher's entries.  Their reads depend on one another (an entry, then the student's logit
// there) and are slow while the rows stream by, so they are started a row ahead.
struct Entries {
    int32_t id[4];
    float u[4], x[4];
};
__device__ __forceinline__ void load_ids(Entries &e, const zn_distill_args &a, int64_t r, int j0, int lane) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int j = j0 + lane + 32 * i;
        e.id[i] = j < a.k ? __ldg(a.ids + r * a.k + j) : -1;
        e.u[i] = j < a.k ? __ldg(a.teacher + r * a.k + j) : -INFINITY;
    }
}
__device__ __forceinline__ void load_logits(Entries &e, const zn_distill_args &a, int64_t r) {
#pragma unroll
    for (int i = 0; i < 4; ++i) e.x[i] = e.id[i] >= 0 && e.id[i] < a.vocab && e.u[i] != -INFINITY ? a.logits[r * a.ld + e.id[i]] : 0.f;
}

// The teacher's entries of a row, by one warp: q = softmax(u / T) over them, the student's logits at their tokens.  The
// first 128 have been loaded.
__device__ void read_teacher(const zn_distill_args &a, int64_t r, Entries e, int lane, float *q, float *xt, int32_t *id, float *together,
                             float *loss_q, int *state, bool report, int *status) {
    const float inv_t = 1.f / a.temperature;
    float um = -INFINITY;
    bool wrong = false, nan = false;
    for (int j0 = 0; j0 < a.k; j0 += 128) {
        if (j0 > 0) {
            load_ids(e, a, r, j0, lane);
            load_logits(e, a, r);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int j = j0 + lane + 32 * i;
            const bool entry = e.id[i] >= 0 && e.u[i] != -INFINITY, fine = entry && e.id[i] < a.vocab;
            wrong = wrong || (entry && !fine);
            nan = nan || (entry && !(e.u[i] < INFINITY));
            if (entry) um = fmaxf(um, e.u[i]);
            if (j < a.k) {
                id[j] = fine ? e.id[i] : -1;
                xt[j] = e.x[i];
                q[j] = e.u[i];
            }
        }
    }
    um = zn_warp_max(um);
    wrong = __any_sync(0xffffffffu, wrong);
    nan = __any_sync(0xffffffffu, nan);
    if (wrong && report && lane == 0) zn_bad_token(status);
    const float c = 1.4426950408889634f * inv_t;
    float mass = 0.f;
    for (int j = lane; j < a.k; j += 32)
        if (id[j] >= 0) mass += zn_exp2((q[j] - um) * c);
    mass = zn_warp_sum(mass);
    const float inv_mass = 1.f / mass, log_mass = logf(mass);
    float lq = 0.f;
    for (int j = lane; j < a.k; j += 32) {
        const float d = q[j] - um, p = id[j] >= 0 ? zn_exp2(d * c) * inv_mass : 0.f;
        if (p > 0.f) lq += p * (d * inv_t - log_mass);
        q[j] = p;
    }
    lq = zn_warp_sum(lq);
    __syncwarp();
    // The first place of an id takes the q of all its places, in their order; the others are taken out.  Few rows list an
    // id twice, so the sums are formed where one is found only.
    for (int j0 = 0; j0 < a.k; j0 += 32) {
        const int j = j0 + lane;
        const int32_t mine = j < a.k ? id[j] : -1;
        int same = 0;
#pragma unroll 8
        for (int i = 0; i < a.k; ++i) same += id[i] == mine;
        float sum = mine >= 0 ? q[j] : -1.f;
        if (mine >= 0 && same > 1) {
            int before = 0;
            sum = 0.f;
            for (int i = 0; i < a.k; ++i)
                if (id[i] == mine) {
                    before += i < j;
                    sum += q[i];
                }
            if (before > 0) sum = -1.f;
        }
        if (j < a.k) together[j] = sum;
    }
    if (lane == 0) {
        *loss_q = lq;
        *state = wrong ? ROW_WRONG : nan ? ROW_NAN : um == -INFINITY ? ROW_NONE : ROW_FINE;
    }
}

// n values of one kind.
template <int THREADS>
__device__ __forceinline__ void fill_slice(float *g, int n, float v) {
    const int from = (int)zn_aligned_from(g, n), vecs = (n - from) / 4, to = from + 4 * vecs;
    for (int i = threadIdx.x; i < vecs; i += THREADS) __stcs(reinterpret_cast<float4 *>(g + from + 4 * i), make_float4(v, v, v, v));
    if (threadIdx.x < from) g[threadIdx.x] = v;
    if (threadIdx.x < n - to) g[to + threadIdx.x] = v;
}

// THREADS of arithmetic and five warps around them: one starts the copies in, one finishes rows and sends them out, and one
// per place of the ring reads the teacher's entries (a chain of dependent reads and small sums, some microseconds long).
// REGS: a slice fits in the threads' registers; else each value's exponential is formed twice.  WHOLE: it fits on chip;
// else what does not is read twice.
template <int THREADS, bool REGS, bool WHOLE>
__global__ void __launch_bounds__(THREADS + 64 + 32 * MAX_RING) distill_kernel(zn_distill_args a, int share, int slice, int keep, int ring, int *status) {
    extern __shared__ __align__(16) float dynamic[];       // ring x (keep + 4) logits, then ring x k of q, x, id, together
    __shared__ Shared s;
    constexpr int WARPS = THREADS / 32;
    const int rank = (int)(blockIdx.x % share), lane = threadIdx.x & 31;
    const int64_t cluster = blockIdx.x / share, clusters = gridDim.x / share;
    const int64_t lo = min((int64_t)rank * slice, a.vocab);
    const int n = (int)(min(a.vocab, lo + slice) - lo);
    const int pitch = keep + 4;
    float *teacher = dynamic + ring * pitch;
    const float inv_t = 1.f / a.temperature, c = 1.4426950408889634f * inv_t;
    if (threadIdx.x == 0) {
        for (int i = 0; i < ring; ++i) {
            zn_bar_init(&s.full[i], 3);
            zn_bar_init(&s.done[i], WARPS);
            zn_bar_init(&s.free_[i], 1);
        }
        zn_bar_init(&s.met[0], 1);
        zn_bar_init(&s.met[1], 1);
        zn_bar_init_done();
    }
    __syncthreads();
    zn_cluster_arrive();         // every block has started before another one writes to its shared memory
    zn_cluster_wait();
    // The aligned part of the slice that fits on chip, from `from` on, `vecs` times four values; the ring holds it at the
    // same place modulo 16 bytes.
    const auto lay_out = [&](int64_t r, const float *&x, int &from, int &vecs, float *&mine, int place) {
        x = a.logits + r * a.ld + lo;
        from = (int)zn_aligned_from(x, n);
        vecs = max(0, (min(n, keep) - from) / 4);
        mine = dynamic + place * pitch + ((4 - from) & 3);
    };
    // the gradient at a listed token
    const auto at_token = [&](float x, float m, float inv_s, float wt, float q) {
        const float e = m == -INFINITY ? 0.f : zn_exp2(__fmul_rn(x - m, c));
        return __fmul_rn(wt, __fmaf_rn(e, inv_s, -q));
    };
    const float *x;
    float *mine;
    int from, vecs;

    if (threadIdx.x >= THREADS) {
        const int helper = (threadIdx.x - THREADS) >> 5;
        int place = 0, turn = 0;
        Entries entries;
        if (helper < ring && cluster + helper * clusters < a.rows) {
            load_ids(entries, a, cluster + helper * clusters, 0, lane);
            load_logits(entries, a, cluster + helper * clusters);
        }
        for (int64_t r = cluster; r < a.rows; r += clusters) {
            float *q = teacher + place * 4 * a.k, *xt = q + a.k, *together = q + 3 * a.k;
            int32_t *id = reinterpret_cast<int32_t *>(q + 2 * a.k);
            if (helper == place) {
                const int64_t after = r + ring * clusters;
                const Entries now = entries;
                if (after < a.rows) load_ids(entries, a, after, 0, lane);
                if (turn > 0) zn_bar_wait(&s.free_[place], (turn - 1) & 1, status, 21);
                read_teacher(a, r, now, lane, q, xt, id, together, &s.loss_q[place], &s.state[place], rank == 0, status);
                __syncwarp();
                if (lane == 0) zn_bar_arrive(&s.full[place]);
                if (after < a.rows) load_logits(entries, a, after);
            } else if (helper == MAX_RING) {
                if (turn > 0) zn_bar_wait(&s.free_[place], (turn - 1) & 1, status, 21);
                lay_out(r, x, from, vecs, mine, place);
                const float w = a.weights ? a.weights[r] : 1.f;
                if (lane == 0) {
                    const uint32_t bytes = w == 0.f ? 0u : 16u * (uint32_t)vecs;
                    zn_bar_expect(&s.full[place], bytes);
                    // in four pieces, so that several copies are under way at once
                    const uint32_t part = ((bytes + 63) / 64) * 16;
                    for (uint32_t at = 0; at < bytes; at += part)
                        zn_bulk_load(reinterpret_cast<char *>(mine + from) + at, reinterpret_cast<const char *>(x + from) + at, min(part, bytes - at),
                                     &s.full[place]);
                    s.weight[place] = w;
                }
                const int to = from + 4 * vecs, at = lane < 4 ? lane : to + lane - 4;
                if (lane < 8) s.ends[place][lane] = w != 0.f && (lane < 4 ? at < from : at < n) ? x[at] : -INFINITY;
                __syncwarp();
                if (lane == 0) zn_bar_arrive(&s.full[place]);
            } else if (helper == MAX_RING + 1) {
                lay_out(r, x, from, vecs, mine, place);
                zn_bar_wait(&s.done[place], turn & 1, status, 24);
                const float m = s.m[place], sum = s.s[place], w = s.weight[place], wt = w * a.temperature;
                const int verdict = s.verdict[place], to = from + 4 * vecs;
                float *g = a.grad ? a.grad + r * a.ld_grad + lo : nullptr;
                if (g && (verdict == FILL_GRADIENT || verdict == FILL_EMPTY)) {
                    // the listed tokens of this slice; an id's first place has the q of all its places
                    const float inv_s = verdict == FILL_EMPTY ? 0.f : 1.f / sum;
                    for (int j = lane; j < a.k; j += 32) {
                        const int64_t col = id[j] - lo;
                        if (together[j] < 0.f || col < 0 || col >= n) continue;
                        const float v = at_token(xt[j], m, inv_s, wt, together[j]);
                        if (s.copy_out[place] && col >= from && col < to) mine[col] = v;
                        else g[col] = v;
                    }
                }
                // the values were written by ordinary stores, here and by the threads that arrived: the copy sees them after this
                zn_async_fence();
                __syncwarp();
                if (lane == 0 && s.copy_out[place]) zn_bulk_store(g + from, mine + from, 16u * (uint32_t)vecs);
                if (a.loss && rank == 0) {
                    // sum q (log q - log p) = sum q log q - sum q log p
                    const float ls = logf(sum);
                    float lp = 0.f;
                    for (int j = lane; j < a.k; j += 32)
                        if (q[j] > 0.f) lp += q[j] * (m == -INFINITY ? -INFINITY : (xt[j] - m) * inv_t - ls);
                    lp = zn_warp_sum(lp);
                    if (lane == 0)
                        a.loss[r] = verdict == FILL_ZERO ? (w != 0.f && s.state[place] == ROW_WRONG ? zn_nan() : 0.f)
                                    : verdict == FILL_NAN ? zn_nan() : wt * a.temperature * (s.loss_q[place] - lp);
                }
                __syncwarp();
                if (lane == 0) {
                    zn_bulk_store_read();
                    zn_bar_arrive(&s.free_[place]);
                }
            }
            if (++place == ring) {
                place = 0;
                ++turn;
            }
        }
        __syncwarp();
    } else {
        int place = 0, phase = 0, side = 0, side_phase = 0;
        for (int64_t r = cluster; r < a.rows; r += clusters) {
            lay_out(r, x, from, vecs, mine, place);
            const int on_chip = from + 4 * vecs;
            zn_bar_wait(&s.full[place], phase, status, 22);
            const int state = s.state[place];
            const float w = s.weight[place];
            // up to eight values outside the aligned part; -inf where there are fewer
            const float end = threadIdx.x < 8 && w != 0.f ? s.ends[place][threadIdx.x] : -INFINITY;
            float v[REGS ? HELD : 1];
            zn_softmax st{-INFINITY, 0.f, 0.f};
            if (REGS) {
#pragma unroll
                for (int j = 0; j < HELD / 4; ++j) {
                    const int i = threadIdx.x + j * THREADS;
                    float4 f = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                    if (i < vecs && w != 0.f) f = *reinterpret_cast<const float4 *>(mine + from + 4 * i);
                    v[4 * j] = f.x; v[4 * j + 1] = f.y; v[4 * j + 2] = f.z; v[4 * j + 3] = f.w;
                    st.m = fmaxf(st.m, fmaxf(fmaxf(f.x, f.y), fmaxf(f.z, f.w)));
                }
                st.m = fmaxf(st.m, end);
                const float base = st.m == -INFINITY ? 0.f : st.m;
                float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < HELD; ++j) {
                    if (j / 4 * THREADS >= vecs) break;                // no thread has more
                    v[j] = zn_exp2(__fmul_rn(v[j] - base, c));
                    part[j & 3] += v[j];
                }
                st.s = (part[0] + part[1]) + (part[2] + part[3]) + zn_exp2(__fmul_rn(end - base, c));
            } else if (w != 0.f) {
                int i = threadIdx.x;
                for (; i + 3 * THREADS < vecs; i += 4 * THREADS) {
                    float u[16];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float4 f = *reinterpret_cast<const float4 *>(mine + from + 4 * (i + j * THREADS));
                        u[4 * j] = f.x; u[4 * j + 1] = f.y; u[4 * j + 2] = f.z; u[4 * j + 3] = f.w;
                    }
                    zn_softmax_add<16, false>(st, u, zn_largest(u), c);
                }
                for (; i < vecs; i += THREADS) {
                    const float4 f = *reinterpret_cast<const float4 *>(mine + from + 4 * i);
                    const float u[4] = {f.x, f.y, f.z, f.w};
                    zn_softmax_add<4, false>(st, u, zn_largest(u), c);
                }
                const float u[1] = {end};
                zn_softmax_add<1, false>(st, u, u[0], c);
                if (!WHOLE)         // up to four of them are in `ends` already
                    for (int j = on_chip + 4 + threadIdx.x; j < n; j += THREADS) {
                        const float o[1] = {x[j]};
                        zn_softmax_add<1, false>(st, o, o[0], c);
                    }
            }
            // over the warp, over the block by its first warp, which sends what they come to to every block of the row
            const float own_m = st.m;
            zn_softmax_raise<false>(st, zn_warp_max(st.m), c);
            st.s = zn_warp_sum(st.s);
            if (lane == 0) {
                s.part[threadIdx.x >> 5][0] = st.m;
                s.part[threadIdx.x >> 5][1] = st.s;
            }
            zn_part_sync(THREADS);
            if (threadIdx.x < 32) {
                zn_softmax all{-INFINITY, 0.f, 0.f};
                if (lane < WARPS) all = {s.part[lane][0], s.part[lane][1], 0.f};
                zn_softmax_raise<false>(all, zn_warp_max(all.m), c);
                all.s = zn_warp_sum(all.s);
                if (lane == 0) zn_bar_expect(&s.met[side], 8u * (uint32_t)share);
                if (lane < share) zn_cluster_send(s.slice[side][rank], all.m, all.s, &s.met[side], lane);
            }
            zn_bar_wait(&s.met[side], side_phase, status, 23);       // from here on nobody still needs the logits in global memory
            zn_softmax row{-INFINITY, 0.f, 0.f};
            if (lane < share) row = {s.slice[side][lane][0], s.slice[side][lane][1], 0.f};
            const float m = zn_warp_max(row.m);
            zn_softmax_raise<false>(row, m, c);
            float sum = row.s;
#pragma unroll
            for (int o = MAX_SHARE / 2; o > 0; o /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            sum = __shfl_sync(0xffffffffu, sum, 0);
            side_phase ^= side;
            side ^= 1;
            const int verdict = w == 0.f || state == ROW_NONE || state == ROW_WRONG ? FILL_ZERO
                                : !(sum >= 0.f) || state == ROW_NAN ? FILL_NAN : m == -INFINITY ? FILL_EMPTY : FILL_GRADIENT;
            float *g = a.grad ? a.grad + r * a.ld_grad + lo : nullptr;
            const bool copy_out = WHOLE && g && verdict == FILL_GRADIENT && vecs > 0 && ((reinterpret_cast<uintptr_t>(g + from)) & 15) == 0;
            if (threadIdx.x == 0) {
                s.m[place] = m;
                s.s[place] = sum;
                s.verdict[place] = verdict;
                s.copy_out[place] = copy_out;
            }
            if (g && verdict == FILL_GRADIENT) {
                const float f = __fmul_rn(w * a.temperature, 1.f / sum);
                const auto p = [&](float u) { return __fmul_rn(f, zn_exp2(__fmul_rn(u - m, c))); };
                if (REGS) {
                    const float fe = __fmul_rn(f, zn_exp2(own_m == m ? 0.f : __fmul_rn(own_m - m, c)));
#pragma unroll
                    for (int j = 0; j < HELD / 4; ++j) {
                        const int i = threadIdx.x + j * THREADS;
                        if (i < vecs)
                            *reinterpret_cast<float4 *>(mine + from + 4 * i) =
                                make_float4(__fmul_rn(fe, v[4 * j]), __fmul_rn(fe, v[4 * j + 1]), __fmul_rn(fe, v[4 * j + 2]), __fmul_rn(fe, v[4 * j + 3]));
                    }
                } else {
#pragma unroll 4
                    for (int i = threadIdx.x; i < vecs; i += THREADS) {
                        float4 *at = reinterpret_cast<float4 *>(mine + from + 4 * i);
                        const float4 u = *at;
                        *at = make_float4(p(u.x), p(u.y), p(u.z), p(u.w));
                    }
                    if (!WHOLE)
                        for (int j = on_chip + 4 + threadIdx.x; j < n; j += THREADS) g[j] = p(x[j]);
                }
                if (threadIdx.x < 8) {
                    const int at = threadIdx.x < 4 ? threadIdx.x : on_chip + threadIdx.x - 4;
                    if (threadIdx.x < 4 ? at < from : at < n) g[at] = p(end);
                }
                if (!copy_out) {
                    // the two blocks do not stand alike: neighbouring lanes take neighbouring values
                    zn_part_sync(THREADS);
#pragma unroll 4
                    for (int i = from + threadIdx.x; i < on_chip; i += THREADS) __stcs(g + i, mine[i]);
                }
            } else if (g) {
                fill_slice<THREADS>(g, n, verdict == FILL_NAN ? zn_nan() : 0.f);
            }
            __syncwarp();
            if (lane == 0) zn_bar_arrive(&s.done[place]);
            if (++place == ring) {
                place = 0;
                phase ^= 1;
            }
        }
    }
    __syncwarp();
    zn_cluster_arrive();         // a block's shared memory may be written by another one until both are here
    zn_cluster_wait();
}

// Blocks per row, values of a slice on chip, places in the ring, and threads.  A row is cut into as few slices as leave
// room for three of them in a block, eight at most (two places in the ring: 621 instead of 457 us for 2048 rows of 131,072);
// larger vocabularies get a shorter ring, and what does not fit even once is read a second time.  (Clusters of sixteen,
// which would hold twice the vocabulary in registers: 592 us for 1024 rows of 200,003 against 472.)  Where there are fewer
// rows than SMs they are spread over more blocks, down to 2048 values each.
constexpr size_t SMEM = 227 * 1024 - sizeof(Shared) - 64;
struct Plan {
    int share, slice, keep, ring, threads;
    size_t smem;
};
Plan distill_plan(int64_t rows, int64_t vocab, int64_t k, int sms) {
    Plan p;
    const auto smem = [&](int64_t keep, int ring) { return (size_t)ring * (size_t)(4 * (keep + 4) + 16 * k); };
    const auto slice_of = [&](int share) { return ((vocab + share - 1) / share + 3) / 4 * 4; };
    p.share = 1;
    while (p.share < MAX_SHARE && (smem(slice_of(p.share), MAX_RING) > SMEM || (rows * p.share * 2 <= sms && slice_of(p.share) > 4096))) p.share *= 2;
    p.slice = (int)slice_of(p.share);
    p.ring = MAX_RING;
    while (p.ring > 1 && smem(p.slice, p.ring) > SMEM) --p.ring;
    p.keep = p.slice;
    if (smem(p.keep, 1) > SMEM) p.keep = (int)((SMEM - 16 * k) / 4 - 8) / 4 * 4;
    p.threads = 64;
    while (p.threads < 512 && p.slice > p.threads * HELD) p.threads *= 2;
    p.smem = smem(p.keep, p.ring);
    return p;
}

template <int THREADS, bool REGS, bool WHOLE>
zn_status launch(zn_ctx *ctx, const zn_distill_args &a, const Plan &p) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)p.share);
    cfg.blockDim = dim3(THREADS + 64 + 32 * MAX_RING);
    cfg.dynamicSmemBytes = p.smem;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)p.share;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    // as many clusters as the GPU holds at once go from row to row
    int &fit = ctx->cluster_fit[{(size_t)(4 * THREADS + 2 * REGS + WHOLE), (size_t)p.share, p.smem}];
    if (fit == 0) {
        ZN_CUDA(ctx, cudaFuncSetAttribute(distill_kernel<THREADS, REGS, WHOLE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM));
        ZN_CUDA(ctx, cudaOccupancyMaxActiveClusters(&fit, distill_kernel<THREADS, REGS, WHOLE>, &cfg));
        if (fit < 1) fit = 1;
    }
    const int clusters = fit > a.rows ? (int)a.rows : fit;
    cfg.gridDim = dim3((unsigned)(clusters * p.share));
    zn_launch_scope scope(ctx, ZN_PROF_LOSS, 6.0 * a.rows * a.vocab, (a.grad ? 8.0 : 4.0) * a.rows * a.vocab);
    ZN_CUDA(ctx, cudaLaunchKernelEx(&cfg, distill_kernel<THREADS, REGS, WHOLE>, a, p.share, p.slice, p.keep, p.ring, ctx->status_dev));
    return ZN_OK;
}

}   // namespace

zn_token_plan zn_plan_distill(size_t rows, size_t vocab, size_t k, int sms) {
    const Plan d = distill_plan((int64_t)rows, (int64_t)vocab, (int64_t)k, sms);
    zn_token_plan p;
    p.threads = d.threads + 64 + 32 * MAX_RING;
    p.share = d.share;
    p.blocks = (rows < (size_t)sms ? (int64_t)rows : sms) * d.share;       // at most; the launch asks how many fit at once
    p.smem = d.smem;
    return p;
}

zn_status zn_k_distill(zn_ctx *ctx, const zn_distill_args &a) {
    const Plan p = distill_plan(a.rows, a.vocab, a.k, ctx->sm_count);
    if (p.keep < p.slice) return launch<512, false, false>(ctx, a, p);
    if (p.slice > p.threads * HELD) return launch<512, false, true>(ctx, a, p);
    switch (p.threads) {
    case 512: return launch<512, true, true>(ctx, a, p);
    case 256: return launch<256, true, true>(ctx, a, p);
    case 128: return launch<128, true, true>(ctx, a, p);
    default: return launch<64, true, true>(ctx, a, p);
    }
}
