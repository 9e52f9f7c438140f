// nc_beams.cuh -- beam search: selection over beams and vocabulary, and the reordering of states by parents.
//
// Selection.  A request has `beams` rows of logits and a score for each (-inf: no beam).  A live beam's candidates are
//   total(b, v) = score_b + x(b, v) - lse_b,   lse_b = M + log sum exp(x - M),
// a finished one's only candidate is its own token `end` at score_b.  The best `beams` by total / norm_b go on, among
// equals the lower beam, then (within a beam the larger logit, and among equal logits) the lower token.
//
// One pass over the logits of live beams, which bound it, as in nc_logprobs.cuh: CTAs stream segments of rows and keep the
// maxima of blocks, from which each segment's best k = min(beams, vocabulary) are found.  The last CTA of a row joins its
// segments, the last row of a request merges the rows' lists, each in order: beams steps of one warp, a lane to a row.  Rows that
// have no beam or have finished are not read.
//
// Accuracy.  Sums of a segment are float32, lse and totals 64-bit: totals of different beams may lie close together.
#pragma once

#include "nc_logprobs.cuh"

namespace nc {

constexpr int BEAM_STAGES = 4;                 // batches of a thread in flight, and the one in work
constexpr int BEAM_COPY_THREADS = 256, BEAM_COPY_VECS = 8;

struct BeamArgs {
    const char *logits;                // [rows][vocab], rows `stride` elements apart
    const float *scores, *norms;       // [rows]; norms may be null
    const int32_t *finished;           // [rows] or null
    int32_t *parent, *new_finished, *grow, *history;      // [rows]; all but parent may be null
    int64_t *tokens;                   // [rows]
    float *new_scores;                 // [rows]
    unsigned int *counter;             // [LP_ROWS] segments of rows, [LP_ROWS] rows of requests: zero before and after
    float2 *part;                      // [rows of a launch][segs]: M, S
    unsigned long long *part_top;      // [rows of a launch][segs][k]
    double *lse;                       // [rows of a launch]
    unsigned long long *best;          // [rows of a launch][k]
    unsigned long long *error;         // null, or the smallest live row whose log-sum is no number
    int64_t stride, vocab, row_first, end;
    int64_t seg_vecs;
    int beams, k, segs;
};

// Doubles in the order of their values, as unsigned numbers above 0; 0 for -inf and NaN.
__device__ __forceinline__ unsigned long long beam_order(double v) {
    if (!(v > -INFINITY)) return 0;
    const unsigned long long u = (unsigned long long)__double_as_longlong(v == 0.0 ? 0.0 : v);
    return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}
// The largest of the warp's values, in every lane.
__device__ __forceinline__ unsigned long long beam_warp_max(unsigned long long v) {
    const uint32_t high = __reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32));
    const uint32_t low = __reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32) == high ? (uint32_t)v : 0u);
    return (unsigned long long)high << 32 | low;
}

struct BeamSums {
    float m, s;
};
__device__ __forceinline__ BeamSums beam_join(const BeamSums &a, const BeamSums &b) {
    const float m = max_nan(a.m, b.m), to = m == -INFINITY ? 0.0f : m;
    return BeamSums{m, __fmaf_rn(a.s, lp_exp2((a.m - to) * LP_LOG2E), b.s * lp_exp2((b.m - to) * LP_LOG2E))};
}
__device__ __forceinline__ BeamSums beam_block_join(BeamSums v, LpSums *room) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const BeamSums w{__shfl_xor_sync(0xffffffffu, v.m, o), __shfl_xor_sync(0xffffffffu, v.s, o)};
        v = beam_join(v, w);
    }
    if ((threadIdx.x & 31) == 0) room[threadIdx.x >> 5] = LpSums{v.m, v.s, 0.0f};
    __syncthreads();
    v = BeamSums{room[0].m, room[0].s};
#pragma unroll
    for (int w = 1; w < LP_THREADS / 32; ++w) v = beam_join(v, BeamSums{room[w].m, room[w].s});
    return v;
}

struct BeamShared {
    LpShared lp;
    __align__(16) uint4 ring[BEAM_STAGES][LP_VECS][LP_THREADS];    // a thread's vectors are its own: no barrier
};

template <int TYPE>
__global__ void __launch_bounds__(LP_THREADS, 2) beam_select_kernel(const __grid_constant__ BeamArgs a) {
    constexpr int N = LpVec<TYPE>::N, SIZE = TYPE == KV_F32 ? 4 : 2;
    constexpr int64_t BATCH = LP_THREADS * LP_VECS;
    extern __shared__ __align__(16) char beam_smem[];
    BeamShared &shared = *reinterpret_cast<BeamShared *>(beam_smem);
    LpShared &sh = shared.lp;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    release_dependents();
    wait_for_producer();
    const int seg = (int)(blockIdx.x % a.segs);
    const int64_t local = blockIdx.x / a.segs, row = a.row_first + local;
    const bool there = a.scores[row] > -INFINITY || a.scores[row] != a.scores[row], ended = there && a.finished && a.finished[row] != 0;
    double lse = 0.0;
    if (!there || ended) {
        if (seg != 0) return;
    } else {
        const char *const base = a.logits + row * a.stride * SIZE;
        const int skew = (int)(((uintptr_t)base & 15) / SIZE);     // element e of the row is element e + skew of the vectors
        const char *const aligned = base - skew * SIZE;
        const int64_t seg0 = (int64_t)seg * a.seg_vecs, v_end = min(seg0 + a.seg_vecs, (a.vocab + skew + N - 1) / N);
        const int64_t v_low = skew ? 1 : 0, v_high = min(v_end, (a.vocab + skew) / N);       // whole vectors
        // Whole vectors come by asynchronous copies, others are put together; -inf past the segment's end.
        auto fetch = [&](int64_t first, int stage) {
#pragma unroll
            for (int i = 0; i < LP_VECS; ++i) {
                const int64_t v = first + tid + i * LP_THREADS;
                uint4 *const to = &shared.ring[stage][i][tid];
                if (v >= v_low && v < v_high) {
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(aligned + v * 16) : "memory");
                } else if (first < v_end) {
                    constexpr uint32_t none = TYPE == KV_F32 ? 0xff800000u : TYPE == KV_F16 ? 0xfc00fc00u : 0xff80ff80u;
                    *to = v < v_end ? lp_partial<TYPE>(base, v * N - skew, a.vocab) : make_uint4(none, none, none, none);
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        for (int i = 0; i < BEAM_STAGES - 1; ++i) fetch(seg0 + i * BATCH, i);
        BeamSums sum{-INFINITY, 0.0f};
        int batches = 0, stage = 0;
        for (int64_t first = seg0; first < v_end; first += BATCH, ++batches) {
            fetch(first + (BEAM_STAGES - 1) * BATCH, stage == 0 ? BEAM_STAGES - 1 : stage - 1);
            asm volatile("cp.async.wait_group %0;" ::"n"(BEAM_STAGES - 1) : "memory");
            uint4 raw[LP_VECS];
#pragma unroll
            for (int i = 0; i < LP_VECS; ++i) raw[i] = shared.ring[stage][i][tid];
            stage = stage == BEAM_STAGES - 1 ? 0 : stage + 1;
            float top = lp_vector_max<TYPE>(raw[0]);
#pragma unroll
            for (int i = 1; i < LP_VECS; ++i) top = max_nan(top, lp_vector_max<TYPE>(raw[i]));
            sh.block[batches][tid] = lp_order(top);
            if (top > sum.m || top != top) {                       // a larger value, or a NaN, which then stays the maximum
                sum.s *= lp_exp2((sum.m - top) * LP_LOG2E);
                sum.m = top;
            }
            const float to = sum.m == -INFINITY ? 0.0f : sum.m;
            const uint64_t unit = pack2(LP_LOG2E, LP_LOG2E), from = pack2(-to, -to);
            uint64_t s2 = pack2(sum.s, 0.0f);
#pragma unroll
            for (int i = 0; i < LP_VECS; ++i) {
                float x[N];
                lp_unpack<TYPE>(raw[i], x);
#pragma unroll
                for (int j = 0; j < N; j += 2) {
                    const float2 u = unpack2(mul2(add2(pack2(x[j], x[j + 1]), from), unit));
                    s2 = add2(s2, pack2(lp_exp2(u.x), lp_exp2(u.y)));
                }
            }
            const float2 s = unpack2(s2);
            sum.s = s.x + s.y;
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        lp_segment_top<TYPE>(a, sh, base, skew, seg0, v_end, batches, lp_order(sum.m));
        sum = beam_block_join(sum, sh.sums);
        if (a.segs > 1) {
            if (tid == 0) a.part[local * a.segs + seg] = make_float2(sum.m, sum.s);
            if (tid < a.k) a.part_top[(local * a.segs + seg) * a.k + tid] = sh.best[tid];
            __threadfence();
            __syncthreads();
            if (tid == 0) sh.arrived = atomicAdd(a.counter + local, 1u);
            __syncthreads();
            if (sh.arrived != (unsigned)a.segs - 1) return;
            __threadfence();
            if (tid == 0) {
                a.counter[local] = 0;
                sh.count = 0;
            }
            sum = BeamSums{-INFINITY, 0.0f};
            const unsigned long long *const tops = a.part_top + local * a.segs * a.k;
            unsigned long long head = 0, floor_key = 0;
            if (tid < a.segs) {
                const float2 p = __ldcg(a.part + local * a.segs + tid);
                sum = BeamSums{p.x, p.y};
                head = __ldcg(tops + tid * a.k);
                floor_key = __ldcg(tops + tid * a.k + a.k - 1);
                sh.heads[tid] = head;
            }
            sum = beam_block_join(sum, sh.sums);
            // A key below the k-th largest of the segments' best, or below a segment's own k-th best, has k better ones.
            if (tid < a.segs) {
                int rank = 0;
                for (int i = 0; i < a.segs; ++i) rank += sh.heads[i] > head;
                if (rank == a.k - 1 && head > floor_key) floor_key = head;
            }
            floor_key = lp_block_max(floor_key, sh.round);
            for (int i = tid; i < a.segs * a.k; i += LP_THREADS) {
                const unsigned long long key = __ldcg(tops + i);
                if (key != 0 && key >= floor_key) sh.cand[atomicAdd(&sh.count, 1)] = key;
            }
            if (tid < a.k) sh.best[tid] = 0;
            __syncthreads();
            lp_rank(sh.cand, sh.count, a.k, sh.best);
            __syncthreads();
        }
        lse = (double)sum.m + log((double)sum.s);                  // -inf where every logit is; then there are no candidates
        if (tid < a.k) a.best[local * a.k + tid] = sh.best[tid];
    }
    // The row is done; the last of its request goes on.
    const int64_t group = local / a.beams;
    if (tid == 0) a.lse[local] = lse;
    __threadfence();
    __syncthreads();
    if (tid == 0) sh.arrived = atomicAdd(a.counter + LP_ROWS + group, 1u);
    __syncthreads();
    if (sh.arrived != (unsigned)a.beams - 1) return;
    __threadfence();
    if (tid == 0) a.counter[LP_ROWS + group] = 0;
    const int64_t first = group * a.beams;
    for (int i = tid; i < a.beams * a.k; i += LP_THREADS) sh.cand[i] = __ldcg(a.best + first * a.k + i);
    __syncthreads();
    if (warp != 0) return;

    const int64_t mine = a.row_first + first + lane;               // a lane to a row
    double score = -INFINITY, norm = 1.0, row_lse = 0.0;
    bool done = true;
    int at = 0, count = 0;
    if (lane < a.beams) {
        score = (double)a.scores[mine];
        if (a.norms) norm = (double)a.norms[mine];
        done = a.finished && a.finished[mine] != 0;
        row_lse = __ldcg(a.lse + first + lane);
        count = done ? 1 : a.k;
        if (!(score > -INFINITY)) {
            if (score != score && a.error) atomicMin(a.error, (unsigned long long)mine);
            count = 0;
        } else if (!done && !(row_lse < INFINITY)) {               // a NaN or an infinity among the logits
            if (a.error) atomicMin(a.error, (unsigned long long)mine);
            count = 0;
        }
    }
    double total = 0.0;
    unsigned long long order = 0;
    int64_t token = 0;
    auto candidate = [&]() {                                       // the lane's next
        order = 0;
        if (at >= count) return;
        if (done) {
            total = score;
            token = a.end;
        } else {
            const unsigned long long key = sh.cand[lane * a.k + at];
            if (key == 0) return;
            total = score + ((double)lp_value((uint32_t)(key >> 32)) - row_lse);
            token = 0xffffffffu - (uint32_t)key;
        }
        order = beam_order(total / norm);
        ++at;
    };
    candidate();
    int parent = -1;
    double best = -INFINITY;
    int64_t chosen = a.end >= 0 ? a.end : 0;
    bool was = false;
    for (int i = 0; i < a.beams; ++i) {
        const unsigned long long most = beam_warp_max(order);
        if (most == 0) break;
        const int winner = __ffs(__ballot_sync(0xffffffffu, order == most)) - 1;
        const double w_total = __shfl_sync(0xffffffffu, total, winner);
        const long long w_token = __shfl_sync(0xffffffffu, (long long)token, winner);
        const bool w_done = __shfl_sync(0xffffffffu, (int)done, winner) != 0;
        if (lane == i) parent = winner, best = w_total, chosen = w_token, was = w_done;
        if (lane == winner) candidate();
    }
    if (lane < a.beams) {
        const bool over = parent < 0 || was || (a.end >= 0 && chosen == a.end);
        const int from = parent < 0 ? -1 : (int)(a.row_first + first) + parent;
        a.parent[mine] = from;
        a.tokens[mine] = chosen;
        a.new_scores[mine] = (float)best;
        if (a.new_finished) a.new_finished[mine] = over;
        if (a.grow) a.grow[mine] = parent >= 0 && !was;
        if (a.history) a.history[mine] = over ? -1 : from;
    }
}

// States.  Plane p of row i: the parent's first `length` lines (all of them without lengths), then one line of `append`.  Bytes are
// moved as they are, a chunk of eight vectors to a thread for each CTA, all of them asked for before the first is stored.
struct ReorderArgs {
    char *to;
    const char *from, *append;         // append: [rows][planes][line] or null
    const int32_t *parent, *lengths, *grow;   // [rows]; lengths and grow may be null
    int32_t *new_lengths;              // [rows] or null
    int64_t to_stride, from_stride, line;     // bytes of a row, of a line
    int rows, planes, capacity;
    int64_t chunks;                    // of a plane
};

template <typename V>
__global__ void __launch_bounds__(BEAM_COPY_THREADS) beam_reorder_kernel(const __grid_constant__ ReorderArgs a) {
    constexpr int64_t CHUNK = (int64_t)BEAM_COPY_THREADS * BEAM_COPY_VECS;
    const int tid = threadIdx.x;
    release_dependents();
    wait_for_producer();
    const int64_t chunk = blockIdx.x % a.chunks, unit = blockIdx.x / a.chunks;
    const int plane = (int)(unit % a.planes), i = (int)(unit / a.planes), parent = a.parent[i];
    const bool known = parent >= 0 && parent < a.rows, leads = chunk == 0;
    const int length = !known ? 0 : a.lengths ? min(max(a.lengths[parent], 0), a.capacity) : a.capacity;
    const bool more = known && a.append && length < a.capacity && (!a.grow || a.grow[i] != 0);
    if (leads && plane == 0 && tid == 0 && a.new_lengths) a.new_lengths[i] = length + more;
    if (!known) return;
    const int64_t plane_at = (int64_t)plane * a.capacity * a.line, vectors = length * a.line / (int64_t)sizeof(V);
    V *const to = (V *)(a.to + i * a.to_stride + plane_at);
    const V *const from = (const V *)(a.from + parent * a.from_stride + plane_at);
    const int64_t first = chunk * CHUNK + tid;
    V v[BEAM_COPY_VECS];
#pragma unroll
    for (int k = 0; k < BEAM_COPY_VECS; ++k)
        if (first + k * BEAM_COPY_THREADS < vectors) v[k] = from[first + k * BEAM_COPY_THREADS];
#pragma unroll
    for (int k = 0; k < BEAM_COPY_VECS; ++k)
        if (first + k * BEAM_COPY_THREADS < vectors) to[first + k * BEAM_COPY_THREADS] = v[k];
    if (!leads) return;
    // What whole vectors leave of the last line, and the line appended.
    char *const rest = (char *)to;
    for (int64_t at = vectors * (int64_t)sizeof(V) + tid; at < length * a.line; at += BEAM_COPY_THREADS) rest[at] = ((const char *)from)[at];
    if (more) {
        const char *const line = a.append + ((int64_t)i * a.planes + plane) * a.line;
        for (int64_t at = tid; at < a.line; at += BEAM_COPY_THREADS) rest[length * a.line + at] = line[at];
    }
}

}  // namespace nc
