// nc_beams.cuh -- beam search: selection over beams and vocabulary, and the reordering of states by parents.
//
// Selection.  A request has `beams` rows of logits and a score for each (-inf: no beam).  A live beam's candidates are
//   total(b, v) = score_b + x(b, v) - lse_b,   lse_b = M + log sum exp(x - M),
// a finished one's only candidate is its own token `end` at score_b.  The best `beams` by total / norm_b go on, among
// equals the lower beam, then (within a beam the larger logit, and among equal logits) the lower token.
//
// One pass over the logits of live beams, which bound it.  Rows without a live beam are not read; the others are one stream of
// batches, of which each CTA has an equal share: parts of one row or several, in segments of up to 16 batches.  As in nc_logprobs.cuh the
// CTA keeps the maxima of blocks, and finds from them each segment's best k = min(beams, vocabulary), with the next segment's first
// batch on its way.  The last CTA of a request's part of the stream joins its segments: the rows' log-sums, a warp to a row; where
// there are many candidates the lists with the first `beams` heads alone; then those that reach a bound, ranked.
//
// 32 requests of 8 beams over 151936 float32 logits: 36 us (3.5 TB/s of 6.5 over the rows that are live), bound by the latency of loads with
// 24 warps on an SM and by the segments' best; 48 of 16 over 50257 bfloat16 logits 43 us, bound by instructions (19 M of warps for 36 M
// logits, 48% of the issue slots) and barriers; one request of 4 beams 13 us, the join's chain of steps most of it.
//
// Accuracy.  Sums of a segment are float32, lse and totals 64-bit: totals of different beams may lie close together.
#pragma once

#include "nc_logprobs.cuh"

namespace nc {

constexpr int BEAM_RESIDENT = 3, BEAM_CTAS = 148 * BEAM_RESIDENT;     // CTAs on an SM, and that there is room for at once
constexpr int BEAM_WARPS = LP_THREADS / 32;
constexpr int BEAM_BATCH = LP_THREADS * LP_VECS;       // vectors
constexpr int BEAM_BATCHES = 16;               // of a segment at most: their maxima are kept
constexpr int BEAM_ROWS = 1024;                // of a launch at most
constexpr int BEAM_LISTS = 512;               // segments of a request at most
constexpr int BEAM_COPY_THREADS = 256, BEAM_COPY_VECS = 8;

struct BeamArgs {
    const char *logits;                // [rows][vocab], rows `stride` elements apart
    const float *scores, *norms;       // [rows]; norms may be null
    const int32_t *finished;           // [rows] or null
    int32_t *parent, *new_finished, *grow, *history;      // [rows]; all but parent may be null
    int64_t *tokens;                   // [rows]
    float *new_scores;                 // [rows]
    unsigned int *counter;             // [BEAM_ROWS] CTAs that are done with requests: zero before and after
    float2 *part;                      // [rows of a launch][lists]: M, S
    unsigned long long *part_top;      // [rows of a launch][lists][k]
    unsigned long long *error;         // null, or the smallest live row whose log-sum is no number
    int64_t stride, vocab, row_first, end;
    int rows, beams, k;                // rows: of the launch
    int lists, batches, least;         // segments of a row at most; batches of a row; of a CTA's share at least
};

// What each CTA has of the stream, in batches, and how a row is cut by that: its first segment is what is left of the share that its
// beginning lies in.
struct BeamShare {
    int size, batches;
    __device__ __forceinline__ static int pieces(int n) { return (n + BEAM_BATCHES - 1) / BEAM_BATCHES; }
    // Segments of the row at `entry` of the stream before the one at batch `at` of the row (all of them for at = batches).
    __device__ __forceinline__ int before(int entry, int at) const {
        const int first = min(size - entry * batches % size, batches);                    // of the share that the row begins in
        if (at < first) return at / BEAM_BATCHES;
        const int rest = at - first, whole = rest / size;
        return pieces(first) + whole * pieces(size) + (at == batches ? pieces(rest - whole * size) : (rest - whole * size) / BEAM_BATCHES);
    }
};

// Doubles in the order of their values, as unsigned numbers above 0; 0 for -inf and NaN.
__device__ __forceinline__ unsigned long long beam_order(double v) {
    if (!(v > -INFINITY)) return 0;
    const unsigned long long u = (unsigned long long)__double_as_longlong(v == 0.0 ? 0.0 : v);
    return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}
struct BeamSums {
    float m, s;
};
__device__ __forceinline__ BeamSums beam_join(const BeamSums &a, const BeamSums &b) {
    const float m = max_nan(a.m, b.m), to = m == -INFINITY ? 0.0f : m;
    return BeamSums{m, __fmaf_rn(a.s, lp_exp2((a.m - to) * LP_LOG2E), b.s * lp_exp2((b.m - to) * LP_LOG2E))};
}
__device__ __forceinline__ BeamSums beam_warp_join(BeamSums v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const BeamSums w{__shfl_xor_sync(0xffffffffu, v.m, o), __shfl_xor_sync(0xffffffffu, v.s, o)};
        v = beam_join(v, w);
    }
    return v;
}

// A candidate: larger totals first (`order`, 0: none), then lower rows, then larger keys.
struct BeamHead {
    unsigned long long order, key;
    int row;
};
__device__ __forceinline__ bool beam_before(const BeamHead &a, const BeamHead &b) {
    return a.order != b.order ? a.order > b.order : a.row != b.row ? a.row < b.row : a.key > b.key;
}
// How many of the n candidates come before each: four neighbouring threads share one.  orders(i) and get(i) are of the i-th; calls use(i,
// before) in one of them.  Orders that are equal, which are few, are looked at again.
template <typename O, typename G, typename F>
__device__ __forceinline__ void beam_ranks(int n, O orders, G get, F use) {
    const int part = threadIdx.x & 3;
    for (int base = 0; base < n; base += LP_THREADS / 4) {
        const int i = base + (threadIdx.x >> 2);
        const unsigned long long mine = orders(min(i, n - 1));
        int before = 0, equal = 0;
#pragma unroll 8
        for (int j = part; j < n; j += 4) {
            const unsigned long long other = orders(j);
            before += other > mine;
            equal += other == mine;
        }
        before += __shfl_xor_sync(0xffffffffu, before, 1);
        before += __shfl_xor_sync(0xffffffffu, before, 2);
        equal += __shfl_xor_sync(0xffffffffu, equal, 1);
        equal += __shfl_xor_sync(0xffffffffu, equal, 2);
        if (equal > 1) {
            const BeamHead h = get(min(i, n - 1));
            int more = 0;
            for (int j = part; j < n; j += 4)
                if (orders(j) == mine) more += beam_before(get(j), h);
            const uint32_t four = 0xfu << (threadIdx.x & 28);
            more += __shfl_xor_sync(four, more, 1);
            more += __shfl_xor_sync(four, more, 2);
            before += more;
        }
        if (part == 0 && i < n) use(i, before);
    }
}

// LpShared with fewer batches.
struct BeamSegment {
    uint32_t block[BEAM_BATCHES][LP_THREADS];
    uint32_t group_max[32];
    LpSums sums[BEAM_WARPS];
    unsigned long long cand[LP_CAND], best[LP_MAX_TOP], round[BEAM_WARPS], heads[LP_SEGS];
    int count, greater, equal;
    uint32_t kth;
};
// What the choice needs.
struct BeamRoom {
    unsigned long long order[LP_MAX_TOP * LP_MAX_TOP], key[LP_MAX_TOP * LP_MAX_TOP], group_most[128], bound;
    double lse[LP_MAX_TOP], score[LP_MAX_TOP], norm[LP_MAX_TOP], total[LP_MAX_TOP];
    int64_t token[LP_MAX_TOP];
    int state[LP_MAX_TOP], parent[LP_MAX_TOP], segs[LP_MAX_TOP];   // state: 0 no beam, 1 live, 2 finished
    uint16_t list[BEAM_LISTS], chosen[LP_MAX_TOP];                 // lists whose heads reach the bound; those of the first `beams` heads
    uint8_t row[LP_MAX_TOP * LP_MAX_TOP];                          // of the candidates
    int count, found, most;
};
static_assert(BEAM_LISTS <= LP_MAX_TOP * LP_MAX_TOP, "heads lie where the candidates do");
struct BeamShared {
    union {
        BeamSegment segment;
        BeamRoom room;
    };
    uint16_t live[BEAM_ROWS];                                      // rows to be read
    uint16_t done[BEAM_ROWS], first[BEAM_ROWS];                    // requests that were this CTA's to choose for, where their live rows begin
    uint8_t rows[BEAM_ROWS];                                       // and how many these are
    int counts[BEAM_WARPS], ndone;
};

__device__ __forceinline__ int beam_state(const BeamArgs &a, int64_t row) {
    const float s = a.scores[row];
    return s == -INFINITY ? 0 : a.finished && a.finished[row] != 0 ? 2 : 1;
}

// A bound that at least k of the threads' values `most` reach, and about as many of all (0: fewer than k are above 0): the k-th largest of
// the values of 32 groups of threads, or of 128.  For all threads; room.group_most is free again after the caller's next barrier.
__device__ __forceinline__ unsigned long long beam_bound(BeamRoom &room, unsigned long long most, int k) {
    const int tid = threadIdx.x;
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
    if (k <= 8) {
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 4));
    }
    const int groups = k <= 8 ? 32 : 128, of = LP_THREADS / groups;
    if (tid % of == 0) room.group_most[tid / of] = most;
    __syncthreads();
    if (tid < groups) {
        const unsigned long long mine = room.group_most[tid];
        int rank = 0;
#pragma unroll 16
        for (int j = 0; j < groups; ++j) {
            const unsigned long long other = room.group_most[j];
            rank += other > mine || (other == mine && j < tid);
        }
        if (rank == k - 1) room.bound = mine;
    }
    __syncthreads();
    return max(1ull, room.bound);
}

// A request's choice, by all threads of a CTA, when its segments are done.  `entry`: where its `live` rows are in the stream.
__device__ __noinline__ void beam_choose(const BeamArgs &a, BeamShared &shared, int group, int entry, int live, BeamShare share) {
    constexpr int MOST = LP_MAX_TOP * LP_MAX_TOP, MINE = MOST / LP_THREADS, HEADS = BEAM_LISTS / LP_THREADS;
    BeamRoom &room = shared.room;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, k = a.k;
    const int64_t first = (int64_t)group * a.beams, row0 = a.row_first + first;
    const unsigned long long *const tops = a.part_top + first * a.lists * k;
    // Everything is asked for before the first is used, but for what the lists' number is needed for.
    float row_score[LP_MAX_TOP / BEAM_WARPS], row_norm[LP_MAX_TOP / BEAM_WARPS];
    int ended[LP_MAX_TOP / BEAM_WARPS];
#pragma unroll
    for (int i = 0; i < LP_MAX_TOP / BEAM_WARPS; ++i) {
        const int r = warp + i * BEAM_WARPS;
        row_score[i] = r < a.beams ? a.scores[row0 + r] : -INFINITY;
        row_norm[i] = r < a.beams && a.norms ? a.norms[row0 + r] : 1.0f;
        ended[i] = r < a.beams && a.finished ? a.finished[row0 + r] : 0;
    }
    if (warp == 0) {
        if (lane < a.beams) room.segs[lane] = 0;
        __syncwarp();
        const int segs = lane < live ? share.before(entry + lane, a.batches) : 0, most = __reduce_max_sync(0xffffffffu, segs);
        if (lane < live) room.segs[shared.live[entry + lane] - first] = segs;
        if (lane < a.beams) {
            room.parent[lane] = -1;
            room.total[lane] = -INFINITY;
        }
        if (lane == 0) {
            room.most = max(most, 1);
            room.count = room.found = 0;
        }
    }
    __syncthreads();
    const int segs = room.most, lists = a.beams * segs;            // as many for every row, some empty
    const bool all = lists * k <= MOST;                            // few enough candidates to take them all
    auto list_key = [&](int list, int at) {
        const int r = list / segs, seg = list - r * segs;
        return seg < room.segs[r] ? __ldcg(tops + ((int64_t)r * a.lists + seg) * k + at) : 0;
    };
    unsigned long long key[MINE];
#pragma unroll
    for (int m = 0; m < MINE; ++m) {
        const int i = tid + m * LP_THREADS;
        key[m] = all ? i < lists * k ? list_key(i / k, i % k) : 0 : m < HEADS && i < lists ? list_key(i, 0) : 0;
    }
#pragma unroll
    for (int i = 0; i < LP_MAX_TOP / BEAM_WARPS; ++i) {
        const int r = warp + i * BEAM_WARPS, state = row_score[i] == -INFINITY ? 0 : ended[i] != 0 ? 2 : 1;
        if (r >= a.beams) break;
        BeamSums sum{-INFINITY, 0.0f};
        for (int j = lane; j < room.segs[r]; j += 32) {
            const float2 p = __ldcg(a.part + (first + r) * a.lists + j);
            sum = beam_join(sum, BeamSums{p.x, p.y});
        }
        sum = beam_warp_join(sum);
        if (lane == 0) {
            const double score = (double)row_score[i], lse = state == 1 ? (double)sum.m + log((double)sum.s) : 0.0;      // -inf where every logit is: no candidate
            // A NaN or an infinity among the logits, or no score.
            const bool bad = state != 0 && (score != score || (state == 1 && !(lse < INFINITY)));
            if (bad && a.error) atomicMin(a.error, (unsigned long long)(row0 + r));
            room.state[r] = bad ? 0 : state;
            room.score[r] = score;
            room.norm[r] = (double)row_norm[i];
            room.lse[r] = lse;
        }
    }
    __syncthreads();
    auto total = [&](int r, unsigned long long v) { return room.score[r] + ((double)lp_value((uint32_t)(v >> 32)) - room.lse[r]); };
    auto order_at = [&](int list, int at, unsigned long long v) {  // of a list's candidate
        const int r = list / segs, state = room.state[r];
        if (state == 2) {                                          // its only candidate, in its first list
            if (list != r * segs || at != 0) return 0ull;
            return beam_order(a.norms ? room.score[r] / room.norm[r] : room.score[r]);
        }
        if (state == 0 || v == 0) return 0ull;
        return beam_order(a.norms ? total(r, v) / room.norm[r] : total(r, v));
    };
    int on = lists;
    if (!all) {                                                    // the lists with the first `beams` heads
        unsigned long long head[HEADS], most = 0;
#pragma unroll
        for (int m = 0; m < HEADS; ++m) {
            const int list = tid + m * LP_THREADS;
            head[m] = list < lists ? order_at(list, 0, key[m]) : 0;
            most = max(most, head[m]);
        }
        const unsigned long long bound = beam_bound(room, most, a.beams);
#pragma unroll
        for (int m = 0; m < HEADS; ++m)
            if (head[m] >= bound) {
                const int to = atomicAdd(&room.count, 1);
                room.order[to] = head[m];
                room.key[to] = key[m];
                room.list[to] = (uint16_t)(tid + m * LP_THREADS);
            }
        __syncthreads();
        on = min(room.count, a.beams);
        beam_ranks(
            room.count, [&](int i) { return room.order[i]; }, [&](int i) { return BeamHead{room.order[i], room.key[i], room.list[i] / segs}; },
            [&](int i, int before) {
                if (before < a.beams) room.chosen[before] = room.list[i];
            });
        __syncthreads();
#pragma unroll
        for (int m = 0; m < MINE; ++m) {
            const int i = tid + m * LP_THREADS;
            key[m] = i < on * k ? list_key(room.chosen[i / k], i % k) : 0;
        }
    }
    unsigned long long order[MINE], most = 0;
#pragma unroll
    for (int m = 0; m < MINE; ++m) {
        const int i = tid + m * LP_THREADS;
        order[m] = 0;
        if (i < on * k) order[m] = order_at(all ? i / k : room.chosen[i / k], i % k, key[m]);
        most = max(most, order[m]);
    }
    const unsigned long long bound = beam_bound(room, most, a.beams);
#pragma unroll
    for (int m = 0; m < MINE; ++m) {
        const int i = tid + m * LP_THREADS;
        if (order[m] < bound) continue;
        const int to = atomicAdd(&room.found, 1);
        room.order[to] = order[m];
        room.key[to] = key[m];
        room.row[to] = (uint8_t)((all ? i / k : room.chosen[i / k]) / segs);
    }
    __syncthreads();
    beam_ranks(
        room.found, [&](int i) { return room.order[i]; }, [&](int i) { return BeamHead{room.order[i], room.key[i], room.row[i]}; },
        [&](int i, int before) {
            if (before >= a.beams) return;
            const int r = room.row[i];
            const bool was = room.state[r] == 2;
            room.parent[before] = r;
            room.token[before] = was ? a.end : (int64_t)(0xffffffffu - (uint32_t)room.key[i]);
            room.total[before] = was ? room.score[r] : total(r, room.key[i]);
        });
    __syncthreads();
    if (tid < a.beams) {
        const int r = room.parent[tid];
        const int64_t token = r < 0 ? max(a.end, (int64_t)0) : room.token[tid], row = row0 + tid;
        const bool was = r >= 0 && room.state[r] == 2, over = r < 0 || was || (a.end >= 0 && token == a.end);
        const int from = r < 0 ? -1 : (int)row0 + r;
        a.parent[row] = from;
        a.tokens[row] = token;
        a.new_scores[row] = (float)room.total[tid];
        if (a.new_finished) a.new_finished[row] = over;
        if (a.grow) a.grow[row] = r >= 0 && !was;
        if (a.history) a.history[row] = over ? -1 : from;
    }
    __syncthreads();
}

template <int TYPE>
__global__ void __launch_bounds__(LP_THREADS, BEAM_RESIDENT) beam_select_kernel(const __grid_constant__ BeamArgs a) {
    constexpr int N = LpVec<TYPE>::N, SIZE = TYPE == KV_F32 ? 4 : 2;
    __shared__ BeamShared shared;
    BeamSegment &sh = shared.segment;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    release_dependents();
    wait_for_producer();
    int live = 0;
    for (int first = 0; first < a.rows; first += LP_THREADS) {
        const int row = first + tid;
        const bool is = row < a.rows && beam_state(a, a.row_first + row) == 1;
        const uint32_t mask = __ballot_sync(0xffffffffu, is);
        if (lane == 0) shared.counts[warp] = __popc(mask);
        __syncthreads();
        int at = live + __popc(mask & ((1u << lane) - 1));
#pragma unroll
        for (int w = 0; w < BEAM_WARPS; ++w) {
            const int n = shared.counts[w];
            if (w < warp) at += n;
            live += n;
        }
        if (is) shared.live[at] = (uint16_t)row;
        __syncthreads();
    }
    if (tid == 0) shared.ndone = 0;
    const int all = live * a.batches, ctas = (int)gridDim.x;       // below 2^24: a row has at most 16 batches to each of 512 segments
    const BeamShare share{max(a.least, (all + ctas - 1) / ctas), a.batches};
    int at = (int)blockIdx.x * share.size;
    const int end = min(all, at + share.size);

    // A segment: element e of its row is element e + skew of the row's 16-byte vectors.
    const char *base = nullptr, *aligned = nullptr;
    int64_t v0 = 0, v_end = 0, v_low = 0, v_high = 0;
    int skew = 0;
    auto open = [&]() {
        const int entry = at / a.batches, inside = at - entry * a.batches, n = min(min(a.batches - inside, end - at), BEAM_BATCHES);
        base = a.logits + (a.row_first + shared.live[entry]) * a.stride * SIZE;
        skew = (int)(((uintptr_t)base & 15) / SIZE);
        aligned = base - skew * SIZE;
        v0 = (int64_t)inside * BEAM_BATCH;
        v_end = min(v0 + (int64_t)n * BEAM_BATCH, (a.vocab + skew + N - 1) / N);
        v_low = skew ? 1 : 0;
        v_high = min(v_end, (a.vocab + skew) / N);                 // whole vectors
        return n;
    };
    auto fetch = [&](int64_t first, uint4 (&raw)[LP_VECS]) {       // -inf past the segment's end
        const char *const from = aligned + (first + tid) * 16;
        if (first >= v_low && first + BEAM_BATCH <= v_high) {
#pragma unroll
            for (int i = 0; i < LP_VECS; ++i) raw[i] = __ldcs((const uint4 *)(from + i * LP_THREADS * 16));
        } else {
#pragma unroll
            for (int i = 0; i < LP_VECS; ++i) {
                constexpr uint32_t none = TYPE == KV_F32 ? 0xff800000u : TYPE == KV_F16 ? 0xfc00fc00u : 0xff80ff80u;
                const int64_t v = first + tid + i * LP_THREADS;
                raw[i] = make_uint4(none, none, none, none);
                if (v >= v_low && v < v_high) raw[i] = __ldcs((const uint4 *)(from + i * LP_THREADS * 16));
                else if (v < v_end) raw[i] = lp_partial<TYPE>(base, v * N - skew, a.vocab);
            }
        }
    };
    uint4 raw[LP_VECS], ahead[LP_VECS];
    int n = 0;
    if (at < end) {
        n = open();
        fetch(v0, raw);
    }
    while (at < end) {
        const int entry = at / a.batches, local = shared.live[entry], group = local / a.beams, seg = share.before(entry, at - entry * a.batches);
        BeamSums sum{-INFINITY, 0.0f};
        int batches = 0;
        for (int64_t first = v0; first < v_end; first += BEAM_BATCH, ++batches) {
            fetch(first + BEAM_BATCH, ahead);
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
#pragma unroll
            for (int i = 0; i < LP_VECS; ++i) raw[i] = ahead[i];
        }
        lp_segment_top<TYPE>(a, sh, base, skew, v0, v_end, batches, lp_order(sum.m));
        at += n;
        if (at < end) {                                            // the next segment's first batch, on its way from here
            n = open();
            fetch(v0, raw);
        }
        sum = beam_warp_join(sum);
        if (lane == 0) sh.sums[warp] = LpSums{sum.m, sum.s, 0.0f};
        __syncthreads();
        if (warp == 0) {
            sum = BeamSums{sh.sums[lane % BEAM_WARPS].m, lane < BEAM_WARPS ? sh.sums[lane % BEAM_WARPS].s : 0.0f};
            sum = beam_warp_join(sum);
            const int64_t list = (int64_t)local * a.lists + seg;
            if (lane == 0) a.part[list] = make_float2(sum.m, sum.s);
            if (lane < a.k) a.part_top[list * a.k + lane] = sh.best[lane];
            __syncwarp();
            // The CTA's last segment of this request?  The request's live rows are neighbours in the stream.
            if (at >= end || shared.live[at / a.batches] / a.beams != group) {
                const int before = entry - 1 - lane, after = entry + 1 + lane;
                const int low = entry - __popc(__ballot_sync(0xffffffffu, before >= 0 && shared.live[max(before, 0)] / a.beams == group));
                const int high = entry + __popc(__ballot_sync(0xffffffffu, after < live && shared.live[min(after, live - 1)] / a.beams == group));
                const int parts = ((high + 1) * a.batches - 1) / share.size - low * a.batches / share.size + 1;
                if (lane == 0) {
                    unsigned int before_me;
                    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before_me) : "l"(a.counter + group) : "memory");
                    if (before_me == (unsigned)parts - 1) {
                        a.counter[group] = 0;
                        shared.done[shared.ndone] = (uint16_t)group;
                        shared.first[shared.ndone] = (uint16_t)low;
                        shared.rows[shared.ndone++] = (uint8_t)(high - low + 1);
                    }
                }
            }
        }
        // Warp 0's other lanes and the other warps go on to the next segment, whose own barriers keep what is read here.
        __syncwarp();
    }
    __syncthreads();
    const int ndone = shared.ndone;
    for (int i = 0; i < ndone; ++i) beam_choose(a, shared, shared.done[i], shared.first[i], shared.rows[i], share);
    // Requests without a live row.
    const int groups = a.rows / a.beams;
    for (int group = blockIdx.x; group < groups; group += gridDim.x) {
        int any = 0;
        if (tid < a.beams) any = beam_state(a, a.row_first + (int64_t)group * a.beams + tid) == 1;
        if (__syncthreads_or(any)) continue;
        beam_choose(a, shared, group, 0, 0, share);
    }
}

// States.  Plane p of row i: the parent's first `length` lines (all of them without lengths), then one line of `append`.  Bytes are
// moved as they are, a chunk of eight vectors to a thread for each CTA, all of them asked for before the first is stored.  Bound by memory: 83 MB
// read and written in 13.6 us (6.1 TB/s), 2.5 GB in 352 (7.0 TB/s, parents that several rows share are read from L2).
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
