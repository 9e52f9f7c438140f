// nc_logprobs.cuh -- log probabilities of given tokens, entropy and the best alternatives of rows of logits.
//
// With M the row's maximum, S = sum exp(x - M) and E = sum exp(x - M) (x - M):
//   log p(t) = (x_t - M) - log S,   entropy = log S - E / S,   log-sum = M + log S,
// and the top k by value, the lowest index first among equals (a NaN counts as the largest, as in the
// LM head's argmax).  A logit of -inf adds nothing; a row of nothing else has log probabilities of
// -inf and entropy 0.
//
// One pass over the logits, which bound it.  A CTA streams a segment of a row in batches of four 16-byte vectors to
// a thread, the next batch's loads in flight while one is worked on.  Each thread keeps its own maximum and sums,
// rescaled only by a batch with a larger value, and leaves the maximum of each batch (a block of 16 or 32
// logits) in shared memory: no barrier and nothing of the top is in the loop.  The top k lie in the blocks whose maxima
// reach the k-th largest one, T.  The k-th largest of the maxima of 32 groups of threads is a bound that about as
// many blocks as k reach: they are read again and their values from there up ranked.  Where that is more blocks than are
// read at once, T is found among them, or bit by bit; where more end in T than are read at once, the first k of its equals
// in the row's order are taken.  The last CTA of a row joins the segments, in their order.
//
// Measured, 151936 logits to a row, 20 best of each: 512 float32 rows 71 us (4.4 TB/s; 59 with no best asked for, 48 at the
// rate of a copy), 512 bfloat16 rows 45 us, where unpacking and exponentials bound it; one row 8.9 us, five of them the
// start, the join and the ranking.  A running list of the best inside the loop took 298 us for the first of these.
#pragma once

#include "nc_kv4.cuh"

namespace nc {

constexpr int LP_THREADS = 256;
constexpr int LP_CTAS = 4;             // resident on an SM
constexpr int LP_VECS = 4;             // vectors of a batch, for each thread
constexpr int LP_BATCHES = 32;         // of a segment at most: their maxima are kept
constexpr int LP_MAX_TOP = 32;
constexpr int LP_CAND = 1024;          // room for candidates: the values of LP_CAND / 8 N blocks
constexpr int LP_ROWS = 4096;          // rows of a launch at most: their finish counters
constexpr int LP_SEGS = LP_THREADS;    // segments of a row at most

struct LogprobArgs {
    const char *logits;                // [rows][vocab], rows `stride` elements apart
    const int64_t *targets;            // [rows][ntargets]
    float *out, *entropy, *lse;        // [rows][ntargets], [rows], [rows]; the last two may be null
    int64_t *top;                      // [rows][k]
    float *top_logprobs;               // [rows][k]
    unsigned int *counter;             // [rows], zero before and after
    float4 *part;                      // [rows][segs]: M, S, E
    unsigned long long *part_top;      // [rows][segs][k]
    unsigned long long *error;         // null, or the smallest row with a target outside the vocabulary
    int64_t stride, vocab, row_first;
    int64_t seg_vecs;                  // vectors of a segment
    int ntargets, k, segs;
};

// Orders (value, index): larger values first, then lower indices.  -0 counts as +0, every NaN as the largest.
__device__ __forceinline__ uint32_t lp_order(float x) { return x != x ? 0xffffffffu : ordered_bits(x == 0.0f ? 0.0f : x); }
__device__ __forceinline__ float lp_value(uint32_t order) {
    return order == 0xffffffffu ? __uint_as_float(0x7fc00000u) : from_ordered_bits(order);
}
__device__ __forceinline__ unsigned long long lp_key(float x, uint32_t index) {
    return (unsigned long long)lp_order(x) << 32 | (0xffffffffu - index);
}

template <int TYPE>
struct LpVec {
    static constexpr int N = TYPE == KV_F32 ? 4 : 8;         // elements of 16 bytes
};

template <int TYPE>
__device__ __forceinline__ void lp_unpack(const uint4 &w, float *x) {
    if constexpr (TYPE == KV_F32) {
        x[0] = __uint_as_float(w.x);
        x[1] = __uint_as_float(w.y);
        x[2] = __uint_as_float(w.z);
        x[3] = __uint_as_float(w.w);
    } else {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (TYPE == KV_F16) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u[i]));
                x[2 * i] = f.x;
                x[2 * i + 1] = f.y;
            } else {
                x[2 * i] = __uint_as_float(u[i] << 16);
                x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
            }
        }
    }
}

// The vector whose first element is element e of a row of n, -inf outside the row; for the row's ends only.
template <int TYPE>
__device__ __noinline__ uint4 lp_partial(const char *row, int64_t e, int64_t n) {
    constexpr int N = LpVec<TYPE>::N;
    uint32_t w[4] = {0, 0, 0, 0};
    for (int j = 0; j < N; ++j) {
        const bool in = e + j >= 0 && e + j < n;
        if constexpr (TYPE == KV_F32) {
            w[j] = in ? ((const uint32_t *)row)[e + j] : 0xff800000u;
        } else {
            const uint32_t v = in ? ((const uint16_t *)row)[e + j] : TYPE == KV_F16 ? 0xfc00u : 0xff80u;
            w[j >> 1] |= v << (16 * (j & 1));
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Sums relative to a maximum: s = sum exp(x - m), e = sum exp(x - m) (x - m); m is -inf with no sums.
struct LpSums {
    float m, s, e;
};
// Of a rounded product with log2(e): a term exp(d) is off by 2^-23 |d| + 2^-22 of itself, least where it counts.  The outputs of the
// measured cases are 2.5e-8 to 8e-8 from 64 bits; elementary torch operations in float32 4e-8 to 6e-8.
__device__ __forceinline__ float lp_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr float LP_LOG2E = 1.4426950408889634f;
constexpr float LP_LEAST = -1000.0f;   // exp is 0 below: keeps 0 * -inf out of the entropy
__device__ __forceinline__ LpSums lp_join(const LpSums &a, const LpSums &b) {
    const float m = max_nan(a.m, b.m), to = m == -INFINITY ? 0.0f : m;
    const float da = max_nan(a.m - to, LP_LEAST), db = max_nan(b.m - to, LP_LEAST);
    const float wa = lp_exp2(da * LP_LOG2E), wb = lp_exp2(db * LP_LOG2E);
    LpSums r;
    r.m = m;
    r.s = __fmaf_rn(a.s, wa, b.s * wb);
    r.e = __fmaf_rn(wa, __fmaf_rn(a.s, da, a.e), wb * __fmaf_rn(b.s, db, b.e));
    return r;
}
// The largest value of a vector, a NaN if there is one.
template <int TYPE>
__device__ __forceinline__ float lp_vector_max(const uint4 &w) {
    if constexpr (TYPE == KV_F32) {
        return max_nan(max_nan(__uint_as_float(w.x), __uint_as_float(w.y)), max_nan(__uint_as_float(w.z), __uint_as_float(w.w)));
    } else if constexpr (TYPE == KV_F16) {
        const __half2 *h = reinterpret_cast<const __half2 *>(&w);
        const float2 m = __half22float2(__hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3])));
        return max_nan(m.x, m.y);
    } else {
        const __nv_bfloat162 *h = reinterpret_cast<const __nv_bfloat162 *>(&w);
        const float2 m = __bfloat1622float2(__hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3])));
        return max_nan(m.x, m.y);
    }
}

__device__ __forceinline__ LpSums lp_warp_join(LpSums v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        LpSums w;
        w.m = __shfl_xor_sync(0xffffffffu, v.m, o);
        w.s = __shfl_xor_sync(0xffffffffu, v.s, o);
        w.e = __shfl_xor_sync(0xffffffffu, v.e, o);
        v = lp_join(v, w);
    }
    return v;
}

// How many of the n keys are above keys[i], for i < n: four neighbouring threads share an i.  Calls use(i, key, above) in
// one thread for each i.
template <typename F>
__device__ __forceinline__ void lp_ranks(const unsigned long long *keys, int n, F use) {
    const int part = threadIdx.x & 3;
    for (int base = 0; base < n; base += LP_THREADS / 4) {
        const int i = base + (threadIdx.x >> 2);
        const unsigned long long mine = i < n ? keys[i] : ~0ull;
        int above = 0;
#pragma unroll 4
        for (int j = part; j < n; j += 4) above += keys[j] > mine;
        above += __shfl_xor_sync(0xffffffffu, above, 1);
        above += __shfl_xor_sync(0xffffffffu, above, 2);
        if (part == 0 && i < n) use(i, mine, above);
    }
}
// The k best of the n keys in `keys` (distinct), in order, to out.
__device__ __forceinline__ void lp_rank(const unsigned long long *keys, int n, int k, unsigned long long *out) {
    lp_ranks(keys, n, [&](int, unsigned long long key, int above) {
        if (above < k) out[above] = key;
    });
}

struct LpShared {
    uint32_t block[LP_BATCHES][LP_THREADS];                        // maxima, in order
    uint32_t group_max[32];
    LpSums sums[LP_THREADS / 32];
    unsigned long long cand[LP_CAND], best[LP_MAX_TOP], round[LP_THREADS / 32], heads[LP_SEGS];
    int count, greater, equal;
    uint32_t kth;
    unsigned int arrived;
};

__device__ __forceinline__ unsigned long long lp_warp_max(unsigned long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long other = __shfl_xor_sync(0xffffffffu, v, o);
        v = other > v ? other : v;
    }
    return v;
}
// The largest of the block's keys, in every thread.  The caller's next write to `round` comes after a barrier.
__device__ __forceinline__ unsigned long long lp_block_max(unsigned long long v, unsigned long long *round) {
    v = lp_warp_max(v);
    if ((threadIdx.x & 31) == 0) round[threadIdx.x >> 5] = v;
    __syncthreads();
    v = round[0];
#pragma unroll
    for (int w = 1; w < LP_THREADS / 32; ++w) v = round[w] > v ? round[w] : v;
    return v;
}

// The k best keys of a segment, in order, to sh.best (0 past its end); `mine`: the largest of the thread's blocks.
template <int TYPE>
__device__ __forceinline__ void lp_segment_top(const LogprobArgs &a, LpShared &sh, const char *base, int skew, int64_t seg0,
                                               int64_t v_end, int batches, uint32_t mine) {
    constexpr int N = LpVec<TYPE>::N, SIZE = LP_VECS * N, MOST = LP_CAND / SIZE;      // values of a block; blocks to read again
    constexpr int64_t BATCH = LP_THREADS * LP_VECS;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint32_t quarter = mine;                                       // of eight threads
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) quarter = max(quarter, __shfl_xor_sync(0xffffffffu, quarter, o));
    if ((lane & 7) == 0) sh.group_max[tid >> 3] = quarter;
    if (tid == 0) sh.count = sh.greater = sh.equal = 0;
    if (tid < a.k) sh.best[tid] = 0;
    __syncthreads();
    const uint32_t group = sh.group_max[lane];
    int rank = 0;
#pragma unroll
    for (int j = 0; j < 32; ++j) {
        const uint32_t other = sh.group_max[j];
        rank += other > group || (other == group && j < lane);
    }
    const uint32_t bound = __shfl_sync(0xffffffffu, group, __ffs(__ballot_sync(0xffffffffu, rank == a.k - 1)) - 1);
    if (mine >= bound)
#pragma unroll 4
        for (int i = 0; i < batches; ++i) {
            const uint32_t most = sh.block[i][tid];
            if (most >= bound) {
                const int at = atomicAdd(&sh.count, 1);
                if (at < LP_CAND) sh.cand[at] = (unsigned long long)most << 32 | (uint32_t)(i * LP_THREADS + tid);
            }
        }
    __syncthreads();
    int *const list = (int *)sh.heads;                             // MOST block numbers; the heads come later
    uint32_t kth = 0;
    bool all = false;
    const int reached = sh.count;
    if (reached <= MOST) {                                         // few enough to be read again as they are
        kth = bound;
        all = true;
        if (tid < reached) list[tid] = (int)(uint32_t)sh.cand[tid];
        if (tid == 0) sh.greater = reached;
    } else if (reached <= LP_CAND) {                               // T, and the blocks above it (fewer than k), then those that end in it
        lp_ranks(sh.cand, reached, [&](int, unsigned long long key, int above) {
            if (above == a.k - 1) sh.kth = (uint32_t)(key >> 32);
        });
        __syncthreads();
        kth = sh.kth;
        for (int i = tid; i < reached; i += LP_THREADS) {
            const uint32_t most = (uint32_t)(sh.cand[i] >> 32);
            if (most > kth) list[atomicAdd(&sh.greater, 1)] = (int)(uint32_t)sh.cand[i];
            else if (most == kth) atomicAdd(&sh.equal, 1);
        }
        __syncthreads();
        all = sh.greater + sh.equal <= MOST;
        __syncthreads();
        if (all)
            for (int i = tid; i < reached; i += LP_THREADS)
                if ((uint32_t)(sh.cand[i] >> 32) == kth) list[atomicAdd(&sh.greater, 1)] = (int)(uint32_t)sh.cand[i];
    } else {                                                       // masses of equals, or of good blocks in few threads:
        for (int bit = 31; bit >= 0; --bit) {                      // bit by bit, the largest T that k blocks reach
            const uint32_t trial = kth | 1u << bit;
            int n = 0;
            for (int i = 0; i < batches; ++i) n += sh.block[i][tid] >= trial;
            n = warp_sum_int(n);
            if (lane == 0) sh.round[warp] = n;
            __syncthreads();
            n = 0;
            for (int w = 0; w < LP_THREADS / 32; ++w) n += (int)sh.round[w];
            if (n >= a.k) kth = trial;
            __syncthreads();
        }
        for (int i = 0; i < batches; ++i)
            if (sh.block[i][tid] > kth) list[atomicAdd(&sh.greater, 1)] = i * LP_THREADS + tid;
    }
    __syncthreads();
    if (tid == 0) sh.count = 0;
    const int values = sh.greater * SIZE;
    __syncthreads();
    for (int base_at = tid; base_at < values; base_at += 4 * LP_THREADS) {
        unsigned long long key[4];
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const int at = base_at + m * LP_THREADS, block = list[min(at, values - 1) / SIZE], u = at % SIZE;
            const int64_t v = seg0 + block / LP_THREADS * BATCH + block % LP_THREADS + u / N * LP_THREADS;
            const int64_t e = v * N - skew + u % N;
            key[m] = at < values && v < v_end && e >= 0 && e < a.vocab ? lp_key(kv_load(base, e, TYPE), (uint32_t)e) : 0;
        }
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const uint32_t order = (uint32_t)(key[m] >> 32);
            if (key[m] != 0 && (all ? order >= kth : order > kth)) sh.cand[atomicAdd(&sh.count, 1)] = key[m];
        }
    }
    __syncthreads();
    if (!all) {                                                    // the first k equals, in the row's order
        static_assert((LP_MAX_TOP - 1) * SIZE + LP_MAX_TOP <= LP_CAND, "values of fewer than k blocks, and k equals");
        int found = 0;
        for (int64_t e0 = max((int64_t)0, seg0 * N - skew); found < a.k && e0 < min(a.vocab, v_end * N - skew); e0 += LP_THREADS) {
            const int64_t e = e0 + tid;
            const unsigned long long key = e < min(a.vocab, v_end * N - skew) ? lp_key(kv_load(base, e, TYPE), (uint32_t)e) : 0;
            const bool is = key != 0 && (uint32_t)(key >> 32) == kth;
            const uint32_t equals = __ballot_sync(0xffffffffu, is);
            if (lane == 0) sh.round[warp] = __popc(equals);
            __syncthreads();
            int rank = found + __popc(equals & ((1u << lane) - 1));
#pragma unroll
            for (int w = 0; w < LP_THREADS / 32; ++w) {
                const int n = (int)sh.round[w];
                if (w < warp) rank += n;
                found += n;
            }
            if (is && rank < a.k) sh.cand[atomicAdd(&sh.count, 1)] = key;
            __syncthreads();
        }
    }
    lp_rank(sh.cand, sh.count, a.k, sh.best);
    __syncthreads();
}

template <int TYPE>
__global__ void __launch_bounds__(LP_THREADS, LP_CTAS) logprobs_kernel(const __grid_constant__ LogprobArgs a) {
    constexpr int N = LpVec<TYPE>::N, SIZE = TYPE == KV_F32 ? 4 : 2;
    constexpr int64_t BATCH = LP_THREADS * LP_VECS;                // vectors
    __shared__ LpShared sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    release_dependents();
    wait_for_producer();
    const int seg = (int)(blockIdx.x % a.segs);
    const int64_t local = blockIdx.x / a.segs, row = a.row_first + local;
    const char *const base = a.logits + row * a.stride * SIZE;
    // Vectors lie on 16-byte boundaries: element e of the row is element e + skew of the vectors.
    const int skew = (int)(((uintptr_t)base & 15) / SIZE);
    const char *const aligned = base - skew * SIZE;
    const int64_t v_end = min((int64_t)(seg + 1) * a.seg_vecs, (a.vocab + skew + N - 1) / N);

    const int64_t v_low = skew ? 1 : 0, v_high = min(v_end, (a.vocab + skew) / N);       // whole vectors
    auto fetch = [&](int64_t first, uint4 (&raw)[LP_VECS]) {
        const char *const from = aligned + (first + tid) * 16;
        if (first >= v_low && first + BATCH <= v_high) {
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

    LpSums sum{-INFINITY, 0.0f, 0.0f};
    float2 pair = make_float2(0.0f, 0.0f), epair = pair;           // the two halves of the thread's sums
    const int64_t seg0 = (int64_t)seg * a.seg_vecs;
    uint4 raw[LP_VECS], ahead[LP_VECS];
    fetch(seg0, raw);
    int batches = 0;
    for (int64_t first = seg0; first < v_end; first += BATCH, ++batches) {
        fetch(first + BATCH, ahead);
        float top = lp_vector_max<TYPE>(raw[0]);
#pragma unroll
        for (int i = 1; i < LP_VECS; ++i) top = max_nan(top, lp_vector_max<TYPE>(raw[i]));
        if (a.k) sh.block[batches][tid] = lp_order(top);
        if (top > sum.m || top != top) {                         // a larger value, or a NaN, which then stays the maximum
            const float s = pair.x + pair.y, e = epair.x + epair.y;
            const float d = max_nan(sum.m - top, LP_LEAST), w = lp_exp2(d * LP_LOG2E);
            pair = make_float2(s * w, 0.0f);
            epair = make_float2(w * __fmaf_rn(s, d, e), 0.0f);
            sum.m = top;
        }
        const float to = sum.m == -INFINITY ? 0.0f : sum.m;
        const uint64_t unit = pack2(LP_LOG2E, LP_LOG2E), from = pack2(-to, -to);
        uint64_t s2 = pack2(pair.x, pair.y), e2 = pack2(epair.x, epair.y);
#pragma unroll
        for (int i = 0; i < LP_VECS; ++i) {
            float x[N];
            lp_unpack<TYPE>(raw[i], x);
#pragma unroll
            for (int j = 0; j < N; j += 2) {
                const float2 d = unpack2(add2(pack2(x[j], x[j + 1]), from));
                const uint64_t d2 = pack2(max_nan(d.x, LP_LEAST), max_nan(d.y, LP_LEAST));
                const float2 u = unpack2(mul2(d2, unit));
                const uint64_t p = pack2(lp_exp2(u.x), lp_exp2(u.y));
                s2 = add2(s2, p);
                e2 = fma2(p, d2, e2);
            }
        }
        pair = unpack2(s2);
        epair = unpack2(e2);
#pragma unroll
        for (int i = 0; i < LP_VECS; ++i) raw[i] = ahead[i];
    }
    sum.s = pair.x + pair.y;
    sum.e = epair.x + epair.y;
    if (a.k) lp_segment_top<TYPE>(a, sh, base, skew, seg0, v_end, batches, lp_order(sum.m));
    sum = lp_warp_join(sum);
    if (lane == 0) sh.sums[warp] = sum;
    __syncthreads();
    sum = sh.sums[0];
#pragma unroll
    for (int w = 1; w < LP_THREADS / 32; ++w) sum = lp_join(sum, sh.sums[w]);

    if (a.segs > 1) {
        if (tid == 0) a.part[local * a.segs + seg] = make_float4(sum.m, sum.s, sum.e, 0.0f);
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
        sum = LpSums{-INFINITY, 0.0f, 0.0f};
        if (tid < a.segs) {
            const float4 p = __ldcg(a.part + local * a.segs + tid);
            sum = LpSums{p.x, p.y, p.z};
        }
        const unsigned long long *const tops = a.part_top + local * a.segs * a.k;
        unsigned long long head = 0, floor_key = 0;
        if (a.k && tid < a.segs) {
            head = __ldcg(tops + tid * a.k);
            floor_key = __ldcg(tops + tid * a.k + a.k - 1);
            sh.heads[tid] = head;
        }
        sum = lp_warp_join(sum);
        if (lane == 0) sh.sums[warp] = sum;
        __syncthreads();
        sum = sh.sums[0];
#pragma unroll
        for (int w = 1; w < LP_THREADS / 32; ++w) sum = lp_join(sum, sh.sums[w]);
        if (a.k) {
            // A key below the k-th largest of the segments' best, or below a segment's own k-th best, has
            // k better ones: at most k * k keys are left to rank.
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
            __syncthreads();
            lp_rank(sh.cand, sh.count, a.k, sh.best);
            __syncthreads();
        }
    }

    // The row's results.
    const float log_s = logf(sum.s);
    const bool none = sum.m == -INFINITY;
    if (tid == 0) {
        if (a.entropy) a.entropy[row] = none ? 0.0f : log_s - fdiv(sum.e, sum.s);
        if (a.lse) a.lse[row] = none ? -INFINITY : sum.m + log_s;
    }
    auto logprob = [&](float x) { return none ? -INFINITY : (x - sum.m) - log_s; };
    for (int j = tid; j < a.ntargets; j += LP_THREADS) {
        const int64_t t = a.targets[row * a.ntargets + j];
        float v = __uint_as_float(0x7fc00000u);
        if (t >= 0 && t < a.vocab) v = logprob(kv_load(base, t, TYPE));
        else if (a.error) atomicMin(a.error, (unsigned long long)row);
        a.out[row * a.ntargets + j] = v;
    }
    if (tid < a.k) {
        const unsigned long long key = sh.best[tid];
        a.top[row * a.k + tid] = 0xffffffffu - (uint32_t)key;
        a.top_logprobs[row * a.k + tid] = logprob(lp_value((uint32_t)(key >> 32)));
    }
}

}  // namespace nc
