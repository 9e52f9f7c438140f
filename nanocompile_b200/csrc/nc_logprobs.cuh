// nc_logprobs.cuh -- log probabilities of given tokens, entropy and the best alternatives of rows of logits.
//
// With M the row's maximum, S = sum exp(x - M) and E = sum exp(x - M) (x - M):
//   log p(t) = (x_t - M) - log S,   entropy = log S - E / S,   log-sum = M + log S,
// and the top k by value, the lowest index first among equals (a NaN counts as the largest, as in the
// LM head's argmax).  A logit of -inf adds nothing; a row of nothing else has log probabilities of
// -inf and entropy 0.
//
// One pass over the logits, which bound it: a CTA takes a segment of a row into registers with one
// burst of 16-byte loads, so its maximum is known before the first exponential and nothing is read
// twice.  The segment's best k: the k-th largest of 32 maxima (each of eight threads' values) is a
// lower bound that at least k values reach; the few that do are ranked by comparing each with all.
// The last CTA of a row joins the segments, in their order.
#pragma once

#include "nc_kv4.cuh"

namespace nc {

constexpr int LP_THREADS = 256;
constexpr int LP_MAX_TOP = 32;
constexpr int LP_CAND = LP_MAX_TOP * LP_MAX_TOP;   // candidates ranked at once; more (masses of equal values) take rounds
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
    int ntargets, k, segs;
};

// Orders (value, index): larger values first, then lower indices.  -0 counts as +0, every NaN as the largest.
__device__ __forceinline__ unsigned long long lp_key(float x, uint32_t index) {
    uint32_t u = x != x ? 0xffffffffu : ordered_bits(x == 0.0f ? 0.0f : x);
    return (unsigned long long)u << 32 | (0xffffffffu - index);
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

__device__ __forceinline__ float lp_block_max(float v, float *buf) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = nan_max(v, __shfl_xor_sync(0xffffffffu, v, o));
    if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
    __syncthreads();
    v = buf[0];
#pragma unroll
    for (int w = 1; w < LP_THREADS / 32; ++w) v = nan_max(v, buf[w]);
    return v;
}

// The k best of the n keys in `keys` (distinct), in order, to out.
__device__ __forceinline__ void lp_rank(const unsigned long long *keys, int n, int k, unsigned long long *out) {
    for (int i = threadIdx.x; i < n; i += LP_THREADS) {
        const unsigned long long mine = keys[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += keys[j] > mine;
        if (rank < k) out[rank] = mine;
    }
}

struct LpShared {
    float warp_max[LP_THREADS / 32], group_max[32];
    float2 sums[LP_THREADS / 32];
    unsigned long long cand[LP_CAND], best[LP_MAX_TOP], round[LP_THREADS / 32], heads[LP_SEGS];
    float4 parts[LP_SEGS];
    int count;
    float bound;
    unsigned int arrived;
};

// EPT elements per thread: a segment is EPT * 256 elements.
template <int TYPE, int EPT>
__global__ void __launch_bounds__(LP_THREADS) logprobs_kernel(const __grid_constant__ LogprobArgs a) {
    constexpr int N = LpVec<TYPE>::N, VECS = EPT / N, SIZE = TYPE == KV_F32 ? 4 : 2;
    __shared__ LpShared sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int seg = (int)(blockIdx.x % a.segs);
    const int64_t local = blockIdx.x / a.segs, row = a.row_first + local;
    wait_for_producer();
    const char *const base = a.logits + row * a.stride * SIZE;
    // Vectors lie on 16-byte boundaries: element e of the row is element e + skew of the vectors.
    const int skew = (int)(((uintptr_t)base & 15) / SIZE);
    const char *const aligned = base - skew * SIZE;
    const int64_t v0 = (int64_t)seg * (LP_THREADS * VECS) + tid;
    float x[EPT];
    uint4 raw[VECS];
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
        const int64_t e = (v0 + i * LP_THREADS) * N - skew;        // the vector's first element
        if (e >= 0 && e + N <= a.vocab) raw[i] = __ldcs((const uint4 *)(aligned + (v0 + i * LP_THREADS) * 16));
    }
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
        const int64_t e = (v0 + i * LP_THREADS) * N - skew;
        if (e >= 0 && e + N <= a.vocab) {
            lp_unpack<TYPE>(raw[i], x + i * N);
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j)
                x[i * N + j] = e + j >= 0 && e + j < a.vocab ? kv_load(base, e + j, TYPE) : -INFINITY;
        }
#pragma unroll
        for (int j = 0; j < N; ++j) top = nan_max(top, x[i * N + j]);
    }
    // 32 maxima, each of the eight threads of one quarter warp, for the top's bound.
    float quarter = top;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) quarter = nan_max(quarter, __shfl_xor_sync(0xffffffffu, quarter, o));
    if ((lane & 7) == 0) sh.group_max[tid >> 3] = quarter;
    if (tid == 0) sh.count = 0;
    const float M = lp_block_max(quarter, sh.warp_max);

    const float L2E = 1.4426950408889634f;
    const float base_m = M == -INFINITY ? 0.0f : M;
    float s = 0.0f, es = 0.0f;
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
        const float d = x[i] - base_m;
        float p;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p) : "f"(d * L2E));
        s += p;
        es = __fmaf_rn(p, fmaxf(d, -1000.0f), es);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, o);
        es += __shfl_xor_sync(0xffffffffu, es, o);
    }
    if (lane == 0) sh.sums[warp] = make_float2(s, es);

    if (a.k) {
        if (warp == 0) {
            const unsigned long long mine = lp_key(sh.group_max[lane], lane);
            int rank = 0;
#pragma unroll
            for (int j = 0; j < 32; ++j) rank += lp_key(sh.group_max[j], j) > mine;
            if (rank == a.k - 1) sh.bound = sh.group_max[lane];
        }
        __syncthreads();
        const float bound = sh.bound;
        // Values at or above the bound (a NaN always is); padding is told from a logit of -inf by its index.
        if (!(top < bound)) {
#pragma unroll
            for (int i = 0; i < EPT; ++i) {
                if (!(x[i] < bound) || bound != bound) {
                    const int64_t e = (v0 + i / N * LP_THREADS) * N - skew + i % N;
                    if (e >= 0 && e < a.vocab && (bound == bound || x[i] != x[i])) {
                        const int at = atomicAdd(&sh.count, 1);
                        if (at < LP_CAND) sh.cand[at] = lp_key(x[i], (uint32_t)e);
                    }
                }
            }
        }
        if (tid < a.k) sh.best[tid] = 0;
        __syncthreads();
        if (sh.count <= LP_CAND) {
            lp_rank(sh.cand, sh.count, a.k, sh.best);
        } else {                                                   // more equals than that: the best, k times over
            unsigned long long last = ~0ull;
            for (int r = 0; r < a.k; ++r) {
                unsigned long long mine = 0;
#pragma unroll
                for (int i = 0; i < EPT; ++i) {
                    const int64_t e = (v0 + i / N * LP_THREADS) * N - skew + i % N;
                    if (e >= 0 && e < a.vocab) {
                        const unsigned long long key = lp_key(x[i], (uint32_t)e);
                        if (key < last && key > mine) mine = key;
                    }
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) {
                    const unsigned long long other = __shfl_xor_sync(0xffffffffu, mine, o);
                    mine = other > mine ? other : mine;
                }
                if (lane == 0) sh.round[warp] = mine;
                __syncthreads();
                mine = sh.round[0];
#pragma unroll
                for (int w = 1; w < LP_THREADS / 32; ++w) mine = sh.round[w] > mine ? sh.round[w] : mine;
                if (tid == 0) sh.best[r] = mine;
                last = mine;
                __syncthreads();
            }
        }
    }
    __syncthreads();
    s = es = 0.0f;
#pragma unroll
    for (int w = 0; w < LP_THREADS / 32; ++w) {
        s += sh.sums[w].x;
        es += sh.sums[w].y;
    }

    float row_m = M, row_s = s, row_e = es;
    if (a.segs > 1) {
        if (tid == 0) a.part[local * a.segs + seg] = make_float4(M, s, es, 0.0f);
        if (tid < a.k) a.part_top[(local * a.segs + seg) * a.k + tid] = sh.best[tid];
        __threadfence();
        __syncthreads();
        if (tid == 0) sh.arrived = atomicAdd(a.counter + local, 1u);
        __syncthreads();
        if (sh.arrived != (unsigned)a.segs - 1) return;
        __threadfence();
        if (tid == 0) a.counter[local] = 0;
        for (int i = tid; i < a.segs; i += LP_THREADS) sh.parts[i] = __ldcg(a.part + local * a.segs + i);
        if (tid == 0) sh.count = 0;
        __syncthreads();
        row_m = -INFINITY;
        for (int i = 0; i < a.segs; ++i) row_m = nan_max(row_m, sh.parts[i].x);
        const float to = row_m == -INFINITY ? 0.0f : row_m;
        row_s = row_e = 0.0f;
        for (int i = 0; i < a.segs; ++i) {
            const float4 p = sh.parts[i];
            if (p.x == -INFINITY) continue;
            float w;
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"((p.x - to) * L2E));
            row_s = __fmaf_rn(p.y, w, row_s);
            row_e = __fmaf_rn(w, __fmaf_rn(p.y, fmaxf(p.x - to, -1000.0f), p.z), row_e);
        }
        if (a.k) {
            // A key below the k-th largest of the segments' best, or below a segment's own k-th best, has
            // k better ones: at most k * k keys are left to rank.
            const unsigned long long *const tops = a.part_top + local * a.segs * a.k;
            unsigned long long floor_key = 0, best = 0;
            if (tid < a.segs) {
                best = __ldcg(tops + tid * a.k);
                floor_key = __ldcg(tops + tid * a.k + a.k - 1);
                sh.heads[tid] = best;
            }
            __syncthreads();
            if (tid < a.segs) {
                int rank = 0;
                for (int i = 0; i < a.segs; ++i) rank += sh.heads[i] > best;
                if (rank == a.k - 1 && best > floor_key) floor_key = best;
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const unsigned long long other = __shfl_xor_sync(0xffffffffu, floor_key, o);
                floor_key = other > floor_key ? other : floor_key;
            }
            if (lane == 0) sh.round[warp] = floor_key;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < LP_THREADS / 32; ++w) floor_key = sh.round[w] > floor_key ? sh.round[w] : floor_key;
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
    const float log_s = logf(row_s);
    const bool none = row_m == -INFINITY;
    const float shift = none ? 0.0f : row_m;
    if (tid == 0) {
        if (a.entropy) a.entropy[row] = none ? 0.0f : log_s - row_e / row_s;
        if (a.lse) a.lse[row] = none ? -INFINITY : row_m + log_s;
    }
    for (int j = tid; j < a.ntargets; j += LP_THREADS) {
        const int64_t t = a.targets[row * a.ntargets + j];
        float v = __uint_as_float(0x7fc00000u);
        if (t >= 0 && t < a.vocab) v = none ? -INFINITY : (kv_load(base, t, TYPE) - shift) - log_s;
        else if (a.error) atomicMin(a.error, (unsigned long long)row);
        a.out[row * a.ntargets + j] = v;
    }
    if (tid < a.k) {
        const unsigned long long key = sh.best[tid];
        const int64_t t = 0xffffffffu - (uint32_t)key;
        a.top[row * a.k + tid] = t;
        a.top_logprobs[row * a.k + tid] = none ? -INFINITY : (kv_load(base, t, TYPE) - shift) - log_s;
    }
}

}  // namespace nc
