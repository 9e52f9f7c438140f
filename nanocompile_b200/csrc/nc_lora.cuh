// nc_lora.cuh -- low-rank adapters of many requests beside a shared projection.
//
// A row r of a sequence with adapter s, output n of target t (targets share x: q, k and v):
//   out[r, n] = base[r, n] + scale[s] sum_j B[s, n, j] h[j],   h[j] = sum_k A[s, t rank + j, k] x[r, k],   j < ranks[s].
//
// The plan groups a call's rows by adapter: sequences sorted by adapter (a bitonic sort in shared memory, in their order among
// equals), rows counted along them, and the groups cut into items of up to `tile` rows, one after another: places for items that there might
// have been come last, so that their clusters take no other's room (64 adapters of 1 MB for two rows each: 38 us with them in between).
// One CTA, bound by its barriers: 4.8 us for 64 sequences, 87 for 8192, once for all layers and projections of a batch.
//
// An item to a cluster of CTAs, in one launch: each multiplies its share of the inputs k, the CTAs add their sums of h through
// distributed shared memory, in the order of the CTAs, and each expands its share of the outputs.  Three kernels do so: for items of up
// to eight rows with much to read nc_lora_stream.cuh, for 128 rows nc_lora_tiles.cuh, and for the others the one here.
//
// lora_rows_kernel: weights are the matrix instruction's 16 rows, eight rows of x its columns (NT = 1), or 32 rows (NT = 4) where the 128 of an item
// are of a 16-bit type other than the weights', not aligned, or of a rank that leaves no room.  Weights go straight into operands, B's share is asked of L2
// at the start.  Bound by its chain of dependent loads: one row of 896 inputs to 1152 outputs at rank 16 takes 8.8 us with the plan.
//
// Accuracy.  Products are mma m16n8k8 tf32: 16-bit weights and rows are tf32 numbers as they are, float32 rows and h go in two parts
// (11 bits and the next 11, rounded: 2^-23 of the value is lost at most, the last bit of some).  The matrix unit cuts sums off rather
// than rounding them, so a chain is 32 inputs long, the small parts first or apart, and the chains are added in float32.
#pragma once

#include "nc_kv4.cuh"

namespace nc {

constexpr int LORA_TARGETS = 8, LORA_RANK = 128, LORA_SEQS = 8192;
constexpr int LORA_LINE = 1 << 23;             // inputs or outputs of a row at most: those of 128 rows are counted in 32 bits
constexpr int LORA_THREADS = 256, LORA_WARPS = LORA_THREADS / 32;
constexpr int LORA_PASS = 192;                 // rows of h at most in a pass: targets x rank in whole 32s
constexpr int LORA_HEAD = 4;                   // words before the plan's items: the rows, sequences and slots it was made for

// What went wrong in a kernel since it was last asked for: LORA_LATE a wait that ran out, LORA_OTHER a plan of other sizes than the call's.
__device__ unsigned int g_lora_fault;
constexpr unsigned int LORA_LATE = 1, LORA_OTHER = 2;

struct LoraPlanArgs {
    const int32_t *adapters;                   // [seqs]; outside 0 .. slots - 1: none
    const int32_t *row_start;                  // [seqs + 1] or null: row i is sequence i's
    int32_t *plan;
    unsigned long long *error;                 // null, or the smallest sequence with an adapter past the slots
    int rows, seqs, slots, tile, items, size;  // size: of the sort, a power of two
};

__device__ __forceinline__ int4 *lora_items(int32_t *plan) { return (int4 *)(plan + LORA_HEAD); }
__device__ __forceinline__ const int4 *lora_items(const int32_t *plan) { return (const int4 *)(plan + LORA_HEAD); }

// Inclusive sums of `v` over the block, in the threads' order; `sums`: 33 words.
__device__ __forceinline__ int lora_scan(int v, int *sums) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int w = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += w;
    }
    if (lane == 31) sums[warp] = v;
    __syncthreads();
    if (warp == 0) {
        int s = lane < warps ? sums[lane] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int w = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += w;
        }
        if (lane < warps) sums[lane] = s;
    }
    __syncthreads();
    if (warp > 0) v += sums[warp - 1];
    return v;
}

// One CTA.  Shared memory: size keys, then size + 1 row offsets, group starts, group adapters and the groups' first items.
__global__ void __launch_bounds__(1024, 1) lora_plan_kernel(const __grid_constant__ LoraPlanArgs a) {
    extern __shared__ __align__(16) char lora_smem[];
    unsigned long long *const key = (unsigned long long *)lora_smem;
    int *const offset = (int *)(key + a.size), *const start = offset + a.size + 1, *const group = start + a.size + 1, *const place = group + a.size + 1;
    __shared__ int sums[33];
    const int tid = threadIdx.x, threads = blockDim.x;
    release_dependents();
    wait_for_producer();
    auto begin_of = [&](int i) { return a.row_start ? min(max(a.row_start[i], 0), a.rows) : min(i, a.rows); };
    auto count_of = [&](int i) { return max(0, min(a.row_start ? a.row_start[i + 1] : i + 1, a.rows) - begin_of(i)); };
    for (int i = tid; i < a.size; i += threads) {
        unsigned long long k = ~0ull;
        if (i < a.seqs) {
            const int s = a.adapters[i];
            if (s >= a.slots && a.error) atomicMin(a.error, (unsigned long long)i);
            k = (unsigned long long)(s >= 0 && s < a.slots ? (unsigned)s : (unsigned)a.slots) << 32 | (unsigned)i;
        }
        key[i] = k;
    }
    for (int width = 2; width <= a.size; width <<= 1)
        for (int step = width >> 1; step > 0; step >>= 1) {
            __syncthreads();
            for (int i = tid; i < a.size / 2; i += threads) {
                const int low = 2 * i - (i & (step - 1)), high = low + step;
                const unsigned long long x = key[low], y = key[high];
                if ((x > y) == ((low & width) == 0)) key[low] = y, key[high] = x;
            }
        }
    __syncthreads();
    // Rows before each sequence of the order, and the groups' starts: both by sums over the order.
    int rows = 0, groups = 0;
    for (int base = 0; base < a.seqs; base += threads) {
        const int i = base + tid;
        const bool in = i < a.seqs;
        const unsigned s = in ? (unsigned)(key[i] >> 32) : 0;
        const int count = in ? count_of((int)(unsigned)key[i]) : 0;
        const bool first = in && (i == 0 || s != (unsigned)(key[i - 1] >> 32));
        const int upto = lora_scan(count, sums) + rows;
        __syncthreads();
        const int number = lora_scan(first, sums) + groups;
        if (in) offset[i] = upto - count;
        if (first) {
            start[number - 1] = upto - count;
            group[number - 1] = (int)s;
        }
        __syncthreads();
        if (tid == threads - 1) sums[32] = upto, sums[0] = number;
        __syncthreads();
        rows = sums[32];
        groups = sums[0];
        __syncthreads();
    }
    rows = min(max(rows, 0), a.rows);                              // otherwise only where row_start does not ascend
    if (tid == 0) {
        start[groups] = rows;
        *(int4 *)a.plan = make_int4(a.rows, a.seqs, a.slots, 0);
    }
    __syncthreads();
    int count = 0;                                                 // of items
    for (int base = 0; base < groups; base += threads) {
        const int i = base + tid, n = i < groups ? max(0, start[i + 1] - start[i] + a.tile - 1) / a.tile : 0;
        const int upto = lora_scan(n, sums) + count;
        if (i < groups) place[i] = upto - n;
        if (tid == threads - 1) sums[32] = upto;
        __syncthreads();
        count = sums[32];
        __syncthreads();
    }
    int4 *const items = lora_items(a.plan);
    for (int i = tid; i < a.items; i += threads) {
        int low = 0, high = groups;                                // the last group whose first item is i or before: those without rows have none
        while (high - low > 1) {
            const int mid = (low + high) >> 1;
            if (place[mid] <= i) low = mid;
            else high = mid;
        }
        int4 item = make_int4(-1, 0, 0, 0);
        if (i < count) {
            const int at = start[low] + (i - place[low]) * a.tile;
            item = make_int4(group[low] < a.slots ? group[low] : -1, at, min(a.tile, start[low + 1] - at), 0);
        }
        items[i] = item;
    }
    int32_t *const order = (int32_t *)(items + a.items);
    if (rows <= 4 * a.seqs) {
        for (int i = tid; i < a.seqs; i += threads) {
            const int seq = (int)(unsigned)key[i], n = count_of(seq), from = begin_of(seq);
            for (int j = 0; j < n; ++j)
                if ((unsigned)(offset[i] + j) < (unsigned)rows) order[offset[i] + j] = from + j;
        }
    } else {
        for (int i = tid >> 5; i < a.seqs; i += threads >> 5) {
            const int seq = (int)(unsigned)key[i], n = count_of(seq), from = begin_of(seq);
            for (int j = tid & 31; j < n; j += 32)
                if ((unsigned)(offset[i] + j) < (unsigned)rows) order[offset[i] + j] = from + j;
        }
    }
}

struct LoraArgs {
    const void *x, *base, *a, *b;              // [rows][inputs], [rows][outputs] or null, [slots][targets rank][inputs], [slots][outputs][rank]
    void *out;                                 // [rows][outputs], may be base
    const int32_t *plan, *ranks;               // ranks: [slots] or null
    const float *scales;                       // [slots] or null
    int64_t x_stride, base_stride, out_stride;
    int rows, seqs, items, tile, inputs, outputs, rank, slots, targets, pass_targets, wtype;
    int x_vectors, pairs, wide;                // 16-byte loads of x; two outputs to an access; 16 bytes of them
    int width[LORA_TARGETS];
};

__device__ __forceinline__ uint32_t lora_rank_of_cluster() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t lora_cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void lora_cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void lora_cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ float lora_peer(const float *p, uint32_t rank) {            // a word of another CTA's shared memory
    float v;
    asm volatile("{\n\t.reg .u32 at;\n\tmapa.shared::cluster.u32 at, %1, %2;\n\tld.shared::cluster.f32 %0, [at];\n\t}"
                 : "=f"(v)
                 : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank)
                 : "memory");
    return v;
}

__device__ __forceinline__ uint32_t lora_tf32(float v) {
    uint32_t r;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(v));
    return r;
}
// v in two tf32 parts.  An infinity or a NaN is its first part alone; what would round to infinity is cut off instead.
__device__ __forceinline__ void lora_split(float v, uint32_t *high, uint32_t *low) {
    *high = lora_tf32(v);
    float rest = fsub(v, __uint_as_float(*high));
    if (!(fabsf(rest) < INFINITY)) {
        rest = 0.0f;
        if (fabsf(v) < INFINITY) {
            *high = __float_as_uint(v) & 0xffffe000u;
            rest = fsub(v, __uint_as_float(*high));
        }
    }
    *low = lora_tf32(rest);
}
// Eight 16-bit weights as tf32.
template <int TW>
__device__ __forceinline__ void lora_weights(const uint4 &w, uint32_t (&v)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (TW == KV_F16) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u[i]));
            v[2 * i] = __float_as_uint(f.x);
            v[2 * i + 1] = __float_as_uint(f.y);
        } else {
            v[2 * i] = u[i] << 16;
            v[2 * i + 1] = u[i] & 0xffff0000u;
        }
    }
}
__device__ __forceinline__ void lora_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Two neighbouring values.
template <int TX>
__device__ __forceinline__ float2 lora_load2(const void *p, int64_t at, bool two, bool pairs) {
    if (pairs && two) {
        if constexpr (TX == KV_F32) return *(const float2 *)((const float *)p + at);
        else if constexpr (TX == KV_F16) return __half22float2(*(const __half2 *)((const __half *)p + at));
        else return __bfloat1622float2(*(const __nv_bfloat162 *)((const __nv_bfloat16 *)p + at));
    }
    return make_float2(kv_load(p, at, TX), two ? kv_load(p, at + 1, TX) : 0.0f);
}
template <int TX>
__device__ __forceinline__ void lora_store2(void *p, int64_t at, float2 v, bool two, bool pairs) {
    if (pairs && two) {
        if constexpr (TX == KV_F32) *(float2 *)((float *)p + at) = v;
        else if constexpr (TX == KV_F16) *(__half2 *)((__half *)p + at) = __floats2half2_rn(v.x, v.y);
        else *(__nv_bfloat162 *)((__nv_bfloat16 *)p + at) = __floats2bfloat162_rn(v.x, v.y);
    } else {
        kv_store(p, at, TX, v.x);
        if (two) kv_store(p, at + 1, TX, v.y);
    }
}

// An item of the plan: slot (-1: none), first place of its rows in the plan's order, how many; no rows where the plan is of other sizes.
__device__ __forceinline__ int4 lora_item(const LoraArgs &a, int i) {
    const int4 head = *(const int4 *)a.plan;
    int4 item = lora_items(a.plan)[i];
    if (head.x != a.rows || head.y != a.seqs || head.z != a.slots) {
        if (threadIdx.x == 0) atomicOr(&g_lora_fault, LORA_OTHER);
        item.z = 0;
    }
    if (item.z < 0 || item.z > a.rows || item.y < 0 || item.y > a.rows - item.z || item.x >= a.slots) item.z = 0;
    return item;
}
// The row at a place of the plan's order; -1 for what is no row of the call.
__device__ __forceinline__ int64_t lora_row(const LoraArgs &a, const int32_t *order, int at) {
    const int row = order[at];
    return row >= 0 && row < a.rows ? row : -1;
}
// Rows without an adapter, or with one of rank 0: columns [from, to) of base, or nought.
template <int TX>
__device__ __forceinline__ void lora_copy(const LoraArgs &a, const int32_t *order, int start, int count, int from, int to) {
    if (a.out == a.base) return;
    for (int i = threadIdx.x; i < (to - from) * count; i += blockDim.x) {
        const int64_t row = lora_row(a, order, start + i / (to - from));
        const int n = from + i % (to - from);
        if (row >= 0) kv_store(a.out, row * a.out_stride + n, TX, a.base ? kv_load(a.base, row * a.base_stride + n, TX) : 0.0f);
    }
}

template <int NT>
struct LoraShape {
    static constexpr int KS = LORA_WARPS / NT, TS = NT, TB = NT == 1 ? 4 : 2;      // warps along k, along the tiles; tiles of a warp at a time
    static constexpr int COLS = 8 * NT, HS = LORA_PASS + 4;                         // stride of h's columns: no bank twice
    static constexpr int PART = LORA_PASS * COLS;
    static constexpr size_t SMEM = (size_t)4 * (KS * PART + PART + COLS * HS);
};

template <int TX, int TW, int NT>
__global__ void __launch_bounds__(LORA_THREADS, 2) lora_rows_kernel(const __grid_constant__ LoraArgs a) {
    using S = LoraShape<NT>;
    constexpr int COLS = S::COLS;
    extern __shared__ __align__(16) char lora_smem[];
    float *const part = (float *)lora_smem, *const sum = part + S::KS * S::PART, *const h = sum + S::PART;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
    const int ctas = (int)lora_cluster_size(), cta = (int)lora_rank_of_cluster();
    release_dependents();
    wait_for_producer();
    // An item's rows from blockIdx.z COLS on.
    const int4 item = lora_item(a, blockIdx.x / ctas);
    const int32_t *const order = (const int32_t *)(lora_items(a.plan) + a.items);
    const int slot = item.x, first = item.y + (int)blockIdx.z * COLS, count = min(COLS, item.z - (int)blockIdx.z * COLS);
    if (count <= 0) return;
    const int t0 = (int)blockIdx.y * a.pass_targets, t1 = min(a.targets, t0 + a.pass_targets);
    int n_first = 0, n_pass = 0, n_tiles = 0;                      // outputs before the pass, of it, tiles of 16 of them
    for (int t = 0; t < t1; ++t) {
        if (t < t0) n_first += a.width[t];
        else n_pass += a.width[t], n_tiles += (a.width[t] + 15) / 16;
    }
    const int r = slot < 0 ? 0 : a.ranks ? min(max(a.ranks[slot], 0), a.rank) : a.rank;
    if (r == 0) {
        const int64_t n = n_pass;
        lora_copy<TX>(a, order, first, count, n_first + (int)(n * cta / ctas), n_first + (int)(n * (cta + 1) / ctas));
        return;
    }
    const float scale = a.scales ? a.scales[slot] : 1.0f;
    const char *const wa = (const char *)a.a + (int64_t)slot * a.targets * a.rank * a.inputs * 2;
    const char *const wb = (const char *)a.b + (int64_t)slot * a.outputs * a.rank * 2;
    const int tile_low = (int)((int64_t)n_tiles * cta / ctas), tile_high = (int)((int64_t)n_tiles * (cta + 1) / ctas);
    {
        // B's share of this CTA, as if the targets' last tiles were whole: at worst some lines that a neighbour reads.
        const int64_t low = ((int64_t)n_first + 16 * tile_low) * a.rank * 2, high = min((int64_t)n_first + n_pass, (int64_t)n_first + 16 * tile_high) * a.rank * 2;
        for (int64_t at = low + tid * 4096; at < high; at += LORA_THREADS * 4096)
            asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(wb + at), "r"((uint32_t)min((int64_t)4096, high - at)) : "memory");
    }
    int64_t row[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) row[i] = 8 * i + g < count ? lora_row(a, order, first + 8 * i + g) : -1;

    // h: tiles of 16 of its rows, units of 32 inputs.
    const int per = (r + 15) / 16, tiles = per * (t1 - t0);
    {
        const int units = (a.inputs + 31) / 32, ksub = warp % S::KS, share = cta * S::KS + ksub, shares = ctas * S::KS;
        const int u_low = (int)((int64_t)units * share / shares), u_high = (int)((int64_t)units * (share + 1) / shares);
        for (int tb = warp / S::KS * S::TB; tb < tiles; tb += S::TS * S::TB) {
            float acc[S::TB][NT][4] = {};
            const uint16_t *from[S::TB][2];
#pragma unroll
            for (int i = 0; i < S::TB; ++i)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int t = (tb + i) / per, j = (tb + i - t * per) * 16 + 8 * k + g;
                    from[i][k] = tb + i < tiles && j < r ? (const uint16_t *)wa + ((int64_t)(t0 + t) * a.rank + j) * a.inputs + 8 * c : nullptr;
                }
#pragma unroll 2
            for (int u = u_low; u < u_high; ++u) {
                const bool in = 32 * u + 8 * c < a.inputs;
                uint4 w[S::TB][2];
#pragma unroll
                for (int i = 0; i < S::TB; ++i)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        w[i][k] = make_uint4(0, 0, 0, 0);
                        if (in && from[i][k]) w[i][k] = __ldg((const uint4 *)(from[i][k] + 32 * u));
                    }
                uint32_t high[NT][8], low[NT][8];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float v[8] = {};
                    if (in && row[n] >= 0) kv_load8(a.x, row[n] * a.x_stride + 32 * u + 8 * c, TX, a.x_vectors, v);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        if constexpr (TX == KV_F32) lora_split(v[e], &high[n][e], &low[n][e]);
                        else high[n][e] = __float_as_uint(v[e]);
                    }
                }
#pragma unroll
                for (int i = 0; i < S::TB; ++i) {
                    if (tb + i >= tiles) break;
                    uint32_t p[8], q[8];
                    lora_weights<TW>(w[i][0], p);
                    lora_weights<TW>(w[i][1], q);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float d[4] = {};
#pragma unroll
                        for (int e = 0; e < 8; e += 2)             // the small parts first, as each step cuts the whole sum off
                            if constexpr (TX == KV_F32) lora_mma(d, p[e], q[e], p[e + 1], q[e + 1], low[n][e], low[n][e + 1]);
#pragma unroll
                        for (int e = 0; e < 8; e += 2) lora_mma(d, p[e], q[e], p[e + 1], q[e + 1], high[n][e], high[n][e + 1]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[i][n][e] = fadd(acc[i][n][e], d[e]);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < S::TB; ++i) {
                if (tb + i >= tiles) break;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float *const to = part + ksub * S::PART + (16 * (tb + i) + g) * COLS + 8 * n + 2 * c;
                    *(float2 *)to = make_float2(acc[i][n][0], acc[i][n][1]);
                    *(float2 *)(to + 8 * COLS) = make_float2(acc[i][n][2], acc[i][n][3]);
                }
            }
        }
    }
    __syncthreads();
    for (int i = tid; i < 16 * tiles * COLS; i += LORA_THREADS) {
        float v = part[i];
#pragma unroll
        for (int k = 1; k < S::KS; ++k) v = fadd(v, part[k * S::PART + i]);
        sum[i] = v;
    }
    lora_cluster_arrive();
    lora_cluster_wait();
    const int rp = (r + 31) / 32 * 32;
    for (int i = tid; i < rp * (t1 - t0) * COLS; i += LORA_THREADS) {
        const int col = i % COLS, at = i / COLS, t = at / rp, j = at - t * rp;
        float v = 0.0f;
        if (j < r) {
            float p[8];                                            // asked for all at once
#pragma unroll
            for (int k = 0; k < 8; ++k) p[k] = k < ctas ? lora_peer(sum + (t * per * 16 + j) * COLS + col, k) : 0.0f;
#pragma unroll
            for (int k = 0; k < 8; ++k) v = fadd(v, p[k]);
        }
        h[col * S::HS + at] = v;
    }
    lora_cluster_arrive();                                         // the peers' sums are read; they may go once all CTAs are here
    __syncthreads();

    int target = t0, tile0 = 0, n_target = n_first;                // the tile's target, its first tile and output
    for (int tile = tile_low + warp; tile < tile_high; tile += LORA_WARPS) {
        while (tile - tile0 >= (a.width[target] + 15) / 16) {
            tile0 += (a.width[target] + 15) / 16;
            n_target += a.width[target];
            ++target;
        }
        const int n = (tile - tile0) * 16 + 2 * g, left = a.width[target] - n;       // the lane's outputs n and n + 1
        const uint16_t *const from = (const uint16_t *)wb + ((int64_t)n_target + n) * a.rank + 8 * c;
        float2 was[NT][2];
        int64_t orow[NT][2];
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int col = 8 * i + 2 * c + k;
                orow[i][k] = col < count && left > 0 ? lora_row(a, order, first + col) : -1;
                was[i][k] = make_float2(0.0f, 0.0f);
                if (a.base && orow[i][k] >= 0) was[i][k] = lora_load2<TX>(a.base, orow[i][k] * a.base_stride + n_target + n, left > 1, a.pairs);
            }
        float acc[NT][4] = {};
        for (int j = 0; j < rp; j += 32) {
            uint4 w[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                w[k] = make_uint4(0, 0, 0, 0);
                if (left > k && j + 8 * c < r) w[k] = __ldg((const uint4 *)(from + k * a.rank + j));
            }
            uint32_t p[8], q[8];
            lora_weights<TW>(w[0], p);
            lora_weights<TW>(w[1], q);
            if (j + 8 * c + 8 > r)                                 // what lies past the adapter's own rank may be anything
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (j + 8 * c + e >= r) p[e] = q[e] = 0;
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const float *const at = h + (8 * i + g) * S::HS + (target - t0) * rp + j + 8 * c;
                const float4 h0 = *(const float4 *)at, h1 = *(const float4 *)(at + 4);
                const float v[8] = {h0.x, h0.y, h0.z, h0.w, h1.x, h1.y, h1.z, h1.w};
                float d[4] = {}, small[4] = {};                    // the small parts' sums apart, as each step cuts the whole sum off
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    uint32_t high[2], low[2];
                    lora_split(v[e], &high[0], &low[0]);
                    lora_split(v[e + 1], &high[1], &low[1]);
                    lora_mma(d, p[e], q[e], p[e + 1], q[e + 1], high[0], high[1]);
                    lora_mma(small, p[e], q[e], p[e + 1], q[e + 1], low[0], low[1]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][e] = fadd(acc[i][e], fadd(small[e], d[e]));
            }
        }
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int k = 0; k < 2; ++k)
                if (orow[i][k] >= 0)
                    lora_store2<TX>(a.out, orow[i][k] * a.out_stride + n_target + n,
                                    make_float2(__fmaf_rn(scale, acc[i][k], was[i][k].x), __fmaf_rn(scale, acc[i][2 + k], was[i][k].y)), left > 1, a.pairs);
    }
    lora_cluster_wait();
}

}  // namespace nc
