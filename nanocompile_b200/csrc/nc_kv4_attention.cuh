// nc_kv4_attention.cuh -- attention of query rows over a paged 4-bit cache (nc_kv4.cuh).
//
//   out[r, h] = sum_t softmax_t(scale * q[r, h] . k[t, h / G]) v[t, h / G],  t = 0 .. position of row r,
// with q rotated (RoPE) where there is a table; zeros, and a log-sum of -inf, for a row that sees nothing.
//
// The products are matrix instructions on the codes themselves.  A code c in the low bits of an f16 is the
// subnormal c 2^-24, in bits 4-7 it is 16 c 2^-24, so one AND makes a pair of operands from packed codes,
// exactly; the 2^-24 and the 16 go into the queries.  The blocks' parameters stay outside the products:
//   q . k[t]   = sum_b scale_k[t, b] (q . code)_b + zero_k[t, b] (sum of q over b)
//   sum p v    = sum_b (p[t] scale_v[t, b]) (code - 7.5)  + (sum_t p[t] (zero_v + 7.5 scale_v)[t, b])
// the first of each line by mma m16n8k16 (S^T = K Q^T with positions as rows; O^T = V^T P^T), the rest in
// 32 bits.  Values average to little where their codes average to 7.5 scales: without the 7.5 the two sums
// of the second line would cancel.
//
// Accuracy.  The matrix unit truncates its sums, at a place set by its operands' exponent fields: a sum of
// products with subnormals loses up to ten bits.  So the values' codes are brought to normal numbers by the
// subtraction of the 7.5 (one FMA for two), and the scores of float32 and float16 callers (HL) are made exact:
// q is brought below 2^11 by a power of two and split into two whole numbers q = hi + lo 2^-11 of at most 11
// bits, whose 32 products with a code fit the unit's bits, in an accumulator for each part.  p scale_v is split
// into two f16 parts (22 bits), summed over one step and added to the running sum in float32.
// bfloat16 callers take one f16 part of q, of p and of p scale_v, and have the parameters' sums made by the matrix unit
// too: sum_b zero_k (sum of q over b) with the sums of q in two parts, sum_t p zero_v and sum_t p scale_v as eight more rows.
//
// Probabilities are held relative to ref = (running maximum) - k, where k lifts p scale_v to just below
// 2^15 for the largest scale_v seen (k <= 15): any power of two cancels in sum p v / sum p, so the f16 range
// costs nothing and no size of input leaves it.
//
// A CTA has the columns (row, head of the group) of one kv head, 8 NT of them; its warps take steps of 64
// or 32 positions in turn, each with its own reference and sums, and meet in shared memory at the end.  A warp
// copies its steps into its own ring of stages (cp.async, from before the queries are ready) and waits for
// nobody else.  Few columns and a long cache are split over CTAs as well (chunks of whole steps); the last
// CTA to finish joins the parts in their order, so results do not depend on the schedule.
//
// Measured (us; memory's floor for the cache in brackets): one sequence of 97 positions and 14 heads on 2 of 64 5.8, the
// start and two steps; 64 of 2048 12.2 (3.3), the latency of the two steps that each of 2048 warps makes; bfloat16, 24
// sequences of up to 16384 and 32 heads on 8 of 128 87 (43), the instruction rate, with lengths that differ; 512 rows of a
// prompt 17.8 (0.6).
#pragma once

#include <type_traits>

#include "nc_kv4.cuh"

namespace nc {

// Tiles that a warp takes at a time: about 5 KB, and few enough values in registers for 16 warps on an SM.
__host__ __device__ constexpr int kv4_step_tiles(int d) { return d <= 64 ? 4 : 2; }

struct Kv4AttnArgs {
    Kv4Rows at;
    Kv4Pool pool;
    void *out;                         // [rows][heads][d]
    const void *q;                     // [rows][heads][d]
    const float *cos_tab, *sin_tab;    // [positions][d / 2] or null
    float *lse;                        // [rows][heads] or null
    unsigned int *counter;             // [groups], zero before the call and after it
    float *part;                       // [groups][splits][8 NT][d + 2]
    int64_t q_stride, out_stride, positions;
    uint64_t page_magic;               // ceil(2^37 / tiles of a page): the tile's page by a multiplication
    float scale_log2e;
    int type, heads, group, col_blocks, splits, chunk;   // chunk: steps of a split; splits * chunk steps hold max_length
    int max_rows, max_length;
};

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], const uint2 &b) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y));
}
__device__ __forceinline__ void mma_f16_k8(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(b));
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t max_f16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
// Pairs of codes less 7.5, times 2^-9 (exact), from c 2^-24 (multiplier 2^15) or 16 c 2^-24 (2^11).
__device__ __forceinline__ uint32_t centred(uint32_t v, uint32_t multiplier) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(v), "r"(multiplier), "r"(0xa380a380u));
    return r;
}
constexpr uint32_t CODE_LOW = 0x78007800u, CODE_HIGH = 0x68006800u;
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_f16(float low, float high) {
    const __half2 h = __floats2half2_rn(low, high);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float2 unpack_f16(uint32_t v) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&v));
}
// Whether a block's parameters are those of a NaN (no others are not finite).
__device__ __forceinline__ bool nan_params(uint32_t w) { return (w & 0x7fffu) > 0x7c00u || (w >> 16 & 0x7fffu) > 0x7c00u; }
// 2^e for -126 <= e <= 127.
__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

__device__ __forceinline__ void copy16_async(void *smem, const void *global) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(smem)), "l"(global)
                 : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Four dimensions from i on of a row and head: value / sum; and the log-sum, of sums relative to 2^base.
template <int D>
__device__ __forceinline__ void kv4_finish(const Kv4AttnArgs &a, int2 row_head, int i, const float4 &v, float sum, float base) {
    const float inv = sum == 0.0f ? 0.0f : fdiv(1.0f, sum);
    const int64_t at = row_head.x * a.out_stride + (int64_t)row_head.y * D + i;
    if (sum == 0.0f) {
#pragma unroll
        for (int k = 0; k < 4; ++k) kv_store(a.out, at + k, a.type, 0.0f);
    } else {
        kv_store(a.out, at, a.type, fmul(v.x, inv));
        kv_store(a.out, at + 1, a.type, fmul(v.y, inv));
        kv_store(a.out, at + 2, a.type, fmul(v.z, inv));
        kv_store(a.out, at + 3, a.type, fmul(v.w, inv));
    }
    if (i == 0 && a.lse)
        a.lse[(int64_t)row_head.x * a.heads + row_head.y] = sum == 0.0f ? -INFINITY : fmul(base + log2f(sum), 0.6931471805599453f);
}

// Joins the parts of a group's splits, in their order: [active][COLS][D] values, then [COLS] (reference, sum) in each.
template <int COLS, int D>
__device__ __forceinline__ void kv4_join(const Kv4AttnArgs &a, const float *parts, int active, int ncol, const int2 *rows) {
    for (int at = threadIdx.x; at < ncol * (D / 4); at += blockDim.x) {
        const int col = at / (D / 4), i = at % (D / 4) * 4;
        float base = -INFINITY, sum = 0.0f;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int s0 = 0; s0 < active; s0 += 8) {                       // eight parts' loads at a time
            float2 rl[8];
            float4 y[8];
            float to = base;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float *const p = parts + (int64_t)min(s0 + k, active - 1) * (COLS * (D + 2));
                rl[k] = __ldcg((const float2 *)(p + COLS * D + 2 * col));
                y[k] = __ldcg((const float4 *)(p + col * D + i));
                if (s0 + k >= active) rl[k] = make_float2(-INFINITY, 0.0f);
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) to = fmaxf(to, rl[k].x);
            const float old = base == -INFINITY ? 0.0f : fast_exp2(base - to);
            v.x *= old, v.y *= old, v.z *= old, v.w *= old;
            sum *= old;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float x = rl[k].x == -INFINITY ? 0.0f : fast_exp2(rl[k].x - to);
                if (s0 + k < active) {
                    v.x = __fmaf_rn(y[k].x, x, v.x);
                    v.y = __fmaf_rn(y[k].y, x, v.y);
                    v.z = __fmaf_rn(y[k].z, x, v.z);
                    v.w = __fmaf_rn(y[k].w, x, v.w);
                    sum = __fmaf_rn(rl[k].y, x, sum);
                }
            }
            base = to;
        }
        kv4_finish<D>(a, rows[col], i, v, sum, base);
    }
}

template <int D, int NT, bool HL, int W, int ST>
struct Kv4AttnShape {
    static constexpr int NB = D / 32, VB = kv4_vb(NB), COLS = 8 * NT, PARTS = HL ? 2 : 1;
    static constexpr int TILES = kv4_step_tiles(D), STEP = TILES * KV4_TILE;   // positions of a step
    static constexpr int MT = TILES < 4 / NT ? TILES : 4 / NT;         // tiles whose scores are held at a time
    static constexpr int STAGE = TILES * 20 * D;                       // bytes
    static constexpr int RING = W * ST * STAGE;
    static constexpr int MERGE = W * COLS * (D + 2) * 4;               // shares the ring's bytes
    static constexpr int BODY = RING > MERGE ? RING : MERGE;
    static constexpr int QF = NB * 2 * NT * PARTS * 32 * 8;
    static constexpr int SMEM = BODY + QF + COLS * (NB + 4) * 4 + NT * 32 * 4;
    static constexpr int CTAS = (NT == 1 ? 16 : 8) / W;              // wanted on an SM
};

template <int D, int NT, bool HL, int W, int ST>
__global__ void __launch_bounds__(32 * W, (Kv4AttnShape<D, NT, HL, W, ST>::CTAS)) kv4_attention_kernel(const __grid_constant__ Kv4AttnArgs a) {
    using S = Kv4AttnShape<D, NT, HL, W, ST>;
    constexpr int NB = S::NB, VB = S::VB, COLS = S::COLS, MT = S::MT, TILES = S::TILES, STEP = S::STEP;
    constexpr int ZB = NB == 3 ? 4 : NB;                               // places of a k8 operand for the blocks' zeros
    extern __shared__ __align__(128) char smem[];
    uint2 *const qf = (uint2 *)(smem + S::BODY);                       // [block][half][nt][part][lane]
    float *const qsum = (float *)(smem + S::BODY + S::QF);             // [block][col]
    float *const qscale = qsum + NB * COLS;                            // [col]
    int2 *const qrow = (int2 *)(qscale + COLS);                        // [col] row and head
    int *const qpos = (int *)(qrow + COLS);                            // [col]
    uint32_t *const qz = (uint32_t *)(qpos + COLS);                    // [nt][lane]: sums of q as B operands (not HL)
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;

    release_dependents();
    wait_for_producer();
    const int split = (int)(blockIdx.x % a.splits);
    const unsigned group = blockIdx.x / a.splits;
    const int cb = a.col_blocks - 1 - (int)(group / a.pool.kv / a.at.seqs);   // the rows that see most first
    const int head = (int)(group % a.pool.kv);
    const int seq = (int)(group / a.pool.kv % a.at.seqs);
    const int length = a.at.lengths[seq];
    const int row0 = a.at.row_start ? a.at.row_start[seq] : seq;
    const int nr = a.at.row_start ? a.at.row_start[seq + 1] - row0 : 1;
    if (row0 < 0 || nr <= 0 || (int64_t)row0 + nr > a.at.rows) return;
    const int cols = min(nr, a.max_rows) * a.group, col0 = cb * COLS;  // the entry point bounds rows * group
    if (col0 >= cols) return;
    const int ncol = min(cols - col0, COLS);
    // Positions 0 .. end - 1 are seen by the block's last row, all of 0 .. first by every row of it: none where a row has no angle.
    const int last = length - nr + (col0 + ncol - 1) / a.group;
    const int first = a.cos_tab && last >= a.positions ? -1 : min(length - nr + col0 / a.group, a.max_length - 1);
    const int end = min(last < 0 ? 0 : last + 1, a.max_length);
    const int steps = (end + STEP - 1) / STEP;
    const int active = steps <= a.chunk ? 1 : (steps + a.chunk - 1) / a.chunk;
    if (split >= active) return;

    // The queries of a column: what they are made of, on its way before the tables of pages are looked at ..
    struct Query {
        float x[NB], y[NB], cos[NB], sin[NB];                          // the values, their partners, the angles
        int row, h, pos;
        bool known;
    };
    auto load_query = [&](int col) {
        Query q;
        const bool have = col < ncol;
        const int r = have ? (col0 + col) / a.group : 0;
        q.row = row0 + r;
        q.h = head * a.group + (have ? col0 + col - r * a.group : 0);
        q.pos = have ? length - nr + r : -1;
        q.known = q.pos >= 0 && (!a.cos_tab || q.pos < a.positions);
        if (q.pos >= 0 && !q.known && a.at.error && lane == 0) atomicMin(a.at.error, (unsigned long long)seq);
        const int64_t at = q.row * a.q_stride + (int64_t)q.h * D;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int i = 32 * b + lane;
            q.x[b] = q.known ? kv_load(a.q, at + i, a.type) : 0.0f;
            q.y[b] = q.cos[b] = q.sin[b] = 0.0f;
            if (q.known && a.cos_tab) {
                q.y[b] = kv_load(a.q, at + (i < D / 2 ? i + D / 2 : i - D / 2), a.type);
                q.cos[b] = a.cos_tab[(int64_t)q.pos * (D / 2) + (i < D / 2 ? i : i - D / 2)];
                q.sin[b] = a.sin_tab[(int64_t)q.pos * (D / 2) + (i < D / 2 ? i : i - D / 2)];
            }
        }
        return q;
    };
    // .. and then: rotated, brought to the f16 range, in the B operand's order.
    auto put_query = [&](int col, const Query &q) {
        float v[NB];
        uint32_t mag = 0;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int i = 32 * b + lane;
            v[b] = q.x[b];
            if (a.cos_tab)
                v[b] = i < D / 2 ? fsub(fmul(q.x[b], q.cos[b]), fmul(q.y[b], q.sin[b])) : fadd(fmul(q.x[b], q.cos[b]), fmul(q.y[b], q.sin[b]));
            mag = max(mag, __float_as_uint(v[b]) & 0x7fffffffu);
        }
        mag = __reduce_max_sync(0xffffffffu, mag);
        int e = 0;                                                     // |q| 2^e < 2^11, or 2^15 for one part
        if (mag != 0 && mag < 0x7f800000u) e = (HL ? 10 : 14) - ((int)(mag >> 23) - 127);
        e = e < -100 ? -100 : e > 100 ? 100 : e;
        if (lane == 0) {
            qscale[col] = fmul(a.scale_log2e, pow2i(24 - e));
            qrow[col] = make_int2(q.row, q.h);
            qpos[col] = q.known ? min(q.pos, a.max_length - 1) : -1;   // the last position that the row sees
        }
        const bool bad = mag >= 0x7f800000u;                           // an infinity or a NaN: it has to show in the sums too
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const float x = fmul(v[b], pow2i(e));
            const float hi = HL ? rintf(x) : __half2float(__float2half_rn(x));
            const float lo = HL ? rintf(fmul(x - hi, 2048.0f)) : 0.0f;
            // The block's sum: of whole numbers, at most 2^11 and 2^10, or 2^24 for x in steps of 2^-9.
            float sum;
            if (HL) {
                const int high = __reduce_add_sync(0xffffffffu, (int)hi), low = __reduce_add_sync(0xffffffffu, (int)lo);
                sum = __fmaf_rn((float)low, 0x1p-11f, (float)high);
            } else {
                sum = fmul((float)__reduce_add_sync(0xffffffffu, __float2int_rn(fmul(x, 512.0f))), 0x1p-9f);
            }
            if (bad) sum = __uint_as_float(0x7fc00000u);
            if (lane == 0) qsum[b * COLS + col] = fmul(sum, 0x1p-24f);
            if (!HL && lane < 2) {                                     // k = b its f16 part, k = ZB + b the rest
                const float z = fmul(sum, 0x1p-24f);
                const __half part = __float2half_rn(z);
                const int k = b + lane * ZB;
                ((__half *)(qz + (col >> 3) * 32 + 4 * (col & 7) + (k >> 1)))[k & 1] = lane ? __float2half_rn(z - __half2float(part)) : part;
            }
            // dimension 8 c' + i of the block: nibble i -> k half (i >> 1) & 1, register i & 1, f16 half i >> 2
            const int i = lane & 7, cc = lane >> 3;
            const float unit = (i & 1) ? 0.0625f : 1.0f;
            const int at = (((b * 2 + ((i >> 1) & 1)) * NT + (col >> 3)) * S::PARTS) * 32 + 4 * (col & 7) + cc;
            __half *const to = (__half *)(qf + at) + (i & 1) * 2 + (i >> 2);
            *to = __float2half_rn(fmul(hi, unit));
            if (HL) to[32 * 4] = __float2half_rn(fmul(lo, unit));
        }
    };
    constexpr int OWN = COLS / W > 0 ? COLS / W : 1;                   // columns of a warp
    Query ahead[OWN < 2 ? OWN : 2];
    if (warp < COLS) {
        ahead[0] = load_query(warp);
        if (OWN > 1) ahead[OWN > 1] = load_query(warp + W);
    }

    char *const ring = smem + warp * ST * S::STAGE;
    const int step0 = split * a.chunk + warp, step_end = min(steps, split * a.chunk + a.chunk);
    const int tiles_per_page = a.at.page / KV4_TILE;
    const int32_t *const table = a.at.table + (int64_t)seq * a.at.width;
    // The page of the lane's tile (lane % TILES) of a step, by the table alone: nothing here waits for what is read.  -2: no
    // such tile.
    auto page_of = [&](int step) {
        const int tile = step * TILES + lane % TILES;
        int page = -2;
        if (step < step_end && tile * KV4_TILE < end) {
            const int j = (int)((uint64_t)tile * a.page_magic >> 37);
            page = -1;
            if (j < a.at.width) page = table[j];
        }
        return page;
    };
    // Where it lies; null where there is none (reported).
    auto tile_at = [&](int step, int page) -> const char * {
        const int tile = step * TILES + lane % TILES, j = (int)((uint64_t)tile * a.page_magic >> 37);
        if (page < 0 || page >= a.at.pages) {
            if (page != -2 && a.at.error) atomicMin(a.at.error, (unsigned long long)seq);
            return nullptr;
        }
        return a.pool.base + page * a.pool.page_bytes + ((int64_t)head * tiles_per_page + (tile - j * tiles_per_page)) * (20 * D);
    };
    auto issue = [&](int stage, const char *from) {
        constexpr int PIECES = 20 * D / 16;                            // 16-byte pieces of a tile
        char *const to = ring + stage * S::STAGE;
#pragma unroll
        for (int k = 0; k < TILES; ++k) {
            const char *const src = (const char *)__shfl_sync(0xffffffffu, (unsigned long long)from, k);
            if (src)
#pragma unroll
                for (int i = 0; i < (PIECES + 31) / 32; ++i)
                    if (i * 32 + 32 <= PIECES || i * 32 + lane < PIECES)
                        copy16_async(to + k * 20 * D + (i * 32 + lane) * 16, src + (i * 32 + lane) * 16);
        }
    };
    uint32_t held[ST];                                                 // which tiles of the steps in flight are there
    int next = step0;
    int pages[ST];
#pragma unroll
    for (int s = 0; s < ST; ++s) pages[s] = page_of(step0 + s * W);
#pragma unroll
    for (int s = 0; s < ST - 1; ++s) {
        const char *const from = tile_at(next, pages[s]);
        held[s] = __ballot_sync(0xffffffffu, from != nullptr);
        issue(s, from);
        copies_commit();
        next += W;
    }
    int page_next = pages[ST - 1];

    if (!HL) {                                                         // the places of no block
        for (int i = threadIdx.x; i < NT * 32; i += 32 * W) qz[i] = 0;
        __syncthreads();
    }
    if (warp < COLS) {
#pragma unroll
        for (int k = 0; k < OWN; k += 2) {
            Query more[2];
            if (k + 2 < OWN) {
                more[0] = load_query(warp + (k + 2) * W);
                more[1] = load_query(warp + (k + 3) * W);
            }
            put_query(warp + k * W, ahead[0]);
            if (OWN > 1) put_query(warp + (k + 1) * W, ahead[OWN > 1]);
            if (k + 2 < OWN) {
                ahead[0] = more[0];
                ahead[OWN > 1] = more[1];
            }
        }
    }
    __syncthreads();

    constexpr int OZ = HL ? NB : 1;                                    // sums of zeros: by block, or rows g of one operand
    float ref[NT][2], l[NT][2], o[NB][2][NT][4], oz[OZ][NT][2];
    float f[NT][2];
    int pos[NT][2];
    int lift = 15;                                                     // k: the same for all columns
    float top[NT][2];                                                  // the running maximum
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int col = 8 * nt + 2 * c + e;
            top[nt][e] = ref[nt][e] = -INFINITY;
            l[nt][e] = 0.0f;
            f[nt][e] = qscale[col];
            pos[nt][e] = qpos[col];
        }
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            oz[b % OZ][nt][0] = oz[b % OZ][nt][1] = 0.0f;
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[b][k][nt][e] = 0.0f;
        }

    int stage = 0;
#pragma unroll 1
    for (int step = step0; step < step_end; step += W) {
        // Start the copies ST - 1 steps ahead, into the stage that the last step read.
        const char *const from = tile_at(next, page_next);
        issue(stage == 0 ? ST - 1 : stage - 1, from);
        copies_commit();
        held[ST - 1] = __ballot_sync(0xffffffffu, from != nullptr);
        next += W;
        page_next = page_of(next);
        copies_wait<ST - 1>();
        __syncwarp();
        const uint32_t whole = held[0];
#pragma unroll
        for (int s = 0; s + 1 < ST; ++s) held[s] = held[s + 1];
        const char *const buf = ring + stage * S::STAGE;
        const bool at_edge = (step + 1) * STEP > first + 1 || whole != 0xffffffffu;

        // EDGE: some position of the step is past the end, masked for some row, or has no page.
        auto body = [&](auto edge_tag, int sub) {
            constexpr bool EDGE = decltype(edge_tag)::value;
            const char *const tiles = buf + sub * 20 * D;
            const int t0 = step * STEP + sub * KV4_TILE + g;           // the lane's positions: t0 + 16 mt + 8 k
            // Whether there is anything at position t0 - g + i of tile mt.
            auto there = [&](int mt, int i) { return (whole >> (sub + mt) & 1) != 0 && t0 - g + 16 * mt + i < end; };
            float sc[MT][NT][4];
            if constexpr (!HL) {
                // Scores begin with the zeros' part.
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    uint32_t z0, z1;                                   // zeros of positions g and 8 + g, blocks 2 c and 2 c + 1
                    const uint32_t *const par = (const uint32_t *)(tiles + mt * 20 * D + 8 * D) + g * NB * 2;
                    if constexpr (NB == 1) {
                        const uint2 w = *(const uint2 *)par;
                        z0 = __byte_perm(w.x, w.x, 0x3232);
                        z1 = __byte_perm(w.y, w.y, 0x3232);
                    } else {
                        const int b = NB == 2 ? 0 : 2 * (c & 1);
                        const uint2 w = *(const uint2 *)(par + b * 2);
                        const uint2 v = NB == 3 && b == 2 ? make_uint2(0, 0) : *(const uint2 *)(par + (NB == 3 && b == 2 ? 0 : b + 1) * 2);
                        z0 = __byte_perm(w.x, v.x, 0x7632);
                        z1 = __byte_perm(w.y, v.y, 0x7632);
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        sc[mt][nt][0] = sc[mt][nt][1] = sc[mt][nt][2] = sc[mt][nt][3] = 0.0f;
                        mma_f16_k8(sc[mt][nt], z0, z1, qz[nt * 32 + lane]);
                    }
                }
            }
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                uint32_t ka[MT][2][4];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    const uint2 w = *(const uint2 *)(tiles + mt * 20 * D + kv4_code_word(VB, b, lane, 0) * 4);
                    ka[mt][0][0] = w.x & 0x000f000fu;
                    ka[mt][0][1] = w.y & 0x000f000fu;
                    ka[mt][0][2] = w.x & 0x00f000f0u;
                    ka[mt][0][3] = w.y & 0x00f000f0u;
                    ka[mt][1][0] = w.x >> 8 & 0x000f000fu;
                    ka[mt][1][1] = w.y >> 8 & 0x000f000fu;
                    ka[mt][1][2] = w.x >> 8 & 0x00f000f0u;
                    ka[mt][1][3] = w.y >> 8 & 0x00f000f0u;
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const uint2 *const qb = qf + (b * 2 * NT + nt) * S::PARTS * 32 + lane;
                    const uint2 q0 = qb[0], q1 = qb[NT * S::PARTS * 32];
                    const uint2 r0 = HL ? qb[32] : q0, r1 = HL ? qb[NT * S::PARTS * 32 + 32] : q1;
                    const float2 zs = HL ? *(const float2 *)(qsum + b * COLS + 8 * nt + 2 * c) : make_float2(0.0f, 0.0f);
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                        mma_f16(acc, ka[mt][0], q0);
                        mma_f16(acc, ka[mt][1], q1);
                        const uint2 par = *(const uint2 *)(tiles + mt * 20 * D + 8 * D + kv4_param_word(NB, b, g) * 4);
                        float *const s = sc[mt][nt];
                        if constexpr (HL) {
                            float low[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                            mma_f16(low, ka[mt][0], r0);
                            mma_f16(low, ka[mt][1], r1);
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc[e] = __fmaf_rn(low[e], 0x1p-11f, acc[e]);
                            const float2 p0 = unpack_f16(par.x), p1 = unpack_f16(par.y);     // (scale, zero)
                            s[0] = __fmaf_rn(p0.x, acc[0], b ? __fmaf_rn(p0.y, zs.x, s[0]) : fmul(p0.y, zs.x));
                            s[1] = __fmaf_rn(p0.x, acc[1], b ? __fmaf_rn(p0.y, zs.y, s[1]) : fmul(p0.y, zs.y));
                            s[2] = __fmaf_rn(p1.x, acc[2], b ? __fmaf_rn(p1.y, zs.x, s[2]) : fmul(p1.y, zs.x));
                            s[3] = __fmaf_rn(p1.x, acc[3], b ? __fmaf_rn(p1.y, zs.y, s[3]) : fmul(p1.y, zs.y));
                        } else {
                            const float p0 = unpack_f16(par.x).x, p1 = unpack_f16(par.y).x;
                            s[0] = __fmaf_rn(p0, acc[0], s[0]);
                            s[1] = __fmaf_rn(p0, acc[1], s[1]);
                            s[2] = __fmaf_rn(p1, acc[2], s[2]);
                            s[3] = __fmaf_rn(p1, acc[3], s[3]);
                        }
                    }
                }
            }
            // The values' parameters of positions g and 8 + g, and the lift that their largest scale allows.
            auto value_params = [&](int mt, int b) {
                uint2 w = *(const uint2 *)(tiles + mt * 20 * D + 18 * D + kv4_param_word(NB, b, g) * 4);
                if (EDGE) {                                            // past the end: whatever was there before
                    if (!there(mt, g)) w.x = 0;
                    if (!there(mt, 8 + g)) w.y = 0;
                }
                return w;
            };
            uint32_t big = 0;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const uint2 w = value_params(mt, b);
                    big = max_f16x2(big, max_f16x2(w.x, w.y));         // a NaN is passed over
                }
            big = __reduce_max_sync(0xffffffffu, big & 0x7fffu);       // scales are not negative; below 2^(exponent + 1)
            lift = min(lift, max(29 - (int)(big >> 10), -1));

            uint32_t seen[MT][NT];                                     // bits: score e of the tile counts
            float alpha[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float most[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    seen[mt][nt] = 15u;
                    if (EDGE) {                                        // masked scores are -inf
                        uint32_t ok = 0;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const bool in = (whole >> (sub + mt) & 1) != 0 && t0 + 16 * mt + 8 * (e >> 1) <= pos[nt][e & 1];
                            if (in) ok |= 1u << e;
                            else sc[mt][nt][e] = -INFINITY;
                        }
                        seen[mt][nt] = ok;
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) most[e & 1] = fmaxf(most[e & 1], sc[mt][nt][e]);
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) most[e] = fmaxf(most[e], __shfl_xor_sync(0xffffffffu, most[e], x));
                    top[nt][e] = fmaxf(top[nt][e], fmul(most[e], f[nt][e]));
                    const bool none = top[nt][e] == -INFINITY;         // nothing seen so far: no reference yet
                    const float base = none ? 0.0f : top[nt][e] - (float)lift;
                    alpha[nt][e] = fast_exp2(ref[nt][e] - base);       // 0 at the first position seen
                    ref[nt][e] = none ? -INFINITY : base;
                    float sum = 0.0f;
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            float &s = sc[mt][nt][2 * k + e];
                            s = fast_exp2(__fmaf_rn(s, f[nt][e], -base));
                            sum += s;
                        }
                    l[nt][e] = __fmaf_rn(l[nt][e], alpha[nt][e], sum);
                }
            }
            // P V, block by block.
            uint2 ph[MT][NT];                                          // not HL: p as B operands, positions 2 c, 2 c + 1, ..
            if constexpr (!HL) {
                float zacc[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) zacc[nt][0] = zacc[nt][1] = zacc[nt][2] = zacc[nt][3] = 0.0f;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    // Rows b: the zeros of block b, rows 4 + b: its scales, at positions 2 c, 2 c + 1, 8 + 2 c, 8 + 2 c + 1.
                    const uint32_t *const par = (const uint32_t *)(tiles + mt * 20 * D + 18 * D) + (2 * c * NB + (g & 3)) * 2;
                    const bool row = NB == 4 || (g & 3) < NB;
                    uint2 w = row ? *(const uint2 *)par : make_uint2(0, 0), v = row ? *(const uint2 *)(par + 2 * NB) : make_uint2(0, 0);
                    if (EDGE) {                                        // nothing there, or a NaN: that is dealt with below
                        if (!there(mt, 2 * c) || nan_params(w.x)) w.x = 0;
                        if (!there(mt, 8 + 2 * c) || nan_params(w.y)) w.y = 0;
                        if (!there(mt, 2 * c + 1) || nan_params(v.x)) v.x = 0;
                        if (!there(mt, 9 + 2 * c) || nan_params(v.y)) v.y = 0;
                    }
                    const uint32_t pick = g < 4 ? 0x7632 : 0x5410;
                    const uint32_t za[4] = {__byte_perm(w.x, v.x, pick), 0, __byte_perm(w.y, v.y, pick), 0};
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        ph[mt][nt] = make_uint2(transpose_8x8(pack_f16(sc[mt][nt][0], sc[mt][nt][1])),
                                                transpose_8x8(pack_f16(sc[mt][nt][2], sc[mt][nt][3])));
                        mma_f16(zacc[nt], za, ph[mt][nt]);
                    }
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    oz[0][nt][0] = __fmaf_rn(oz[0][nt][0], alpha[nt][0], zacc[nt][0]);
                    oz[0][nt][1] = __fmaf_rn(oz[0][nt][1], alpha[nt][1], zacc[nt][1]);
                }
            }
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                float acc[2][NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    if (HL) {
                        oz[b % OZ][nt][0] = fmul(oz[b % OZ][nt][0], alpha[nt][0]);
                        oz[b % OZ][nt][1] = fmul(oz[b % OZ][nt][1], alpha[nt][1]);
                    }
#pragma unroll
                    for (int k = 0; k < 2; ++k)
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[k][nt][e] = 0.0f;
                }
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    const uint2 w = *(const uint2 *)(tiles + mt * 20 * D + 10 * D + kv4_code_word(VB, b, lane, 0) * 4);
                    uint32_t va[2][4];
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const uint32_t x = k ? w.x >> 8 : w.x, y = k ? w.y >> 8 : w.y;
                        va[k][0] = centred(x & 0x000f000fu, CODE_LOW);
                        va[k][1] = centred(x & 0x00f000f0u, CODE_HIGH);
                        va[k][2] = centred(y & 0x000f000fu, CODE_LOW);
                        va[k][3] = centred(y & 0x00f000f0u, CODE_HIGH);
                    }
                    if constexpr (HL) {
                        const uint2 vp = value_params(mt, b);
                        float2 par[2] = {unpack_f16(vp.x), unpack_f16(vp.y)};   // (scale, zero)
                        par[0].y = __fmaf_rn(7.5f, par[0].x, par[0].y);
                        par[1].y = __fmaf_rn(7.5f, par[1].x, par[1].y);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            float *const z = oz[b % OZ][nt];
                            uint2 hi, lo;
#pragma unroll
                            for (int k = 0; k < 2; ++k) {
                                const float p0 = sc[mt][nt][2 * k], p1 = sc[mt][nt][2 * k + 1];
                                float x0 = fmul(p0, par[k].x), x1 = fmul(p1, par[k].x);
                                float y0 = __fmaf_rn(p0, par[k].y, z[0]), y1 = __fmaf_rn(p1, par[k].y, z[1]);
                                if (EDGE) {                            // a masked position counts for nothing, NaN or not
                                    if (!(seen[mt][nt] >> (2 * k) & 1)) x0 = 0.0f, y0 = z[0];
                                    if (!(seen[mt][nt] >> (2 * k + 1) & 1)) x1 = 0.0f, y1 = z[1];
                                }
                                z[0] = y0;
                                z[1] = y1;
                                const uint32_t h = pack_f16(x0, x1);
                                (k ? hi.y : hi.x) = transpose_8x8(h);
                                const float2 back = unpack_f16(h);
                                (k ? lo.y : lo.x) = transpose_8x8(pack_f16(x0 - back.x, x1 - back.y));
                            }
                            mma_f16(acc[0][nt], va[0], hi);
                            mma_f16(acc[1][nt], va[1], hi);
                            mma_f16(acc[0][nt], va[0], lo);
                            mma_f16(acc[1][nt], va[1], lo);
                        }
                    } else {
                        const uint32_t *const par = (const uint32_t *)(tiles + mt * 20 * D + 18 * D) + (2 * c * NB + b) * 2;
                        uint2 even = *(const uint2 *)par, odd = *(const uint2 *)(par + 2 * NB);
                        if (EDGE) {
                            if (!there(mt, 2 * c) || nan_params(even.x)) even.x = 0;
                            if (!there(mt, 8 + 2 * c) || nan_params(even.y)) even.y = 0;
                            if (!there(mt, 2 * c + 1) || nan_params(odd.x)) odd.x = 0;
                            if (!there(mt, 9 + 2 * c) || nan_params(odd.y)) odd.y = 0;
                        }
                        const uint32_t s0 = __byte_perm(even.x, odd.x, 0x5410), s1 = __byte_perm(even.y, odd.y, 0x5410);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            const uint2 x = make_uint2(mul_f16x2(ph[mt][nt].x, s0), mul_f16x2(ph[mt][nt].y, s1));
                            mma_f16(acc[0][nt], va[0], x);
                            mma_f16(acc[1][nt], va[1], x);
                        }
                    }
                    if (EDGE && !HL) {                                 // a NaN's columns that see its position
                        const uint2 vp = value_params(mt, b);
                        const bool nan0 = nan_params(vp.x), nan1 = nan_params(vp.y);
                        if (__any_sync(0xffffffffu, nan0 || nan1)) {
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    const bool hit = (nan0 && (seen[mt][nt] >> e & 1)) || (nan1 && (seen[mt][nt] >> (2 + e) & 1));
                                    if (__ballot_sync(0xffffffffu, hit) & (0x11111111u << c))
                                        acc[0][nt][e] = acc[0][nt][2 + e] = acc[1][nt][e] = acc[1][nt][2 + e] = __uint_as_float(0x7fc00000u);
                                }
                        }
                    }
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int k = 0; k < 2; ++k)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            o[b][k][nt][e] = __fmaf_rn(o[b][k][nt][e], alpha[nt][e & 1], acc[k][nt][e]);
            }
        };
#pragma unroll 1
        for (int sub = 0; sub < TILES; sub += MT) {
            if (at_edge) body(std::true_type{}, sub);
            else body(std::false_type{}, sub);
        }
        __syncwarp();
        stage = stage + 1 == ST ? 0 : stage + 1;
    }
    copies_wait<0>();
    __syncthreads();

    // The warps' parts meet: [warp][col][D] values, then [warp][col] (reference, sum).
    const int busy = max(1, min(W, step_end - split * a.chunk));       // warps that had a step
    float *const mo = (float *)smem;
    float2 *const ml = (float2 *)(mo + W * COLS * D);
    if (warp < busy) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float sum = l[nt][e];
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
            const int col = 8 * nt + 2 * c + e;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                float z;
                if (HL) {
                    z = oz[b % OZ][nt][e];
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) z += __shfl_xor_sync(0xffffffffu, z, x);
                } else {                                               // rows b and 4 + b: of the zeros and of the scales
                    z = __fmaf_rn(7.5f, __shfl_sync(0xffffffffu, oz[0][nt][e], 4 * (4 + b) + c), __shfl_sync(0xffffffffu, oz[0][nt][e], 4 * b + c));
                }
                float4 v;                                              // 2^9: the codes' unit
                v.x = __fmaf_rn(o[b][0][nt][e], 512.0f, z);
                v.y = __fmaf_rn(o[b][0][nt][2 + e], 512.0f, z);
                v.z = __fmaf_rn(o[b][1][nt][e], 512.0f, z);
                v.w = __fmaf_rn(o[b][1][nt][2 + e], 512.0f, z);
                *(float4 *)(mo + ((warp * COLS + col) * D + 32 * b + 4 * g)) = v;
            }
            if (g == 0) ml[warp * COLS + col] = make_float2(ref[nt][e], sum);
        }
    }
    __syncthreads();

    // Four dimensions of a column to a thread; weights of the parts relative to their largest reference.
    const bool alone = active == 1;
    float *const part = alone ? nullptr : a.part + ((int64_t)group * a.splits + split) * (COLS * (D + 2));
    for (int at = threadIdx.x; at < ncol * (D / 4); at += 32 * W) {
        const int col = at / (D / 4), i = at % (D / 4) * 4;
        float base = -INFINITY;
#pragma unroll 4
        for (int w = 0; w < busy; ++w) base = fmaxf(base, ml[w * COLS + col].x);
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float sum = 0.0f;
#pragma unroll 4
        for (int w = 0; w < busy; ++w) {
            const float2 rl = ml[w * COLS + col];
            const float x = rl.x == -INFINITY ? 0.0f : fast_exp2(rl.x - base);
            const float4 y = *(const float4 *)(mo + (w * COLS + col) * D + i);
            v.x = __fmaf_rn(y.x, x, v.x);
            v.y = __fmaf_rn(y.y, x, v.y);
            v.z = __fmaf_rn(y.z, x, v.z);
            v.w = __fmaf_rn(y.w, x, v.w);
            sum = __fmaf_rn(rl.y, x, sum);
        }
        if (alone) {
            kv4_finish<D>(a, qrow[col], i, v, sum, base);
        } else {
            *(float4 *)(part + col * D + i) = v;
            if (i == 0) *(float2 *)(part + COLS * D + 2 * col) = make_float2(base, sum);
        }
    }
    if (alone) return;

    // The last CTA of the group joins the splits' parts, in their order.
    __shared__ unsigned int arrived;
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) arrived = atomicAdd(a.counter + group, 1u);
    __syncthreads();
    if (arrived != (unsigned)active - 1) return;
    __threadfence();
    if (threadIdx.x == 0) a.counter[group] = 0;
    kv4_join<COLS, D>(a, a.part + (int64_t)group * a.splits * (COLS * (D + 2)), active, ncol, qrow);
}

}  // namespace nc
