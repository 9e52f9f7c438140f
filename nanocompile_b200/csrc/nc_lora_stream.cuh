// nc_lora_stream.cuh -- low-rank adapters for single tokens: what nc_lora.cuh computes, for items of up to eight rows, as one stream of weights.
//
// An item to a cluster.  A CTA's part of the adapter, its share of A's inputs and then its share of B's outputs, comes through a
// ring of stages by bulk copies: 16 of A's rows by up to 512 inputs, or whole rows of B, to a stage.  Two warps ask for them, every other
// stage each, as a warp needs 40 ns for a copy.  Two teams of four warps multiply what has come, every other stage each, so that
// memory is busy from the start to the end: B is on its way while the CTAs add up their sums of h.  A stage gives a warp four
// units of 32 inputs, or two tiles of 16 outputs, at once: with one, its chain of loads, products and sums took as long.  The rows' shares
// of x are in shared memory from the start, as operands, and those of base where they fit.
//
// Bound by the adapters' bytes where each request has its own, beside a start of 10 us (the plan's words, x as operands, the sums'
// way through the cluster).  Adapters of 4096 inputs and outputs at rank 64 (1 MB each), bfloat16, with the plan: one 11.4 us, 16
// of them 13.2, 64 23.0 (3.0 TB/s), 128 44.7 (3.1 TB/s of 6.5: two rounds of clusters; 67 with one tile of outputs to a warp at a time).
//
// Accuracy.  Products are mma m16n8k16 of the weights' type.  Rows of that type are taken as they are, others and h go in parts: three of
// bfloat16 for float32 rows, which hold them, else two.  Two of bfloat16 hold float16 rows; of h they lose 2^-17 at most, where a bfloat16
// output is rounded by 2^-8, a float16 one by 2^-11.  Two of float16 lose 2^-23 at most, or 2^-39 of the row's largest: a row of x or h is
// first brought to [2^14, 2^15) by a power of two, so that no size leaves its range.  A chain of
// the matrix unit, which cuts sums off, is 32 inputs long, the largest parts last; chains are added in float32.
#pragma once

#include "nc_lora_tiles.cuh"

namespace nc {

constexpr int LS_WIDTH = 512;                  // inputs of a stage at most
constexpr int LS_LINE = LS_WIDTH * 2 + 16;     // bytes from a row of A to the next: no bank twice in a quarter of a warp
constexpr int LS_STAGE = 16 * LS_LINE, LS_B = 16 * 1024;               // bytes of a stage, and of B's rows in one
constexpr int LS_STAGES = 8, LS_TEAM = LORA_WARPS / 2, LS_ASKERS = 2, LS_THREADS = LORA_THREADS + 32 * LS_ASKERS;
constexpr int LS_BYTES = 110 * 1024;           // with two CTAs on an SM
static_assert(LS_STAGES % 2 == 0 && LS_ASKERS == 2 && LORA_WARPS == 2 * LS_TEAM, "two teams, and a warp that asks for each");
constexpr int LS_BASE = 8 * 1024;              // bytes for the rows' base
constexpr int LS_BYTES_ALONE = 2 * LS_BYTES - 4096;                    // with one CTA on an SM

template <int TX, int TW>
struct LoraStream {
    static constexpr bool F32 = TX == KV_F32, SCALED_X = TW == KV_F16 && TX != KV_F16, SCALED_H = TW == KV_F16;
    static constexpr int PX = TX == TW ? 1 : F32 && TW == KV_BF16 ? 3 : 2, PH = F32 && TW == KV_BF16 ? 3 : 2;
    static constexpr int SIZE = F32 ? 4 : 2;
};

// How shared memory is laid out, by the most tiles of 16 rows of h in a pass and the inputs of a CTA at most.
struct LoraStreamPlan {
    int stages, tiles;
    int x_line, h_line;                        // bytes from a row's operand to the next: whole 32s of inputs or of each target's h, and 16
    int part_at, sum_at, x_at, h_at, base_at, bytes;
    bool fits;
};
inline LoraStreamPlan lora_stream_plan(int targets, int rank, int inputs, int px, int ph) {
    LoraStreamPlan p{};
    p.tiles = targets * ((rank + 15) / 16);
    p.x_line = (inputs + 31) / 32 * 64 + 16;
    p.h_line = targets * ((rank + 31) / 32 * 64) + 16;
    const int part = LORA_WARPS * p.tiles * 512, sum = 8 * (p.tiles * 64 + 16), rest = part + sum + 8 * (px * p.x_line + ph * p.h_line) + LS_BASE;
    // An even number, that a stage is always the same team's: one that had skipped a round of a stage's barrier would take the
    // round before the one that it waits for, of the same parity, for that.
    p.stages = (LS_BYTES - rest) / LS_STAGE / 2 * 2;
    if (p.stages < 4) p.stages = (LS_BYTES_ALONE - rest) / LS_STAGE / 2 * 2;
    if (p.stages > LS_STAGES) p.stages = LS_STAGES;
    p.part_at = p.stages * LS_STAGE;
    p.sum_at = p.part_at + part;
    p.x_at = p.sum_at + sum;
    p.h_at = p.x_at + 8 * px * p.x_line;
    p.base_at = p.h_at + 8 * ph * p.h_line;
    p.bytes = p.base_at + LS_BASE;
    p.fits = p.stages >= 4;
    return p;
}

// D[16 x 8] += A[16 x 16] B[16 x 8].
template <int TW>
__device__ __forceinline__ void ls_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (TW == KV_BF16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 32 inputs: a lane has eight of two rows of weights, and of a column's parts, `step` bytes apart.
template <int TW, int PARTS>
__device__ __forceinline__ void ls_unit(float (&acc)[4], const uint4 &p, const uint4 &q, const char *column, int step) {
    float d[4] = {};
#pragma unroll
    for (int i = PARTS - 1; i >= 0; --i) {                             // the largest last, as each step cuts the whole sum off
        const uint4 x = *(const uint4 *)(column + i * step);
        ls_mma<TW>(d, p.x, q.x, p.y, q.y, x.x, x.y);
        ls_mma<TW>(d, p.z, q.z, p.w, q.w, x.z, x.w);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = fadd(acc[i], d[i]);
}
// The power of two that brings `most` to [2^14, 2^15), and its inverse; 1 for what is nought, tiny or no number.
__device__ __forceinline__ float ls_scale(float most, float *back) {
    const uint32_t exponent = __float_as_uint(most) >> 23;
    *back = 1.0f;
    if (exponent <= 20 || exponent >= 255) return 1.0f;
    *back = __uint_as_float((exponent - 14) << 23);
    return __uint_as_float((268 - exponent) << 23);
}

template <int TX, int TW>
__global__ void __launch_bounds__(LS_THREADS, 2) lora_stream_kernel(const __grid_constant__ LoraArgs a, const __grid_constant__ LoraStreamPlan plan) {
    using S = LoraStream<TX, TW>;
    extern __shared__ __align__(128) char ls_raw[];
    __shared__ float x_back[8], h_back[8];
    __shared__ uint64_t full[LS_STAGES], empty[LS_STAGES];
    __shared__ int failed;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
    const int ctas = (int)lora_cluster_size(), cta = (int)lora_rank_of_cluster();
    release_dependents();
    wait_for_producer();
    const int4 item = lora_item(a, blockIdx.x / ctas);
    const int32_t *const order = (const int32_t *)(lora_items(a.plan) + a.items);
    const int slot = item.x, first = item.y, count = min(8, item.z);
    if (count <= 0) return;
    const int t0 = (int)blockIdx.y * a.pass_targets, t1 = min(a.targets, t0 + a.pass_targets);
    int n_first = 0, n_pass = 0, n_tiles = 0;                          // outputs before the pass, of it, tiles of 16 of them
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
    const char *const wa = (const char *)a.a + ((int64_t)slot * a.targets + t0) * a.rank * a.inputs * 2;
    const char *const wb = (const char *)a.b + (int64_t)slot * a.outputs * a.rank * 2;
    const int units = (a.inputs + 31) / 32, k_low = 32 * (int)((int64_t)units * cta / ctas), k_high = min(a.inputs, 32 * (int)((int64_t)units * (cta + 1) / ctas));
    const int chunks = (k_high - k_low + LS_WIDTH - 1) / LS_WIDTH, per = (r + 15) / 16, tiles = per * (t1 - t0), rp = (r + 31) / 32 * 32;
    const int tile_low = (int)((int64_t)n_tiles * cta / ctas), tile_high = (int)((int64_t)n_tiles * (cta + 1) / ctas);
    const int at_once = max(1, LS_B / (32 * a.rank));                  // tiles of B in a stage
    if (tid == 0) {
        for (int i = 0; i < plan.stages; ++i) lt_init(&full[i], 1), lt_init(&empty[i], LS_TEAM);
        failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    const long long limit = g_wait_cycles;
    auto wait = [&](uint64_t *bar, unsigned parity) {                  // one that runs out is the last one
        if (kvt_mbar_wait(bar, parity, *(volatile int *)&failed ? 0 : limit)) return true;
        *(volatile int *)&failed = 1;
        atomicOr(&g_lora_fault, LORA_LATE);
        return false;
    };
    // B's stages: tiles [tile, tile + n) of one target, from output n0 on.
    struct Piece {
        int target, tile, n, n0;
    };
    int target = t0, tile0 = 0, n_target = n_first;                    // the target that is being gone through, its first tile and output
    auto piece = [&](int tile) {
        while (tile - tile0 >= (a.width[target] + 15) / 16) {
            tile0 += (a.width[target] + 15) / 16;
            n_target += a.width[target];
            ++target;
        }
        return Piece{target, tile, min(min(at_once, tile_high - tile), tile0 + (a.width[target] + 15) / 16 - tile), n_target + 16 * (tile - tile0)};
    };
    const uint32_t ring = kvt_smem(ls_raw);
    if (warp >= LORA_WARPS) {
        lora_cluster_arrive();                                         // for the CTAs' sums, which this warp has no part in
        asm volatile("bar.sync 2, %0;" ::"n"(LS_THREADS) : "memory");  // the rows' inputs are asked for: they would come after all of the ring
        int stage = 0, round = 0, asked = 0;
        bool good = true;
        auto mine = [&]() { return asked % LS_ASKERS == warp - LORA_WARPS; };
        auto begin = [&](int bytes) {                                  // once the stage is free
            if (round > 0) good = wait(&empty[stage], (round - 1) & 1);
            good = __all_sync(0xffffffffu, good);
            if (good && lane == 0)
                asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(kvt_smem(&full[stage])), "r"(bytes) : "memory");
            __syncwarp();
        };
        auto copy = [&](uint32_t to, const char *from, int bytes) {
            asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(ring + stage * LS_STAGE + to), "l"(from), "r"(bytes),
                         "r"(kvt_smem(&full[stage]))
                         : "memory");
        };
        int last = -1;                                                 // the last stage's number that this warp asked for
        auto go_on = [&]() {
            ++asked;
            if (++stage == plan.stages) stage = 0, ++round;
        };
        for (int tile = 0; tile < tiles && good; ++tile)
            for (int chunk = 0; chunk < chunks && good; ++chunk, go_on()) {
                if (!mine()) continue;
                const int t = tile / per, j = (tile - t * per) * 16, rows = min(16, r - j), k = k_low + chunk * LS_WIDTH, bytes = min(LS_WIDTH, k_high - k) * 2;
                begin(rows * bytes);
                if (!good) break;
                if (lane < rows) copy(lane * LS_LINE, wa + (((int64_t)t * a.rank + j + lane) * a.inputs + k) * 2, bytes);
                last = asked;
            }
        for (int tile = tile_low; tile < tile_high && good; go_on()) {
            const Piece p = piece(tile);
            tile += p.n;
            if (!mine()) continue;
            const int bytes = min(16 * p.n, a.width[p.target] - 16 * (p.tile - tile0)) * a.rank * 2;
            begin(bytes);
            if (!good) break;
            if (lane == 0) copy(0, wb + (int64_t)p.n0 * a.rank * 2, bytes);
            last = asked;
        }
        // What is in flight comes to its end before the CTA does, also where nobody waited for it: the last copies to each stage (of
        // earlier ones the barrier does not know any more).
        for (int i = max(0, asked - plan.stages); i <= last; ++i)
            if (i % LS_ASKERS == warp - LORA_WARPS) kvt_mbar_wait(&full[i % plan.stages], (i / plan.stages) & 1, NC_DRAIN_CYCLES);
        __syncwarp();
        lora_cluster_wait();
        lora_cluster_arrive();
        lora_cluster_wait();
        return;
    }

    const int team = warp / LS_TEAM, member = warp % LS_TEAM;
    int stage = 0, round = 0, number = 0;                              // of the stage that comes next
    auto ours = [&]() { return number % 2 == team; };
    auto take = [&]() { wait(&full[stage], round & 1); __syncwarp(); };
    auto leave = [&]() {
        __syncwarp();
        if (lane == 0) lt_arrive(&empty[stage]);
    };
    auto go_on = [&]() {
        ++number;
        if (++stage == plan.stages) stage = 0, ++round;
    };
    // The rows' shares of x, a row to a warp: eight inputs of every 256 to a lane, in parts.
    const int slice = k_high - k_low;
    char *const x_room = ls_raw + plan.x_at, *const h_room = ls_raw + plan.h_at, *const base_room = ls_raw + plan.base_at;
    // Those of base, where they fit: of whole tiles of the targets, but for their ends.
    int b_first = 0, b_last = 0;
    {
        int tile = 0, n = n_first;
        for (int t = t0; t < t1; ++t) {
            const int all = (a.width[t] + 15) / 16;
            if (tile <= tile_low && tile_low < tile + all) b_first = n + 16 * (tile_low - tile);
            if (tile < tile_high && tile_high <= tile + all) b_last = min(n + 16 * (tile_high - tile), n + a.width[t]);
            tile += all;
            n += a.width[t];
        }
    }
    const int b_width = b_last - b_first, b_line = (b_width * S::SIZE + 15) / 16 * 16;
    const bool b_pairs = a.pairs && b_first % 2 == 0, b_here = a.base && b_pairs && count * b_line <= LS_BASE;
    {
        const int64_t row = warp < count ? lora_row(a, order, first + warp) : -1;
        // 1024 inputs at a time; where they are scaled, a first time for the largest.
        constexpr int M = 4;
        float v[M][8], by = 1.0f, largest = 0.0f;                  // largest: of the row, once scaled, where that is a number
        auto load = [&](int from) {
#pragma unroll
            for (int m = 0; m < M; ++m) {
                const int e = from + 256 * m + 8 * lane;
#pragma unroll
                for (int i = 0; i < 8; ++i) v[m][i] = 0.0f;
                if (e < slice && row >= 0) kv_load8(a.x, row * a.x_stride + k_low + e, TX, a.x_vectors, v[m]);
            }
        };
        load(0);
        __syncwarp();
        asm volatile("bar.arrive 2, %0;" ::"n"(LS_THREADS) : "memory");
        if (b_here && row >= 0) {
            const char *const from = (const char *)a.base + (row * a.base_stride + b_first) * S::SIZE;
            const uint32_t to = kvt_smem(base_room + warp * b_line);
            for (int n = 2 * lane; n + 1 < b_width; n += 64)
                asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to + n * S::SIZE), "l"(from + n * S::SIZE), "n"(2 * S::SIZE) : "memory");
            if (lane == 0 && b_width % 2) kv_store(base_room + warp * b_line, b_width - 1, TX, kv_load(from, b_width - 1, TX));
        }
        if constexpr (S::SCALED_X) {
            float most = 0.0f;
            for (int from = 0; from < slice; from += 256 * M) {
                if (from > 0) load(from);
#pragma unroll
                for (int m = 0; m < M; ++m)
#pragma unroll
                    for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(v[m][i]));
            }
            float back;
            by = ls_scale(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most))), &back);
            if (lane == 0) x_back[warp] = back;
            if (slice > 256 * M) load(0);
            if (__any_sync(0xffffffffu, !(most < INFINITY))) largest = INFINITY;
        }
        for (int from = 0; from * 2 < plan.x_line - 16; from += 256 * M) {
            if (from > 0) load(from);
            if constexpr (S::PX > 1 && !S::SCALED_X) {
                largest = 0.0f;
#pragma unroll
                for (int m = 0; m < M; ++m)
#pragma unroll
                    for (int i = 0; i < 8; ++i) largest = fmaxf(largest, fabsf(v[m][i]));
            }
            lt_sure<TW>(largest, [&](auto sure) {                      // rows of the weights' type are their only part, whatever they are
#pragma unroll
                for (int m = 0; m < M; ++m) {
                    const int e = from + 256 * m + 8 * lane;
                    if (e * 2 >= plan.x_line - 16) continue;
                    float2 pair[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        pair[i] = S::SCALED_X ? make_float2(fmul(v[m][2 * i], by), fmul(v[m][2 * i + 1], by)) : make_float2(v[m][2 * i], v[m][2 * i + 1]);
#pragma unroll
                    for (int p = 0; p < S::PX; ++p) {
                        uint32_t w[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) w[i] = lt_part<TW, decltype(sure)::value>(pair[i]);
                        *(uint4 *)(x_room + (p * 8 + warp) * plan.x_line + e * 2) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
            });
        }
    }
    asm volatile("bar.sync 1, %0;" ::"n"(LORA_THREADS) : "memory");
    float *const part = (float *)(ls_raw + plan.part_at), *const sum = (float *)(ls_raw + plan.sum_at);
    // Rows past the rank hold what was there before: theirs are rows of h that are not looked at.
    for (int tile = 0; tile < tiles; ++tile) {
        float acc[4] = {};
        for (int chunk = 0; chunk < chunks; ++chunk, go_on()) {
            if (!ours()) continue;
            constexpr int U = LS_WIDTH / (32 * LS_TEAM);
            const int width = min(LS_WIDTH, slice - chunk * LS_WIDTH);
            take();
            const char *const from = ls_raw + stage * LS_STAGE + g * LS_LINE + 16 * c, *const column = x_room + g * plan.x_line + chunk * LS_WIDTH * 2 + 16 * c;
            uint4 p[U], q[U];
#pragma unroll
            for (int m = 0; m < U; ++m) {
                const int e = 32 * (member + LS_TEAM * m);
                p[m] = *(const uint4 *)(from + e * 2);
                q[m] = *(const uint4 *)(from + 8 * LS_LINE + e * 2);
                if (e + 32 > width && e + 8 * c >= width) p[m] = q[m] = make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int m = 0; m < U; ++m) {
                const int e = 32 * (member + LS_TEAM * m);
                if (e < width) ls_unit<TW, S::PX>(acc, p[m], q[m], column + e * 2, 8 * plan.x_line);
            }
            leave();
        }
        if constexpr (S::SCALED_X) {
            const float b0 = x_back[2 * c], b1 = x_back[2 * c + 1];
            acc[0] = fmul(acc[0], b0), acc[1] = fmul(acc[1], b1), acc[2] = fmul(acc[2], b0), acc[3] = fmul(acc[3], b1);
        }
        float *const to = part + (warp * plan.tiles + tile) * 128 + g * 8 + 2 * c;
        *(float2 *)to = make_float2(acc[0], acc[1]);
        *(float2 *)(to + 64) = make_float2(acc[2], acc[3]);
    }
    asm volatile("bar.sync 1, %0;" ::"n"(LORA_THREADS) : "memory");
    // A column after another, as the peers read it: with the columns side by side their lanes met two banks alone, and 64 rows of eight adapters
    // (896 -> 896 at rank 64) took 23.7 us, 13.0 now, 64 rows of 16 of 1 MB 24.5, now 15.8.
    const int pitch = 16 * plan.tiles + 4;
    for (int i = tid; i < tiles * 128; i += LORA_THREADS) {
        float v = part[i];
#pragma unroll
        for (int k = 1; k < LORA_WARPS; ++k) v = fadd(v, part[k * plan.tiles * 128 + i]);
        sum[(i & 7) * pitch + (i >> 3)] = v;
    }
    lora_cluster_arrive();
    lora_cluster_wait();
    // h, a column to a warp: two rows of every 64 to a lane, in parts.
    {
        constexpr int M = LORA_PASS / 64;
        float2 v[M];
        float most = 0.0f;
#pragma unroll
        for (int m = 0; m < M; ++m) {
            v[m] = make_float2(0.0f, 0.0f);
            const int at = 64 * m + 2 * lane, t = at / rp, j = at - t * rp;
            if (warp >= count || t >= t1 - t0 || j >= r) continue;
            const float *const from = sum + warp * pitch + t * per * 16 + j;
            float p[8], q[8];                                          // asked for all at once
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                p[k] = k < ctas ? lora_peer(from, k) : 0.0f;
                q[k] = k < ctas && j + 1 < r ? lora_peer(from + 1, k) : 0.0f;
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) v[m].x = fadd(v[m].x, p[k]), v[m].y = fadd(v[m].y, q[k]);
            most = fmaxf(most, fmaxf(fabsf(v[m].x), fabsf(v[m].y)));
        }
        if constexpr (S::SCALED_H) {
            float back;
            const float by = ls_scale(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most))), &back);
            if (lane == 0) h_back[warp] = back;
#pragma unroll
            for (int m = 0; m < M; ++m) v[m].x = fmul(v[m].x, by), v[m].y = fmul(v[m].y, by);
            if (most < INFINITY) most = fmul(most, by);                // where the row has an infinity it is as it was, and may be too large
        }
        lt_sure<TW>(most, [&](auto sure) {
#pragma unroll
            for (int m = 0; m < M; ++m) {
                const int at = 64 * m + 2 * lane;
                if (at >= rp * (t1 - t0)) continue;
#pragma unroll
                for (int p = 0; p < S::PH; ++p) *(uint32_t *)(h_room + (p * 8 + warp) * plan.h_line + at * 2) = lt_part<TW, decltype(sure)::value>(v[m]);
            }
        });
    }
    lora_cluster_arrive();                                             // the peers' sums are read; they may go once all CTAs are here
    asm volatile("cp.async.wait_all;" ::: "memory");
    asm volatile("bar.sync 1, %0;" ::"n"(LORA_THREADS) : "memory");

    float out_scale[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) out_scale[k] = S::SCALED_H ? scale * h_back[2 * c + k] : scale;
    int64_t out_row[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) out_row[k] = 2 * c + k < count ? lora_row(a, order, first + 2 * c + k) : -1;
    for (int tile = tile_low; tile < tile_high; go_on()) {
        const Piece p = piece(tile);
        tile += p.n;
        if (!ours()) continue;
        const int ends = a.width[p.target] - 16 * (p.tile - tile0);    // the target's outputs from the piece on
        take();
        const char *const stage_at = ls_raw + stage * LS_STAGE, *const column = h_room + g * plan.h_line + ((p.target - t0) * rp + 8 * c) * 2;
        // Two tiles at once.  Outputs past the target's are products with what was there before, and not stored.
        for (int u = member; u < p.n; u += 2 * LS_TEAM) {
            float2 was[2][2];
            float acc[2][4] = {};
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int n = 16 * (u + LS_TEAM * i) + 2 * g;
                    was[i][k] = make_float2(0.0f, 0.0f);
                    if (!a.base || out_row[k] < 0 || u + LS_TEAM * i >= p.n || n >= ends) continue;
                    if (b_here) was[i][k] = lora_load2<TX>(base_room + (2 * c + k) * b_line, p.n0 + n - b_first, ends - n > 1, true);
                    else was[i][k] = lora_load2<TX>(a.base, out_row[k] * a.base_stride + p.n0 + n, ends - n > 1, a.pairs);
                }
            const int second = u + LS_TEAM < p.n ? LS_TEAM : 0;
            const char *const from = stage_at + ((16 * u + 2 * g) * a.rank + 8 * c) * 2;
            for (int j = 0; j < rp; j += 32) {
                uint4 w[2][2];
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int k = 0; k < 2; ++k) w[i][k] = *(const uint4 *)(from + ((16 * second * i + k) * a.rank + min(j, a.rank - 8 * c - 8)) * 2);
                if (j + 32 > r) {                                      // what lies past the adapter's own rank may be anything
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            uint32_t v[4] = {w[i][k].x, w[i][k].y, w[i][k].z, w[i][k].w};
#pragma unroll
                            for (int e = 0; e < 4; ++e) v[e] = j + 8 * c + 2 * e >= r ? 0u : j + 8 * c + 2 * e + 1 >= r ? v[e] & 0xffffu : v[e];
                            w[i][k] = make_uint4(v[0], v[1], v[2], v[3]);
                        }
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) ls_unit<TW, S::PH>(acc[i], w[i][0], w[i][1], column + j * 2, 8 * plan.h_line);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int n = 16 * (u + LS_TEAM * i) + 2 * g;
                    if (out_row[k] < 0 || u + LS_TEAM * i >= p.n || n >= ends) continue;
                    lora_store2<TX>(a.out, out_row[k] * a.out_stride + p.n0 + n,
                                    make_float2(__fmaf_rn(out_scale[k], acc[i][k], was[i][k].x), __fmaf_rn(out_scale[k], acc[i][2 + k], was[i][k].y)), ends - n > 1, a.pairs);
                }
        }
        leave();
    }
    lora_cluster_wait();
}

}  // namespace nc
