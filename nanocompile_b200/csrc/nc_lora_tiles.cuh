// nc_lora_tiles.cuh -- low-rank adapters for prompts: what nc_lora.cuh computes, for items of up to 128 rows, on the tensor cores.
//
// An item to a cluster.  First each CTA multiplies its share of the inputs, 64 at a time: D1 [128 rows][h] += x A^T, tcgen05.mma with the
// rows and the adapter's A copied asynchronously into 128-byte swizzled tiles, D1 in tensor memory.  The CTAs' sums of h are added
// through distributed shared memory, each CTA taking 128 / CTAs rows and giving them to all, already split into the operand's
// parts.  Then each CTA expands its share of the outputs, 256 bytes of a row at a time: D2 [128][outputs] = h B^T in two halves of
// tensor memory, while the warps add the last tile to base: base is asked for a tile ahead, and goes by way of a warp's own
// shared memory from a row to a thread to whole lines of rows.  The targets' h lie side by side, whole 16s to each.
//
// Accuracy.  16-bit rows and weights are multiplied as they are, h goes in two parts (16 bits and the next 16: bfloat16 2^-17 of it is
// lost, float16 2^-22; float16's h is first brought to [2^14, 2^15) by a power of two for each row, so that no size leaves its
// range).  Sums are float32 in tensor memory.
#pragma once

#include "nc_kv4_prompt.cuh"
#include "nc_lora.cuh"

namespace nc {

constexpr int LT_ROWS = 128, LT_WARPS = 8, LT_WORKERS = 32 * LT_WARPS, LT_THREADS = LT_WORKERS + 32, LT_TMEM = 256;
constexpr int LT_BLOCK = LT_ROWS * 128;        // 128 rows of 128 bytes
constexpr int LT_HALF = LT_ROWS * 64;          // 128 rows of 64 bytes
constexpr int LT_STAGES = 6;                   // of the first products at most
constexpr int LT_TWICE = 110 * 1024, LT_ONCE = 200 * 1024;             // bytes of tiles with two CTAs on an SM, with one
constexpr int LT_LINE = 36;                    // floats from a row to the next of a warp's 32 x 32: no bank twice in a quarter

__device__ unsigned int g_lora_fault;          // set when a matrix instruction did not come to its end within the wait limit

template <int TX>
struct LoraTiles {
    static constexpr int PH = 2;                                       // parts of h
    static constexpr int COLS = TX == KV_F32 ? 64 : 128;               // outputs of a tile
    static constexpr int CHUNKS = COLS / 64;                           // of 32 outputs, for each warp
    static constexpr int SIZE = TX == KV_F32 ? 4 : 2;
};

// How shared memory is laid out, by the most rows of h in a pass: h's operand, then the sums of h; over these B and the warps'
// lines; over all of it the stages of the first products.
struct LoraTilesPlan {
    int wide;                                  // rows of h in whole 16s
    int stages, a_bytes;                       // of a stage: LT_BLOCK for rows, a_bytes for A
    int h_blocks, b_blocks;                    // blocks of 32 for a part of h, for B
    int sum_at, line_at, bytes;
};
inline LoraTilesPlan lora_tiles_plan(int targets, int rank, int parts, int cols) {
    LoraTilesPlan p{};
    p.wide = targets * ((rank + 15) / 16 * 16);
    p.a_bytes = p.wide * 128;
    p.h_blocks = (p.wide + 31) / 32;
    p.b_blocks = (rank + 31) / 32;
    p.sum_at = parts * p.h_blocks * LT_HALF;
    p.line_at = p.sum_at + 2 * p.b_blocks * cols * 64;
    const int sums = LT_ROWS * (p.wide + 4) * 4, lines = LT_WARPS * 32 * LT_LINE * 4;
    p.bytes = p.line_at + lines > p.sum_at + sums ? p.line_at + lines : p.sum_at + sums;
    const int stage = LT_BLOCK + p.a_bytes, most = p.bytes > LT_TWICE ? LT_ONCE : LT_TWICE;       // room for two CTAs on an SM, or one
    p.stages = most / stage < LT_STAGES ? most / stage : LT_STAGES;
    if (p.stages * stage > p.bytes) p.bytes = p.stages * stage;
    return p;
}

struct LoraTilesShared {                       // before the tiles
    uint64_t full[LT_STAGES], empty[LT_STAGES], d1_done, b_full[2], d2_done[2], d2_free[2], drained;
    float row_scale[LT_ROWS];
    int row[LT_ROWS];
    uint32_t tmem;
    int failed;
};

__device__ __forceinline__ void lt_init(uint64_t *bar, int count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(kvt_smem(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void lt_arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(kvt_smem(bar)) : "memory");
}
// D[128 x n] (+)= A[128 x 16] B[16 x n], both K-major in shared memory; 16-bit with float32 sums.
template <int TW>
__device__ __forceinline__ void lt_mma(uint32_t d, uint64_t a, uint64_t b, int n, bool add) {
    constexpr uint32_t format = TW == KV_BF16 ? 1u << 7 | 1u << 10 : 0u;
    const uint32_t kind = 1u << 4 | format | (uint32_t)(n >> 3) << 17 | (uint32_t)(128 >> 4) << 24;
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(kind), "r"((uint32_t)add)
        : "memory");
}
// A K-major operand of 64-byte swizzled rows: eight rows are 512 bytes, and bits 4 and 5 of an address are flipped by its bits 7 and 8.
__device__ __forceinline__ uint64_t lt_desc64(uint32_t address) {
    return (uint64_t)((address & 0x3ffff) >> 4) | (uint64_t)1 << 16 | (uint64_t)(512 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)4 << 61;
}
__device__ __forceinline__ void lt_async_fence() { asm volatile("fence.proxy.async;" ::: "memory"); }
// 16 bytes from `from`, of which `bytes` are there: the others become nought.
__device__ __forceinline__ void lt_copy16(uint32_t to, const void *from, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void lt_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void lt_wait_copies() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint32_t lt_peer(uint32_t at, uint32_t rank) {                        // of another CTA's shared memory
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(at), "r"(rank));
    return r;
}
__device__ __forceinline__ void lt_store_peer(uint32_t at, uint32_t v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory"); }
__device__ __forceinline__ void lt_store_peer(uint32_t at, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
// Two values rounded to 16 bits, and what that leaves.
template <int TW>
__device__ __forceinline__ uint32_t lt_part(float2 &v) {
    uint32_t w;
    float2 r;
    if constexpr (TW == KV_BF16) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(v.x, v.y);
        w = *reinterpret_cast<const uint32_t *>(&b);
        r = __bfloat1622float2(b);
    } else {
        const __half2 b = __floats2half2_rn(v.x, v.y);
        w = *reinterpret_cast<const uint32_t *>(&b);
        r = __half22float2(b);
    }
    // Nothing is left of what is no number, or rounds to none.
    v.x = fabsf(r.x) < INFINITY ? fsub(v.x, r.x) : 0.0f;
    v.y = fabsf(r.y) < INFINITY ? fsub(v.y, r.y) : 0.0f;
    return w;
}
// Eight outputs from 16 bytes of base and float32 sums.
template <int TX>
__device__ __forceinline__ uint4 lt_add(const uint4 &was, const float (&v)[8], float scale) {
    const uint32_t u[4] = {was.x, was.y, was.z, was.w};
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (TX == KV_F16) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u[i]));
            const __half2 r = __floats2half2_rn(__fmaf_rn(scale, v[2 * i], f.x), __fmaf_rn(scale, v[2 * i + 1], f.y));
            w[i] = *reinterpret_cast<const uint32_t *>(&r);
        } else {
            const __nv_bfloat162 r = __floats2bfloat162_rn(__fmaf_rn(scale, v[2 * i], __uint_as_float(u[i] << 16)),
                                                           __fmaf_rn(scale, v[2 * i + 1], __uint_as_float(u[i] & 0xffff0000u)));
            w[i] = *reinterpret_cast<const uint32_t *>(&r);
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int TX>
__global__ void __launch_bounds__(LT_THREADS, 2) lora_tiles_kernel(const __grid_constant__ LoraArgs a, const __grid_constant__ LoraTilesPlan plan) {
    using S = LoraTiles<TX>;
    extern __shared__ __align__(1024) char lt_raw[];
    char *const tiles = lt_raw + ((1024 - (kvt_smem(lt_raw) & 1023)) & 1023);
    __shared__ LoraTilesShared sh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const bool worker = warp < LT_WARPS;
    const int ctas = (int)lora_cluster_size(), cta = (int)lora_rank_of_cluster();
    wait_for_producer();
    const int4 item = lora_items(a.plan)[blockIdx.x / ctas];
    const int32_t *const order = (const int32_t *)(lora_items(a.plan) + a.items);
    const int slot = item.x, first = item.y, count = min(LT_ROWS, item.z);
    if (count <= 0 || first < 0 || first > a.rows - count || slot >= a.slots) return;        // nothing there, or no plan of this call's sizes
    const int t0 = (int)blockIdx.y * a.pass_targets, t1 = min(a.targets, t0 + a.pass_targets);
    int n_first = 0, n_pass = 0, n_tiles = 0;                          // outputs before the pass, of it, tiles of them
    for (int t = 0; t < t1; ++t) {
        if (t < t0) n_first += a.width[t];
        else n_pass += a.width[t], n_tiles += (a.width[t] + S::COLS - 1) / S::COLS;
    }
    const int r = slot < 0 ? 0 : a.ranks ? min(max(a.ranks[slot], 0), a.rank) : a.rank;
    if (r == 0) {
        const int64_t n = n_pass;
        lora_copy<TX>(a, order, first, count, n_first + (int)(n * cta / ctas), n_first + (int)(n * (cta + 1) / ctas));
        return;
    }
    const int rp = (r + 15) / 16 * 16, wide = (t1 - t0) * rp;
    const float scale = a.scales ? a.scales[slot] : 1.0f;
    const char *const wa = (const char *)a.a + ((int64_t)slot * a.targets + t0) * a.rank * a.inputs * 2;
    const char *const wb = (const char *)a.b + (int64_t)slot * a.outputs * a.rank * 2;
    const int tile_low = (int)((int64_t)n_tiles * cta / ctas), tile_high = (int)((int64_t)n_tiles * (cta + 1) / ctas), my_tiles = tile_high - tile_low;
    const int blocks = (a.inputs + 63) / 64, k_low = (int)((int64_t)blocks * cta / ctas), k_blocks = (int)((int64_t)blocks * (cta + 1) / ctas) - k_low;
    {
        const int64_t low = ((int64_t)n_first + S::COLS * tile_low) * a.rank * 2, high = min((int64_t)n_first + n_pass, (int64_t)n_first + S::COLS * tile_high) * a.rank * 2;
        for (int64_t at = low + tid * 4096; at < high; at += LT_THREADS * 4096)
            asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(wb + at), "r"((uint32_t)min((int64_t)4096, high - at)) : "memory");
    }
    if (warp == LT_WARPS) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(kvt_smem(&sh.tmem)), "n"(LT_TMEM) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid == 0) {
        for (int i = 0; i < plan.stages; ++i) lt_init(&sh.full[i], LT_WORKERS), lt_init(&sh.empty[i], 1);
        lt_init(&sh.d1_done, 1);
        lt_init(&sh.drained, 1);
        for (int i = 0; i < 2; ++i) lt_init(&sh.b_full[i], LT_WORKERS), lt_init(&sh.d2_done[i], 1), lt_init(&sh.d2_free[i], LT_WORKERS);
        sh.failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (tid < LT_ROWS) sh.row[tid] = tid < count ? (int)lora_row(a, order, first + tid) : -1;
    kvt_before();
    __syncthreads();
    kvt_after();
    release_dependents();                      // not before this CTA has its tensor memory: a dependent may hold all the rest
    const uint32_t tmem = sh.tmem, base_at = kvt_smem(tiles);
    const long long limit = g_wait_cycles;
    // A wait that runs out is the last one: the CTA goes on without waiting and its outputs are not to be used.
    auto wait = [&](uint64_t *bar, unsigned parity) {
        if (kvt_mbar_wait(bar, parity, *(volatile int *)&sh.failed ? 0 : limit)) return true;
        *(volatile int *)&sh.failed = 1;
        g_lora_fault = 1;
        return false;
    };
    const int stage_bytes = LT_BLOCK + plan.a_bytes, c = tid & 7, line = tid >> 3;               // a worker's 16 bytes of every 32nd row

    // h, in parts: D1 = x A^T over this CTA's inputs.
    if (worker) {
        const char *x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = sh.row[line + 32 * i];
            x[i] = row < 0 ? nullptr : (const char *)a.x + (int64_t)row * a.x_stride * 2;
        }
        int from[LORA_PASS / 32];                                      // of A's rows; -1: none there
#pragma unroll
        for (int i = 0; i < LORA_PASS / 32; ++i) {
            const int j = line + 32 * i, t = j / rp;
            from[i] = j < wide && j - t * rp < r ? (t * a.rank + j - t * rp) * a.inputs : -1;
        }
        const uint32_t swizzled = (uint32_t)line * 128 + (uint32_t)((c ^ (line & 7)) << 4);
        auto issue = [&](int k) {
            const uint32_t to = base_at + (uint32_t)(k % plan.stages) * stage_bytes + swizzled;
            const int e = (k_low + k) * 64 + 8 * c;
            const bool in = e < a.inputs;
#pragma unroll
            for (int i = 0; i < 4; ++i) lt_copy16(to + i * 4096, in && x[i] ? x[i] + e * 2 : a.x, in && x[i] ? 16 : 0);
#pragma unroll
            for (int i = 0; i < LORA_PASS / 32; ++i)
                if (line + 32 * i < wide) lt_copy16(to + LT_BLOCK + i * 4096, in && from[i] >= 0 ? wa + (int64_t)(from[i] + e) * 2 : wa, in && from[i] >= 0 ? 16 : 0);
        };
        // A stage is asked for again when the products two blocks back are done with it, not those just begun.
        const int ahead = max(1, plan.stages - 2);
        for (int k = 0; k < ahead; ++k) {
            if (k < k_blocks) issue(k);
            lt_commit();
        }
        for (int k = 0; k < k_blocks; ++k) {
            const int next = k + ahead;
            if (next < k_blocks) {
                if (next >= plan.stages) wait(&sh.empty[next % plan.stages], (next / plan.stages - 1) & 1);
                issue(next);
            }
            lt_commit();
            switch (ahead) {                                           // the oldest of `ahead` + 1 groups is there
                case 1: lt_wait_copies<1>(); break;
                case 2: lt_wait_copies<2>(); break;
                case 3: lt_wait_copies<3>(); break;
                default: lt_wait_copies<4>(); break;
            }
            lt_async_fence();
            lt_arrive(&sh.full[k % plan.stages]);
        }
        lt_wait_copies<0>();
    } else if (lane == 0) {
        for (int k = 0; k < k_blocks; ++k) {
            const int stage = k % plan.stages;
            if (!wait(&sh.full[stage], (k / plan.stages) & 1)) break;
            kvt_after();
            const uint32_t at = base_at + (uint32_t)stage * stage_bytes;
            const int steps = min(4, (a.inputs - (k_low + k) * 64 + 15) / 16);
            for (int s = 0; s < steps; ++s) lt_mma<TX>(tmem, kvt_desc(at + 32 * s), kvt_desc(at + LT_BLOCK + 32 * s), wide, k > 0 || s > 0);
            kvt_commit(&sh.empty[stage]);
        }
        kvt_commit(&sh.d1_done);
    }
    __syncwarp();
    wait(&sh.d1_done, 0);
    kvt_after();
    // B's tiles: outputs' rows in blocks of 32, 64 bytes each; a worker has 16 bytes of every 64th row.
    const int b_bytes = plan.b_blocks * S::COLS * 64, bc = tid & 3, bl = tid >> 2;
    int target = t0, tile0 = 0, n_target = n_first;                    // of the tile that is asked for next
    auto issue_b = [&](int i) {
        const int tile = tile_low + i;
        while (tile - tile0 >= (a.width[target] + S::COLS - 1) / S::COLS) {
            tile0 += (a.width[target] + S::COLS - 1) / S::COLS;
            n_target += a.width[target];
            ++target;
        }
        const int n0 = (tile - tile0) * S::COLS;
        const uint32_t to = base_at + plan.sum_at + (uint32_t)(i & 1) * b_bytes;
#pragma unroll
        for (int n = bl; n < S::COLS; n += 64)
            for (int j = 8 * bc; j < rp; j += 32) {
                const uint32_t at = to + (uint32_t)(j >> 5) * (S::COLS * 64) + (uint32_t)n * 64 + (uint32_t)((bc ^ ((n >> 1) & 3)) << 4);
                const char *const from = wb + (((int64_t)n_target + n0 + n) * a.rank + j) * 2;
                const bool there = n0 + n < a.width[target];
                if (j + 8 <= r || j >= r || !there) {
                    lt_copy16(at, there && j < r ? from : wb, there && j < r ? 16 : 0);
                } else {                                               // what lies past the adapter's own rank may be anything
                    const uint4 w = __ldg((const uint4 *)from);
                    uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) u[e] = j + 2 * e >= r ? 0u : j + 2 * e + 1 >= r ? u[e] & 0xffffu : u[e];
                    store16_shared(at, u[0], u[1], u[2], u[3]);
                }
            }
    };
    lora_cluster_arrive();                     // every CTA is done with its stages: sums may lie over them
    lora_cluster_wait();
    const int mine = LT_ROWS / ctas, pitch = plan.wide + 4;            // rows that a CTA adds up
    if (worker) {
        // The CTA's sums go to the CTAs that add them up: a row to a thread, 16 columns at a time, a half of them to a warp.
        const int row = 32 * (warp & 3) + lane;
        const uint32_t to = lt_peer(base_at + plan.sum_at + (uint32_t)((cta * mine + row % mine) * pitch) * 4, row / mine);
        for (int j = 16 * (warp >> 2); j < wide; j += 32) {
            uint32_t v[16];
            kvt_load16(tmem + ((uint32_t)(32 * (warp & 3)) << 16) + j, v);
            kvt_wait_ld();
            if (k_blocks == 0)                                         // more CTAs than blocks of inputs
#pragma unroll
                for (int e = 0; e < 16; ++e) v[e] = 0;
#pragma unroll
            for (int e = 0; e < 16; e += 4) lt_store_peer(to + (j + e) * 4, v[e], v[e + 1], v[e + 2], v[e + 3]);
        }
    }
    kvt_before();
    lora_cluster_arrive();
    lora_cluster_wait();
    kvt_after();
    if (worker) {
        // A row to a warp, two columns of every 64 to a lane.
        const float *const sums = (const float *)(tiles + plan.sum_at) + 2 * lane;
        uint32_t keep = 0;                                             // columns that are h's
#pragma unroll
        for (int m = 0; m < LORA_PASS / 64; ++m) {
            const int col = 64 * m + 2 * lane, j = col % rp;
            if (col < wide) keep |= (uint32_t)((j < r) | (j + 1 < r) << 1 | 4) << (4 * m);
        }
        for (int i = warp; i < mine; i += LT_WARPS) {
            const int row = cta * mine + i;
            float2 v[LORA_PASS / 64];
            float most = 0.0f;
#pragma unroll
            for (int m = 0; m < LORA_PASS / 64; ++m) {
                v[m] = make_float2(0.0f, 0.0f);
                if (!(keep >> (4 * m) & 4)) continue;
                for (int k = 0; k < ctas; ++k) {
                    const float2 p = *(const float2 *)(sums + (k * mine + i) * pitch + 64 * m);
                    v[m].x = fadd(v[m].x, p.x);
                    v[m].y = fadd(v[m].y, p.y);
                }
                if (!(keep >> (4 * m) & 1)) v[m].x = 0.0f;
                if (!(keep >> (4 * m) & 2)) v[m].y = 0.0f;
                most = fmaxf(most, fmaxf(fabsf(v[m].x), fabsf(v[m].y)));
            }
            if constexpr (TX == KV_F16) {
                const uint32_t exponent = __reduce_max_sync(0xffffffffu, __float_as_uint(most)) >> 23;
                float back = 1.0f;
                if (exponent > 20 && exponent < 255) {                 // 2^14 <= most * 2^(141 - exponent) < 2^15
                    const float to = __uint_as_float((268 - exponent) << 23);
                    back = __uint_as_float((exponent - 14) << 23);
#pragma unroll
                    for (int m = 0; m < LORA_PASS / 64; ++m) v[m].x = fmul(v[m].x, to), v[m].y = fmul(v[m].y, to);
                }
                if (lane < ctas) lt_store_peer(lt_peer(kvt_smem(&sh.row_scale[row]), lane), __float_as_uint(back));
            }
            uint32_t w[LORA_PASS / 64][S::PH];
#pragma unroll
            for (int m = 0; m < LORA_PASS / 64; ++m)
#pragma unroll
                for (int p = 0; p < S::PH; ++p) w[m][p] = lt_part<TX>(v[m]);
            const uint32_t at = base_at + (uint32_t)(lane >> 4) * LT_HALF + (uint32_t)row * 64 + (uint32_t)(((lane >> 2 & 3) ^ ((row >> 1) & 3)) << 4) + (uint32_t)(lane & 3) * 4;
            for (int k = 0; k < ctas; ++k) {
                const uint32_t to = lt_peer(at, k);
#pragma unroll
                for (int m = 0; m < LORA_PASS / 64; ++m)
                    if (keep >> (4 * m) & 4)
#pragma unroll
                        for (int p = 0; p < S::PH; ++p) lt_store_peer(to + (uint32_t)(p * plan.h_blocks + 2 * m) * LT_HALF, w[m][p]);
            }
        }
    }
    lt_async_fence();
    lora_cluster_arrive();
    lora_cluster_wait();                       // nothing of a peer's shared memory is read or written from here on
    lt_async_fence();
    if (worker) {
        for (int i = 0; i < min(2, my_tiles); ++i) issue_b(i);
        lt_commit();
        lt_wait_copies<0>();
        lt_async_fence();
        lt_arrive(&sh.b_full[0]);
        lt_arrive(&sh.b_full[1]);
    }

    if (!worker) {
        if (lane == 0) {
            int mt = t0, mt0 = 0;
            for (int i = 0; i < my_tiles; ++i) {
                while (tile_low + i - mt0 >= (a.width[mt] + S::COLS - 1) / S::COLS) mt0 += (a.width[mt] + S::COLS - 1) / S::COLS, ++mt;
                if (!wait(&sh.b_full[i & 1], (i >> 1) & 1)) break;
                if (i >= 2 && !wait(&sh.d2_free[i & 1], ((i >> 1) - 1) & 1)) break;
                kvt_after();
                const uint32_t b = base_at + plan.sum_at + (uint32_t)(i & 1) * b_bytes;
                bool add = false;
                for (int p = 0; p < S::PH; ++p)
                    for (int j = 0; j < rp; j += 16, add = true) {
                        const int at = (mt - t0) * rp + j;
                        lt_mma<TX>(tmem + (uint32_t)(i & 1) * 128, lt_desc64(base_at + (uint32_t)(p * plan.h_blocks + (at >> 5)) * LT_HALF + (uint32_t)(at & 31) * 2),
                                   lt_desc64(b + (uint32_t)(j >> 5) * (S::COLS * 64) + (uint32_t)(j & 31) * 2), S::COLS, add);
                    }
                kvt_commit(&sh.d2_done[i & 1]);
            }
            kvt_commit(&sh.drained);
        }
        __syncwarp();
    } else {
        // A warp: 32 rows, a half of the tile's outputs in chunks of 32.  For base and out lane l has 16 bytes of row 8 i + l / 4.
        const int q = warp & 3, half = warp >> 2, rl = lane >> 2, cl = (lane & 3) * 8;
        float *const lines = (float *)(tiles + plan.line_at) + warp * 32 * LT_LINE;
        int et = t0, et0 = 0, en = n_first;                            // of the tile whose base is asked for
        uint4 was[S::CHUNKS][4];
        int n_of = 0, left_of = 0;                                     // of that tile: the first output, those of its target from there on
        auto look_up = [&](int i) {
            const int tile = tile_low + i;
            while (tile - et0 >= (a.width[et] + S::COLS - 1) / S::COLS) {
                et0 += (a.width[et] + S::COLS - 1) / S::COLS;
                en += a.width[et];
                ++et;
            }
            n_of = en + (tile - et0) * S::COLS;
            left_of = a.width[et] - (tile - et0) * S::COLS;
        };
        auto ask = [&](int m) {
            if (!a.base || !a.wide) return;
            const int col = half * (S::COLS / 2) + 32 * m + cl;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int row = sh.row[32 * q + 8 * k + rl];
                if (row >= 0 && col + 8 <= left_of) was[m][k] = __ldcs((const uint4 *)((const char *)a.base + ((int64_t)row * a.base_stride + n_of + col) * 2));
            }
        };
        if (!a.base)
#pragma unroll
            for (int m = 0; m < S::CHUNKS; ++m)
#pragma unroll
                for (int k = 0; k < 4; ++k) was[m][k] = make_uint4(0, 0, 0, 0);
        if (my_tiles > 0) {
            look_up(0);
#pragma unroll
            for (int m = 0; m < S::CHUNKS; ++m) ask(m);
        }
        for (int i = 0; i < my_tiles; ++i) {
            const int n = n_of, left = left_of;
            if (i + 1 < my_tiles) look_up(i + 1);
            wait(&sh.d2_done[i & 1], (i >> 1) & 1);
            kvt_after();
            if (i + 2 < my_tiles) issue_b(i + 2);
            lt_commit();
#pragma unroll
            for (int m = 0; m < S::CHUNKS; ++m) {
                uint32_t v[32];
                kvt_load32(tmem + ((uint32_t)(32 * q) << 16) + (uint32_t)(i & 1) * 128 + half * (S::COLS / 2) + 32 * m, v);
                kvt_wait_ld();
                if (m == S::CHUNKS - 1) {
                    kvt_before();
                    lt_arrive(&sh.d2_free[i & 1]);
                }
                __syncwarp();
#pragma unroll
                for (int e = 0; e < 32; e += 4)
                    *(float4 *)(lines + lane * LT_LINE + e) = make_float4(__uint_as_float(v[e]), __uint_as_float(v[e + 1]), __uint_as_float(v[e + 2]), __uint_as_float(v[e + 3]));
                __syncwarp();
                const int col = half * (S::COLS / 2) + 32 * m + cl;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int at = 8 * k + rl, row = sh.row[32 * q + at];
                    if (row < 0 || col >= left) continue;
                    const float4 s0 = *(const float4 *)(lines + at * LT_LINE + cl), s1 = *(const float4 *)(lines + at * LT_LINE + cl + 4);
                    const float s[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
                    const float by = TX == KV_F16 ? scale * sh.row_scale[32 * q + at] : scale;
                    const int64_t to = (int64_t)row * a.out_stride + n + col;
                    if (a.wide && col + 8 <= left) {
                        __stcs((uint4 *)((char *)a.out + to * 2), lt_add<TX>(was[m][k], s, by));
                    } else {
                        for (int e = 0; e < min(8, left - col); ++e)
                            kv_store(a.out, to + e, TX, __fmaf_rn(by, s[e], a.base ? kv_load(a.base, (int64_t)row * a.base_stride + n + col + e, TX) : 0.0f));
                    }
                }
                if (i + 1 < my_tiles) ask(m);                          // of the next tile
            }
            lt_wait_copies<0>();
            lt_async_fence();
            if (i + 2 < my_tiles) lt_arrive(&sh.b_full[i & 1]);
        }
    }
    // Nothing reads or writes tensor memory any more once the last matrix instruction has come to its end.
    kvt_mbar_wait(&sh.drained, 0, NC_DRAIN_CYCLES);
    kvt_before();
    __syncthreads();
    kvt_after();
    if (warp == LT_WARPS) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(LT_TMEM) : "memory");
}

}  // namespace nc
