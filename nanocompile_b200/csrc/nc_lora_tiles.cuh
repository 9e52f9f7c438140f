// nc_lora_tiles.cuh -- low-rank adapters for prompts: what nc_lora.cuh computes, for items of up to 128 rows, on the tensor cores.
//
// An item to a cluster.  First each CTA multiplies its share of the inputs, 64 at a time: D1 [128 rows][h] += x A^T, tcgen05.mma with the
// rows and the adapter's A copied asynchronously into 128-byte swizzled tiles, D1 in tensor memory (float32 rows: each 64 inputs a D1 of
// their own, two in turn where there is room, added up by the four warps that load later).  The CTAs' sums of h are added
// through distributed shared memory: each CTA is sent its share of the rows, and copies them, added up and split into the
// operand's parts, to all.  Then each CTA expands its share of the outputs, 256 bytes of a row at a time: D2 [128][outputs] = h B^T in two
// halves of tensor memory.  Four warps ask for B and, up to four tiles ahead, for base; four warps add a tile's D2 to its base in shared
// memory, a row to a thread, and store it, whole rows to half a warp; four others have the next tile.  The targets' h lie side by side,
// whole 16s to each.
//
// Bound by the bytes of x, base and outputs, behind 14 us that no size takes away (tensor memory, two ways through the cluster).  8192
// bfloat16 rows of 4096 inputs to 6144 outputs at rank 32: 82 us (3.3 TB/s of 6.5; its products are 13 GFLOP, 8 us at the measured rate); 512 of them 29; float32
// rows 165 (3.3 TB/s), beside float16 weights 212.  While the sums of h were read from the peers the bfloat16 rows took 171 us, with base loaded
// by the warps that add it 122, in bulk copies of a row each 201.
//
// Accuracy.  16-bit rows and weights are multiplied as they are, h goes in two parts (bfloat16: 2^-17 of it is lost at most, float16
// 2^-23, or 2^-39 of the row's largest: that is first brought to [2^14, 2^15) by a power of two, so that no size leaves its range).  float32
// rows and their h go in three bfloat16 parts, float16 weights beside them in two, which hold them; of the products' parts 2^-25 is
// left out.  Sums are float32 in tensor memory; the matrix unit cuts them off at each step, always towards nought, which adds up along a
// chain.  So float32 rows have chains of 64 inputs, the largest parts' four steps last, added in float32: 8192 rows of 4096 inputs are
// 1.6e-7 of the result (rms) from 64 bits; in a chain of 2048 inputs they were 7.0e-6 beside bfloat16 weights, 1.2e-5 beside float16.
// 16-bit rows have one chain (float16: 1.7e-6 towards nought there, in outputs that are rounded by 2e-4).
#pragma once

#include "nc_kv4_prompt.cuh"
#include "nc_lora.cuh"

#include <type_traits>

namespace nc {

constexpr int LT_ROWS = 128, LT_WARPS = 8, LT_WORKERS = 32 * LT_WARPS, LT_LOADERS = 128;
constexpr int LT_MMA = LT_WARPS, LT_THREADS = LT_WORKERS + 32 + LT_LOADERS;            // the warp after the workers', then those that load
constexpr int LT_BLOCK = LT_ROWS * 128;        // 128 rows of 128 bytes
constexpr int LT_HALF = LT_ROWS * 64;          // 128 rows of 64 bytes
constexpr int LT_STAGES = 6;                   // of the first products at most
constexpr int LT_BYTES = 216 * 1024;           // of tiles at most
constexpr int LT_LINE = 272, LT_SLOT = LT_ROWS * LT_LINE;              // bytes from a row to the next of a tile of base: no bank twice in a quarter
// Rows that a CTA adds up, whole fours, and of all CTAs' shares at most: the last one's may be shorter (six CTAs have 24 rows each).
__host__ __device__ constexpr int lt_share(int ctas) { return (LT_ROWS / 4 + ctas - 1) / ctas * 4; }
constexpr int LT_SUM_ROWS = 144;
static_assert(2 * lt_share(2) <= LT_SUM_ROWS && 3 * lt_share(3) <= LT_SUM_ROWS && 4 * lt_share(4) <= LT_SUM_ROWS && 5 * lt_share(5) <= LT_SUM_ROWS &&
                  6 * lt_share(6) <= LT_SUM_ROWS && 7 * lt_share(7) <= LT_SUM_ROWS && 8 * lt_share(8) <= LT_SUM_ROWS,
              "room for the sums of every share");
constexpr int LT_SLOTS = 4;                    // tiles of base on their way or in work, at most

template <int TX, int TW>
struct LoraTiles {
    static constexpr bool F32 = TX == KV_F32;
    static constexpr int T = F32 ? (int)KV_BF16 : TX;                  // of the operands
    static constexpr int PX = F32 ? 3 : 1, PW = F32 && TW == KV_F16 ? 2 : 1, PH = F32 ? 3 : 2;   // parts of x, of weights, of h
    static constexpr int COLS = F32 ? 64 : 128;                        // outputs of a tile
    static constexpr int SIZE = F32 ? 4 : 2;
    static constexpr int TMEM = F32 ? 512 : 256;                       // columns: two halves of D2, before them D1, of float32 rows the chains and their sums
};

// How shared memory is laid out, by the most rows of h in a pass: h's operand, two tiles of B, the slots of base; over these the stages of
// the first products.  Where there is room the sums of h lie past the stages and the first two slots (`early`): then they may come while
// a CTA is still at its stages, and the first tiles of B and base while they are added up.  Else they lie over B and the slots.
struct LoraTilesPlan {
    int wide;                                  // rows of h in whole 16s
    int stages, a_bytes;                       // of a stage: LT_BLOCK for a part of the rows, a_bytes for one of A
    int h_blocks, b_blocks;                    // blocks of 32 for a part of h, for B
    int b_at, slot_at, slots, sum_at, early, bytes;
    int chains, chain_step;                    // float32 rows: chains of products in tensor memory, 32s of columns apart, and their sums behind
};
template <typename S>
inline LoraTilesPlan lora_tiles_plan(int targets, int rank) {
    LoraTilesPlan p{};
    p.wide = targets * ((rank + 15) / 16 * 16);
    p.a_bytes = p.wide * 128;
    p.h_blocks = (p.wide + 31) / 32;
    p.b_blocks = (rank + 31) / 32;
    p.b_at = S::PH * p.h_blocks * LT_HALF;
    p.slot_at = p.b_at + 2 * S::PW * p.b_blocks * S::COLS * 64;
    // Two or four, that a slot is always the same warps': they wait for every second tile only, and would take the round of a slot's
    // barrier before the one that they wait for, of the same parity, for that.
    p.slots = (LT_BYTES - p.slot_at) / LT_SLOT / 2 * 2;
    if (p.slots > LT_SLOTS) p.slots = LT_SLOTS;
    p.bytes = p.slot_at + p.slots * LT_SLOT;
    const int sums = LT_SUM_ROWS * (p.wide + 4) * 4, stage = S::PX * LT_BLOCK + S::PW * p.a_bytes;
    p.sum_at = p.slot_at + 2 * LT_SLOT;
    p.early = p.sum_at + sums <= LT_BYTES && 2 * stage <= p.sum_at;
    if (!p.early) p.sum_at = p.b_at;
    if (p.sum_at + sums > p.bytes) p.bytes = p.sum_at + sums;
    const int room = p.early ? p.sum_at : LT_BYTES;
    p.stages = room / stage < LT_STAGES ? room / stage : LT_STAGES;
    if (p.stages * stage > p.bytes) p.bytes = p.stages * stage;
    p.chain_step = p.h_blocks * 32;
    p.chains = 3 * p.chain_step <= S::TMEM ? 2 : 1;
    return p;
}

struct LoraTilesShared {                       // before the tiles
    uint64_t full[LT_STAGES], empty[LT_STAGES], chain_full[2], chain_free[2], d1_done, b_full[2], d2_done[2], d2_free[2], slot_full[LT_SLOTS], slot_free[LT_SLOTS], h_full, drained;
    __align__(16) float row_scale[LT_ROWS];
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
__device__ __forceinline__ void lt_async_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
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
__device__ __forceinline__ void lt_store_peer(uint32_t at, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
template <int TW>
__device__ constexpr float lt_most() { return TW == KV_BF16 ? 3.3895314e38f : 65504.0f; }        // the largest number
// Two values rounded to 16 bits, and what that leaves: nothing of an infinity.  What would round to an infinity is cut off.  SURE: neither is
// larger than lt_most, nor an infinity.
template <int TW, bool SURE = false>
__device__ __forceinline__ uint32_t lt_part(float2 &v) {
    auto round = [](float2 f, float2 *r) {
        uint32_t w;
        if constexpr (TW == KV_BF16) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(f.x, f.y);
            w = *reinterpret_cast<const uint32_t *>(&b);
            *r = __bfloat1622float2(b);
        } else {
            const __half2 b = __floats2half2_rn(f.x, f.y);
            w = *reinterpret_cast<const uint32_t *>(&b);
            *r = __half22float2(b);
        }
        return w;
    };
    float2 r;
    uint32_t w = round(v, &r);
    if (!SURE && !(fabsf(r.x) < INFINITY && fabsf(r.y) < INFINITY)) {
        constexpr float most = lt_most<TW>();
        auto cut = [](float f) { return fabsf(f) < INFINITY ? fminf(fmaxf(f, -most), most) : f; };
        w = round(make_float2(cut(v.x), cut(v.y)), &r);
        v.x = fabsf(r.x) < INFINITY ? fsub(v.x, r.x) : 0.0f;
        v.y = fabsf(r.y) < INFINITY ? fsub(v.y, r.y) : 0.0f;
        return w;
    }
    v.x = fsub(v.x, r.x);
    v.y = fsub(v.y, r.y);
    return w;
}
// v += sum.
__device__ __forceinline__ void lt_sums(uint32_t (&v)[16], const uint32_t (&sum)[16]) {
#pragma unroll
    for (int e = 0; e < 16; e += 2) {
        const float2 f = unpack2(add2(pack2(__uint_as_float(sum[e]), __uint_as_float(sum[e + 1])), pack2(__uint_as_float(v[e]), __uint_as_float(v[e + 1]))));
        v[e] = __float_as_uint(f.x);
        v[e + 1] = __float_as_uint(f.y);
    }
}
// 16 bytes of outputs from those of base and float32 sums.
template <int TX>
__device__ __forceinline__ uint4 lt_add(const uint4 &was, const uint32_t *sums, float scale) {
    const float *const v = reinterpret_cast<const float *>(sums);
    if constexpr (TX == KV_F32)
        return make_uint4(__float_as_uint(__fmaf_rn(scale, v[0], __uint_as_float(was.x))), __float_as_uint(__fmaf_rn(scale, v[1], __uint_as_float(was.y))),
                          __float_as_uint(__fmaf_rn(scale, v[2], __uint_as_float(was.z))), __float_as_uint(__fmaf_rn(scale, v[3], __uint_as_float(was.w))));
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

// What a worker has of a block of float32 rows, and of float16 weights beside them.
struct LtBlock {
    float4 x[8];
    uint4 w[LORA_PASS / 32];
};
// The products of parts that count: of p + q up to the third, the largest last, as each step cuts off what the whole sum has no bits for.
template <int P, int Q, typename F>
__device__ __forceinline__ void lt_parts(F use) {
#pragma unroll
    for (int s = 2; s >= 0; --s)
#pragma unroll
        for (int q = 0; q < Q; ++q)
            if (s - q >= 0 && s - q < P) use(s - q, q);
}
// use(std::true_type) where numbers up to `most` are sure, else use(std::false_type).
template <int TW, typename F>
__device__ __forceinline__ void lt_sure(float most, F use) {
    if (most <= lt_most<TW>()) use(std::true_type());
    else use(std::false_type());
}
// Eight float16 weights in two bfloat16 parts, which hold them exactly.
__device__ __forceinline__ void lt_two_parts(const uint4 &w, uint4 *high, uint4 *low) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
    uint32_t h[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u[i]));
        float2 rest = f;
        h[i] = lt_part<KV_BF16, true>(rest);
        rest = make_float2(fabsf(f.x) < INFINITY ? rest.x : 0.0f, fabsf(f.y) < INFINITY ? rest.y : 0.0f);
        l[i] = lt_part<KV_BF16, true>(rest);
    }
    *high = make_uint4(h[0], h[1], h[2], h[3]);
    *low = make_uint4(l[0], l[1], l[2], l[3]);
}

template <int TX, int TW>
__global__ void __launch_bounds__(LT_THREADS, 1) lora_tiles_kernel(const __grid_constant__ LoraArgs a, const __grid_constant__ LoraTilesPlan plan) {
    using S = LoraTiles<TX, TW>;
    extern __shared__ __align__(1024) char lt_raw[];
    char *const tiles = lt_raw + ((1024 - (kvt_smem(lt_raw) & 1023)) & 1023);
    __shared__ LoraTilesShared sh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const bool worker = warp < LT_WARPS;
    const int ctas = (int)lora_cluster_size(), cta = (int)lora_rank_of_cluster();
    wait_for_producer();
    const int4 item = lora_item(a, blockIdx.x / ctas);
    const int32_t *const order = (const int32_t *)(lora_items(a.plan) + a.items);
    const int slot = item.x, first = item.y, count = min(LT_ROWS, item.z);
    if (count <= 0) return;
    const int t0 = (int)blockIdx.y * a.pass_targets, t1 = min(a.targets, t0 + a.pass_targets);
    int n_first = 0, n_pass = 0, n_tiles = 0;                          // outputs before the pass, of it, tiles of them
    for (int t = 0; t < t1; ++t) {
        if (t < t0) n_first += a.width[t];
        else n_pass += a.width[t], n_tiles += (a.width[t] + S::COLS - 1) / S::COLS;
    }
    // What depends on the item is asked for together.
    const int my_row = tid < count ? (int)lora_row(a, order, first + tid) : -1, rank = a.ranks ? a.ranks[max(slot, 0)] : a.rank;
    const float scale = a.scales ? a.scales[max(slot, 0)] : 1.0f;
    const int r = slot < 0 ? 0 : min(max(rank, 0), a.rank);
    if (r == 0) {
        const int64_t n = n_pass;
        lora_copy<TX>(a, order, first, count, n_first + (int)(n * cta / ctas), n_first + (int)(n * (cta + 1) / ctas));
        return;
    }
    const int rp = (r + 15) / 16 * 16, wide = (t1 - t0) * rp;
    const char *const wa = (const char *)a.a + ((int64_t)slot * a.targets + t0) * a.rank * a.inputs * 2;
    const char *const wb = (const char *)a.b + (int64_t)slot * a.outputs * a.rank * 2;
    const int tile_low = (int)((int64_t)n_tiles * cta / ctas), tile_high = (int)((int64_t)n_tiles * (cta + 1) / ctas), my_tiles = tile_high - tile_low;
    const int blocks = (a.inputs + 63) / 64, k_low = (int)((int64_t)blocks * cta / ctas), k_blocks = (int)((int64_t)blocks * (cta + 1) / ctas) - k_low;
    {
        const int64_t low = ((int64_t)n_first + S::COLS * tile_low) * a.rank * 2, high = min((int64_t)n_first + n_pass, (int64_t)n_first + S::COLS * tile_high) * a.rank * 2;
        for (int64_t at = low + tid * 4096; at < high; at += LT_THREADS * 4096)
            asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(wb + at), "r"((uint32_t)min((int64_t)4096, high - at)) : "memory");
    }
    if (warp == LT_MMA) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(kvt_smem(&sh.tmem)), "n"(S::TMEM) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid == 0) {
        for (int i = 0; i < plan.stages; ++i) lt_init(&sh.full[i], LT_WORKERS), lt_init(&sh.empty[i], 1);
        lt_init(&sh.d1_done, S::F32 ? LT_LOADERS : 1);
        for (int i = 0; i < 2; ++i) lt_init(&sh.chain_full[i], 1), lt_init(&sh.chain_free[i], LT_LOADERS);
        lt_init(&sh.drained, 1);
        for (int i = 0; i < 2; ++i) lt_init(&sh.b_full[i], LT_LOADERS), lt_init(&sh.d2_done[i], 1), lt_init(&sh.d2_free[i], LT_ROWS);
        for (int i = 0; i < LT_SLOTS; ++i) lt_init(&sh.slot_full[i], LT_LOADERS), lt_init(&sh.slot_free[i], LT_ROWS);
        lt_init(&sh.h_full, 1);
        sh.failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (tid < LT_ROWS) sh.row[tid] = my_row;
    kvt_before();
    const bool all_rows = __syncthreads_and(tid >= LT_ROWS || my_row >= 0);    // 128 of them, and each is one of the call
    kvt_after();
    release_dependents();                      // not before this CTA has its tensor memory: a dependent may hold all the rest
    if (plan.early) lora_cluster_arrive();     // this CTA is there: peers may write to its shared memory
    const uint32_t tmem = sh.tmem, base_at = kvt_smem(tiles);
    const long long limit = g_wait_cycles;
    // A wait that runs out is the last one: the CTA goes on without waiting and its outputs are not to be used.
    auto wait = [&](uint64_t *bar, unsigned parity) {
        if (kvt_mbar_wait(bar, parity, *(volatile int *)&sh.failed ? 0 : limit)) return true;
        *(volatile int *)&sh.failed = 1;
        atomicOr(&g_lora_fault, LORA_LATE);
        return false;
    };
    const int stage_bytes = S::PX * LT_BLOCK + S::PW * plan.a_bytes, c = tid & 7, line = tid >> 3;             // a worker's 16 bytes of every 32nd row

    // h, in parts: D1 = x A^T over this CTA's inputs.  Of float32 rows each block of 64 inputs is a chain of its own; the warps that load
    // later add up all but the last in tensor memory.
    const uint32_t d1 = S::F32 ? tmem + plan.chains * plan.chain_step : tmem;
    if (worker) {
        int from[LORA_PASS / 32];                                      // of A's rows; -1: none there
#pragma unroll
        for (int i = 0; i < LORA_PASS / 32; ++i) {
            const int j = line + 32 * i, t = j / rp;
            from[i] = j < wide && j - t * rp < r ? (t * a.rank + j - t * rp) * a.inputs : -1;
        }
        const uint32_t swizzled = (uint32_t)line * 128 + (uint32_t)((c ^ (line & 7)) << 4);
        auto ask_a = [&](int k) {
            const uint32_t to = base_at + (uint32_t)(k % plan.stages) * stage_bytes + S::PX * LT_BLOCK + swizzled;
            const int e = (k_low + k) * 64 + 8 * c;
#pragma unroll
            for (int i = 0; i < LORA_PASS / 32; ++i) {
                const bool there = e < a.inputs && from[i] >= 0;
                if (line + 32 * i < wide) lt_copy16(to + i * 4096, there ? wa + (int64_t)(from[i] + e) * 2 : wa, there ? 16 : 0);
            }
        };
        if constexpr (!S::F32) {
            const char *x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = sh.row[line + 32 * i];
                x[i] = row < 0 ? nullptr : (const char *)a.x + (int64_t)row * a.x_stride * 2;
            }
            auto issue = [&](int k) {
                const uint32_t to = base_at + (uint32_t)(k % plan.stages) * stage_bytes + swizzled;
                const int e = (k_low + k) * 64 + 8 * c;
                const bool in = e < a.inputs;
#pragma unroll
                for (int i = 0; i < 4; ++i) lt_copy16(to + i * 4096, in && x[i] ? x[i] + e * 2 : a.x, in && x[i] ? 16 : 0);
                ask_a(k);
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
                switch (ahead) {                                       // the oldest of `ahead` + 1 groups is there
                    case 1: lt_wait_copies<1>(); break;
                    case 2: lt_wait_copies<2>(); break;
                    case 3: lt_wait_copies<3>(); break;
                    default: lt_wait_copies<4>(); break;
                }
                lt_async_fence();
                lt_arrive(&sh.full[k % plan.stages]);
            }
        } else {
            // float32 rows go through registers, a block ahead: four values of every 16th row to a thread, split into parts on the way.  Few
            // instructions count here, more than loads further ahead: 8192 rows 4096 -> 6144 take 165 us, 178 with two blocks ahead, 172 with
            // the loop unrolled and the parts of seldom numbers in it.
            const int c4 = tid & 15, line4 = tid >> 4;
            auto fetch = [&](int k, int i) {
                const int e = (k_low + k) * 64 + 4 * c4, row = sh.row[line4 + 16 * i];
                return row >= 0 && e < a.inputs ? __ldg((const float4 *)((const float *)a.x + (int64_t)row * a.x_stride + e)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            };
            auto load = [&](int k, LtBlock &block) {
#pragma unroll
                for (int i = 0; i < 8; ++i) block.x[i] = fetch(k, i);
            };
            auto load_a = [&](int k, LtBlock &block) {
                if constexpr (S::PW == 1) {
                    ask_a(k);
                } else {
                    const int ea = (k_low + k) * 64 + 8 * c;
#pragma unroll
                    for (int i = 0; i < LORA_PASS / 32; ++i) {
                        block.w[i] = make_uint4(0, 0, 0, 0);
                        if (from[i] >= 0 && ea < a.inputs) block.w[i] = __ldg((const uint4 *)(wa + (int64_t)(from[i] + ea) * 2));
                    }
                }
                lt_commit();
            };
            auto store = [&](int k, const LtBlock &block) {
                const uint32_t at = base_at + (uint32_t)(k % plan.stages) * stage_bytes;
                float most = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    most = fmaxf(fmaxf(most, fmaxf(fabsf(block.x[i].x), fabsf(block.x[i].y))), fmaxf(fabsf(block.x[i].z), fabsf(block.x[i].w)));
                auto put = [&](int i, const float4 &from, auto sure) {
                    const int row = line4 + 16 * i;
                    const uint32_t to = at + (uint32_t)row * 128 + (uint32_t)(((c4 >> 1) ^ (row & 7)) << 4) + (uint32_t)(c4 & 1) * 8;
                    float2 x = make_float2(from.x, from.y), y = make_float2(from.z, from.w);
#pragma unroll
                    for (int p = 0; p < S::PX; ++p) {
                        const uint32_t u = lt_part<KV_BF16, decltype(sure)::value>(x), v = lt_part<KV_BF16, decltype(sure)::value>(y);
                        asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(to + p * LT_BLOCK), "r"(u), "r"(v) : "memory");
                    }
                };
#pragma unroll
                for (int i = 0; i < 8; ++i) put(i, block.x[i], std::true_type());
                if (!(most <= lt_most<KV_BF16>()))                     // seldom: once more, in few instructions
#pragma unroll 1
                    for (int i = 0; i < 8; ++i) put(i, fetch(k, i), std::false_type());
                if constexpr (S::PW == 2) {
#pragma unroll
                    for (int i = 0; i < LORA_PASS / 32; ++i) {
                        if (line + 32 * i >= wide) continue;
                        uint4 high, low;
                        lt_two_parts(block.w[i], &high, &low);
                        const uint32_t to = at + S::PX * LT_BLOCK + swizzled + i * 4096;
                        store16_shared(to, high.x, high.y, high.z, high.w);
                        store16_shared(to + plan.a_bytes, low.x, low.y, low.z, low.w);
                    }
                }
            };
            LtBlock now, next;
            auto wait_for = [&](int k) {                               // the stage of block k
                if (k >= plan.stages) wait(&sh.empty[k % plan.stages], (k / plan.stages - 1) & 1);
            };
            if (k_blocks > 0) load(0, now), load_a(0, now);
#pragma unroll 1
            for (int k = 0; k < k_blocks; ++k) {
                if (k + 1 < k_blocks) {
                    load(k + 1, next);                                 // before the wait: 8192 rows 194 us behind it
                    if constexpr (S::PW == 1) wait_for(k + 1);
                    load_a(k + 1, next);
                } else {
                    lt_commit();
                }
                if constexpr (S::PW == 2) wait_for(k);                 // its weights come through registers, and nothing before the store needs the stage
                store(k, now);
                lt_wait_copies<1>();
                lt_async_fence();
                lt_arrive(&sh.full[k % plan.stages]);
                now = next;
            }
        }
        lt_wait_copies<0>();
    } else if (warp == LT_MMA && lane == 0) {
        for (int k = 0; k < k_blocks; ++k) {
            const int stage = k % plan.stages, chain = S::F32 ? k % plan.chains : 0, turn = S::F32 ? k / plan.chains : 0;
            const int steps = min(4, (a.inputs - (k_low + k) * 64 + 15) / 16);
            const uint32_t at = base_at + (uint32_t)stage * stage_bytes, to = tmem + chain * plan.chain_step;
            const uint64_t x = kvt_desc(at), w = kvt_desc(at + S::PX * LT_BLOCK);                 // addresses in them are in 16s of bytes
            if (turn > 0 && !wait(&sh.chain_free[chain], (turn - 1) & 1)) break;
            if (!wait(&sh.full[stage], (k / plan.stages) & 1)) break;
            kvt_after();
            bool add = !S::F32 && k > 0;
            lt_parts<S::PX, S::PW>([&](int p, int q) {
#pragma unroll
                for (int s = 0; s < 4; ++s, add = true)
                    if (s < steps) lt_mma<S::T>(to, x + (p * LT_BLOCK + 32 * s) / 16, w + (q * plan.a_bytes + 32 * s) / 16, wide, add);
            });
            kvt_commit(&sh.empty[stage]);
            if (S::F32) kvt_commit(&sh.chain_full[chain]);
        }
        if (!S::F32) kvt_commit(&sh.d1_done);
    } else if (S::F32 && warp > LT_MMA) {
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        for (int k = 0; k + 1 < k_blocks; ++k) {                       // the last one's stays where it is
            const int chain = k % plan.chains;
            wait(&sh.chain_full[chain], (k / plan.chains) & 1);
            kvt_after();
            __syncwarp();
            for (int j = 0; j < wide; j += 16) {
                uint32_t v[16], sum[16];
                kvt_load16(tmem + lanes + chain * plan.chain_step + j, v);
                if (k > 0) kvt_load16(d1 + lanes + j, sum);
                kvt_wait_ld();
                if (k > 0) lt_sums(v, sum);
                kvt_store16(d1 + lanes + j, v);
            }
            kvt_before();
            lt_arrive(&sh.chain_free[chain]);
            kvt_wait_st();
        }
        kvt_before();
        lt_arrive(&sh.d1_done);
    }
    __syncwarp();
    wait(&sh.d1_done, 0);
    const uint32_t last = S::F32 && k_blocks > 0 ? (k_blocks - 1) % plan.chains : 0;
    if (S::F32 && k_blocks > 0) wait(&sh.chain_full[last], ((k_blocks - 1) / plan.chains) & 1);
    kvt_after();
    __syncwarp();
    if (!plan.early) lora_cluster_arrive();    // this CTA is done with its stages: sums may lie over them
    lora_cluster_wait();
    const int mine = lt_share(ctas), pitch = plan.wide + 4;
    if (worker) {
        // The CTA's sums go to the CTAs that add them up: a row to a thread, 16 columns at a time, a half of them to a warp.
        const int row = 32 * (warp & 3) + lane;
        const bool here = row / mine == cta;
        const uint32_t at = base_at + plan.sum_at + (uint32_t)((cta * mine + row % mine) * pitch) * 4, to = lt_peer(at, row / mine);
        for (int j = 16 * (warp >> 2); j < wide; j += 32) {
            uint32_t v[16], sum[16];
            kvt_load16(tmem + ((uint32_t)(32 * (warp & 3)) << 16) + last * plan.chain_step + j, v);
            if (S::F32 && k_blocks > 1) kvt_load16(d1 + ((uint32_t)(32 * (warp & 3)) << 16) + j, sum);
            kvt_wait_ld();
            if (S::F32 && k_blocks > 1) lt_sums(v, sum);
            if (k_blocks == 0)                                         // more CTAs than blocks of inputs
#pragma unroll
                for (int e = 0; e < 16; ++e) v[e] = 0;
#pragma unroll
            for (int e = 0; e < 16; e += 4)
                if (here) store16_shared(at + (j + e) * 4, v[e], v[e + 1], v[e + 2], v[e + 3]);
                else lt_store_peer(to + (j + e) * 4, v[e], v[e + 1], v[e + 2], v[e + 3]);
        }
    }
    kvt_before();
    __syncwarp();
    lora_cluster_arrive();
    if (warp <= LT_MMA) lora_cluster_wait();   // those that load go on
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
        // Four rows at a time, that their loads do not wait for one another.
        constexpr int M = LORA_PASS / 64, R = 4;
        const int rows = min(mine, LT_ROWS - cta * mine);
        for (int i0 = warp; i0 < rows; i0 += R * LT_WARPS) {
            float2 v[R][M];
#pragma unroll
            for (int u = 0; u < R; ++u)
#pragma unroll
                for (int m = 0; m < M; ++m) v[u][m] = make_float2(0.0f, 0.0f);
            for (int k = 0; k < ctas; ++k)
#pragma unroll
                for (int u = 0; u < R; ++u) {
                    const int i = min(i0 + u * LT_WARPS, rows - 1);
#pragma unroll
                    for (int m = 0; m < M; ++m) {
                        if (!(keep >> (4 * m) & 4)) continue;
                        const float2 p = *(const float2 *)(sums + (k * mine + i) * pitch + 64 * m);
                        v[u][m].x = fadd(v[u][m].x, p.x);
                        v[u][m].y = fadd(v[u][m].y, p.y);
                    }
                }
#pragma unroll
            for (int u = 0; u < R; ++u) {
                if (i0 + u * LT_WARPS >= rows) break;
                const int row = cta * mine + i0 + u * LT_WARPS;
                float most = 0.0f;
#pragma unroll
                for (int m = 0; m < M; ++m) {
                    if (!(keep >> (4 * m) & 1)) v[u][m].x = 0.0f;
                    if (!(keep >> (4 * m) & 2)) v[u][m].y = 0.0f;
                    most = fmaxf(most, fmaxf(fabsf(v[u][m].x), fabsf(v[u][m].y)));
                }
                if constexpr (TX == KV_F16) {
                    const uint32_t exponent = __reduce_max_sync(0xffffffffu, __float_as_uint(most)) >> 23;
                    float back = 1.0f;
                    if (exponent > 20 && exponent < 255) {             // 2^14 <= most * 2^(141 - exponent) < 2^15
                        const float to = __uint_as_float((268 - exponent) << 23);
                        back = __uint_as_float((exponent - 14) << 23);
#pragma unroll
                        for (int m = 0; m < M; ++m) v[u][m].x = fmul(v[u][m].x, to), v[u][m].y = fmul(v[u][m].y, to);
                        most = 1.0f;                               // some number
                    }
                    if (lane == 0) sh.row_scale[row] = back;
                }
                const uint32_t at = base_at + (uint32_t)(lane >> 4) * LT_HALF + (uint32_t)row * 64 + (uint32_t)(((lane >> 2 & 3) ^ ((row >> 1) & 3)) << 4) + (uint32_t)(lane & 3) * 4;
                lt_sure<S::T>(most, [&](auto sure) {
#pragma unroll
                    for (int m = 0; m < M; ++m) {
                        if (!(keep >> (4 * m) & 4)) continue;
#pragma unroll
                        for (int p = 0; p < S::PH; ++p) {
                            const uint32_t w = lt_part<S::T, decltype(sure)::value>(v[u][m]);
                            asm volatile("st.shared.u32 [%0], %1;" ::"r"(at + (uint32_t)(p * plan.h_blocks + 2 * m) * LT_HALF), "r"(w) : "memory");
                        }
                    }
                });
            }
        }
        lt_async_fence();
    }
    if (worker) {
        asm volatile("bar.sync 1, %0;" ::"n"(LT_WORKERS) : "memory");  // h's rows of this CTA are there, and the sums read:
        asm volatile("bar.arrive 2, %0;" ::"n"(LT_WORKERS + LT_LOADERS) : "memory");             // what lies over them may come
    }
    if (warp == 0) {
        // To each peer this CTA's rows of every block, 64 bytes each, and their scales: one bulk copy a lane.
        const int from_row = cta * mine, rows = min(mine, LT_ROWS - from_row), used = (wide + 31) / 32, per = S::PH * used + (TX == KV_F16);
        if (lane == 0)
            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(kvt_smem(&sh.h_full)),
                         "r"((LT_ROWS - rows) * (S::PH * used * 64 + (TX == KV_F16 ? 4 : 0)))
                         : "memory");
        __syncwarp();
        for (int i = lane; i < per * (ctas - 1); i += 32) {
            const int k = i / per, peer = k + (k >= cta), which = i - k * per;
            const bool scales = which == S::PH * used;
            const uint32_t at = scales ? kvt_smem(&sh.row_scale[from_row]) : base_at + (uint32_t)(which / used * plan.h_blocks + which % used) * LT_HALF + (uint32_t)from_row * 64;
            asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(lt_peer(at, peer)), "r"(at),
                         "r"(rows * (scales ? 4 : 64)), "r"(lt_peer(kvt_smem(&sh.h_full), peer))
                         : "memory");
        }
        __syncwarp();
    }

    // Tiles: `look_up` goes on to tile i of this CTA, in ascending order.
    int target = t0, tile0 = 0, n_target = n_first;
    auto look_up = [&](int i) {
        while (tile_low + i - tile0 >= (a.width[target] + S::COLS - 1) / S::COLS) {
            tile0 += (a.width[target] + S::COLS - 1) / S::COLS;
            n_target += a.width[target];
            ++target;
        }
        return (tile_low + i - tile0) * S::COLS;                       // the tile's first output of its target
    };
    const int b_part = plan.b_blocks * S::COLS * 64, b_bytes = S::PW * b_part;
    const bool staged = a.wide != 0;
    if (warp > LT_MMA) {
        // B's rows in blocks of 32, 64 bytes each, 16 of every 32nd row to a thread; base's rows, 16 bytes of every eighth to a thread.
        const int at = tid - LT_WORKERS - 32, bc = at & 3, bl = at >> 2, cc = at & 15, cl = at >> 4;
        // float16 weights beside float32 rows go through registers, a tile ahead.
        constexpr int BN = S::PW == 2 ? S::COLS / 32 : 1, BJ = S::PW == 2 ? LORA_RANK / 32 : 1;
        uint4 held[BN][BJ];
        auto fetch_b = [&](int n0) {
#pragma unroll
            for (int n = 0; n < BN; ++n)
#pragma unroll
                for (int j = 0; j < BJ; ++j) {
                    held[n][j] = make_uint4(0, 0, 0, 0);
                    if (32 * j + 8 * bc < r && n0 + bl + 32 * n < a.width[target])
                        held[n][j] = __ldg((const uint4 *)(wb + (((int64_t)n_target + n0 + bl + 32 * n) * a.rank + 32 * j + 8 * bc) * 2));
                }
        };
        // What lies past the adapter's own rank may be anything.
        auto within = [&](const uint4 &w, int j) {
            uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) u[e] = j + 2 * e >= r ? 0u : j + 2 * e + 1 >= r ? u[e] & 0xffffu : u[e];
            return make_uint4(u[0], u[1], u[2], u[3]);
        };
        auto issue_b = [&](int i, int n0) {
            const uint32_t to = base_at + plan.b_at + (uint32_t)(i & 1) * b_bytes;
            if constexpr (S::PW == 2) {
#pragma unroll
                for (int n = 0; n < BN; ++n)
#pragma unroll
                    for (int j = 0; j < BJ; ++j) {
                        if (32 * j + 8 * bc >= rp) continue;
                        const uint32_t dst = to + (uint32_t)(j * S::COLS + bl + 32 * n) * 64 + (uint32_t)((bc ^ ((bl >> 1) & 3)) << 4);
                        uint4 high, low;
                        lt_two_parts(within(held[n][j], 32 * j + 8 * bc), &high, &low);
                        store16_shared(dst, high.x, high.y, high.z, high.w);
                        store16_shared(dst + b_part, low.x, low.y, low.z, low.w);
                    }
                lt_commit();
                return;
            }
            if (r == rp && n0 + S::COLS <= a.width[target]) {
                const char *const from = wb + (((int64_t)n_target + n0 + bl) * a.rank + 8 * bc) * 2;
                const uint32_t dst = to + (uint32_t)bl * 64 + (uint32_t)((bc ^ ((bl >> 1) & 3)) << 4);     // the same for every 32nd row
                for (int j = 0; 8 * bc + j < rp; j += 32)
#pragma unroll
                    for (int n = 0; n < S::COLS; n += LT_LOADERS / 4)
                        lt_copy16(dst + (uint32_t)(j >> 5) * (S::COLS * 64) + n * 64, from + ((int64_t)n * a.rank + j) * 2, 16);
                lt_commit();
                return;
            }
            for (int n = bl; n < S::COLS; n += LT_LOADERS / 4)
                for (int j = 8 * bc; j < rp; j += 32) {
                    const uint32_t dst = to + (uint32_t)(j >> 5) * (S::COLS * 64) + (uint32_t)n * 64 + (uint32_t)((bc ^ ((n >> 1) & 3)) << 4);
                    const char *const from = wb + (((int64_t)n_target + n0 + n) * a.rank + j) * 2;
                    const bool there = n0 + n < a.width[target];
                    if (j + 8 <= r || j >= r || !there) {
                        lt_copy16(dst, there && j < r ? from : wb, there && j < r ? 16 : 0);
                    } else {
                        const uint4 w = within(__ldg((const uint4 *)from), j);
                        store16_shared(dst, w.x, w.y, w.z, w.w);
                    }
                }
            lt_commit();
        };
        auto ask_base = [&](int i, int n0) {
            const int slot_i = i % plan.slots, left = a.width[target] - n0;
            if (i >= plan.slots) wait(&sh.slot_free[slot_i], (i / plan.slots - 1) & 1);
            const uint32_t to = base_at + plan.slot_at + (uint32_t)(slot_i * LT_SLOT + cc * 16);
            const char *const from = (const char *)a.base + ((int64_t)n_target + n0) * S::SIZE + cc * 16;
            if (all_rows && left >= S::COLS) {
#pragma unroll
                for (int k = 0; k < LT_ROWS; k += LT_LOADERS / 16)
                    lt_copy16(to + (k + cl) * LT_LINE, from + (int64_t)sh.row[k + cl] * a.base_stride * S::SIZE, 16);
            } else if ((cc + 1) * (16 / S::SIZE) <= left)
#pragma unroll 4
                for (int k = cl; k < LT_ROWS; k += LT_LOADERS / 16) {
                    const int row = sh.row[k];
                    if (row >= 0) lt_copy16(to + k * LT_LINE, from + (int64_t)row * a.base_stride * S::SIZE, 16);
                }
            asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(kvt_smem(&sh.slot_full[slot_i])) : "memory");
        };
        // Tile i's B is waited for once the next one's is asked for; base is asked for as slots become free, and its copies
        // report to the slot's barrier themselves.
        const int late = plan.early ? min(2, my_tiles) : 0;            // the first tile that lies over the sums
        if constexpr (S::PW == 2)
            if (my_tiles > 0) fetch_b(look_up(0));
        for (int i = 0; i <= my_tiles; ++i) {
            int n0 = 0;
            if (i == late) asm volatile("bar.sync 2, %0;" ::"n"(LT_WORKERS + LT_LOADERS) : "memory");
            if (i < my_tiles) {
                if (i >= 2) wait(&sh.d2_done[i & 1], ((i >> 1) - 1) & 1);
                n0 = look_up(i);
                issue_b(i, n0);
            }
            if (i > 0) {
                if (i < my_tiles) lt_wait_copies<1>();
                else lt_wait_copies<0>();
                lt_async_fence();
                lt_arrive(&sh.b_full[(i - 1) & 1]);
            }
            if (i == my_tiles) break;
            if (staged && a.base) ask_base(i, n0);
            if constexpr (S::PW == 2)
                if (i + 1 < my_tiles) fetch_b(look_up(i + 1));
        }
        lt_wait_copies<0>();
        __syncwarp();
        lora_cluster_wait();                   // for the sums
    } else if (warp == LT_MMA) {
        if (lane == 0) {
            const bool ready = wait(&sh.h_full, 0);
            lt_async_fence();
            for (int i = 0; i < my_tiles && ready; ++i) {
                look_up(i);
                if (!wait(&sh.b_full[i & 1], (i >> 1) & 1)) break;
                if (i >= 2 && !wait(&sh.d2_free[i & 1], ((i >> 1) - 1) & 1)) break;
                kvt_after();
                const uint32_t b = base_at + plan.b_at + (uint32_t)(i & 1) * b_bytes;
                bool add = false;
                lt_parts<S::PH, S::PW>([&](int p, int q) {
                    for (int j = 0; j < rp; j += 16, add = true) {
                        const int at = (target - t0) * rp + j;
                        lt_mma<S::T>(tmem + (uint32_t)(i & 1) * 128, lt_desc64(base_at + (uint32_t)(p * plan.h_blocks + (at >> 5)) * LT_HALF + (uint32_t)(at & 31) * 2),
                                     lt_desc64(b + q * b_part + (uint32_t)(j >> 5) * (S::COLS * 64) + (uint32_t)(j & 31) * 2), S::COLS, add);
                    }
                });
                kvt_commit(&sh.d2_done[i & 1]);
            }
            kvt_commit(&sh.drained);
        }
        __syncwarp();
    } else {
        // Every other tile, a row to a thread.
        if constexpr (TX == KV_F16) wait(&sh.h_full, 0);               // the rows' scales
        const int at = 32 * (warp & 3) + lane, row = sh.row[at], half = warp >> 2, cc = lane & 15, cl = lane >> 4;
        const float by = TX == KV_F16 ? scale * sh.row_scale[at] : scale;
        constexpr int STEP = 16 / S::SIZE;                             // outputs of 16 bytes
        const bool full_rows = __all_sync(0xffffffffu, row >= 0);
        const uint32_t d2 = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + (uint32_t)half * 128;
        for (int i = half; i < my_tiles; i += 2) {
            const int n0 = look_up(i), left = min(S::COLS, a.width[target] - n0), n = n_target + n0, slot_i = i % plan.slots;
            char *const slot_line = tiles + plan.slot_at + slot_i * LT_SLOT + at * LT_LINE;
            wait(&sh.d2_done[half], (i >> 1) & 1);
            kvt_after();
            if (staged && a.base) wait(&sh.slot_full[slot_i], (i / plan.slots) & 1);
            const bool whole = staged && left == S::COLS;
#pragma unroll 1
            for (int m = 0; m < S::COLS; m += 32) {
                uint32_t v[32];
                __syncwarp();
                kvt_load32(d2 + m, v);
                kvt_wait_ld();
                if (m + 32 == S::COLS) {
                    kvt_before();
                    lt_arrive(&sh.d2_free[half]);
                }
                if (whole) {                                           // the same way for all rows, also those that are none
                    uint4 was[32 / STEP];
#pragma unroll
                    for (int e = 0; e < 32 / STEP; ++e) was[e] = a.base ? *(const uint4 *)(slot_line + (m + e * STEP) * S::SIZE) : make_uint4(0, 0, 0, 0);
#pragma unroll
                    for (int e = 0; e < 32 / STEP; ++e) *(uint4 *)(slot_line + (m + e * STEP) * S::SIZE) = lt_add<TX>(was[e], v + e * STEP, by);
                    continue;
                }
                if (row < 0 || m >= left) continue;
#pragma unroll
                for (int e = 0; e < 32; e += STEP) {
                    if (staged && m + e + STEP <= left) {
                        uint4 *const was = (uint4 *)(slot_line + (m + e) * S::SIZE);
                        *was = lt_add<TX>(a.base ? *was : make_uint4(0, 0, 0, 0), v + e, by);
                    } else {
                        const int64_t to = (int64_t)row * a.out_stride + n + m + e, was = (int64_t)row * a.base_stride + n + m + e;
#pragma unroll
                        for (int k = 0; k < STEP; ++k)
                            if (m + e + k < left) kv_store(a.out, to + k, TX, __fmaf_rn(by, __uint_as_float(v[e + k]), a.base ? kv_load(a.base, was + k, TX) : 0.0f));
                    }
                }
            }
            if (!staged) continue;
            __syncwarp();
            const char *const from = tiles + plan.slot_at + slot_i * LT_SLOT + (32 * (warp & 3)) * LT_LINE + cc * 16;
            char *const to = (char *)a.out + (int64_t)n * S::SIZE + cc * 16;
            if (whole && full_rows) {
#pragma unroll
                for (int k = 0; k < 32; k += 2)
                    __stcs((uint4 *)(to + (int64_t)sh.row[32 * (warp & 3) + k + cl] * a.out_stride * S::SIZE), *(const uint4 *)(from + (k + cl) * LT_LINE));
            } else if ((cc + 1) * STEP <= left)
#pragma unroll 4
                for (int k = cl; k < 32; k += 2) {
                    const int to_row = sh.row[32 * (warp & 3) + k];
                    if (to_row >= 0) __stcs((uint4 *)(to + (int64_t)to_row * a.out_stride * S::SIZE), *(const uint4 *)(from + k * LT_LINE));
                }
            __syncwarp();
            lt_arrive(&sh.slot_free[slot_i]);
        }
    }
    // What this CTA has been sent is there, also where a wait for it has run out; so what it has sent is, once every CTA has come here.
    kvt_mbar_wait(&sh.h_full, 0, NC_DRAIN_CYCLES);
    __syncwarp();
    lora_cluster_arrive();
    // Nothing reads or writes tensor memory any more once the last matrix instruction has come to its end.
    kvt_mbar_wait(&sh.drained, 0, NC_DRAIN_CYCLES);
    kvt_before();
    __syncthreads();
    kvt_after();
    if (warp == LT_MMA) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(S::TMEM) : "memory");
    lora_cluster_wait();
}

}  // namespace nc
