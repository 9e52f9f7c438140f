// nc_kv4_prompt.cuh -- attention of many bfloat16 rows over a paged 4-bit cache on the tensor cores (tcgen05).
//
// What nc_kv4_attention.cuh computes, for prompts: 128 columns (row, head of the group) of one kv head to a CTA, 64
// positions at a time.  Each tile's keys and values are brought from their codes to f16 in shared memory once for all
// columns; then S = Q K^T and O += P V are tcgen05.mma kind::f16 with Q, S, P and O in tensor memory (256 columns: Q d / 2,
// S 64 with P over it, O d), accumulated in float32.
//
//   keys    zero + scale * code, with scale and zero times a power of two for each tile, that the scores get back; of blocks far from
//           nought (|zero| above 16 scales) scale * code alone, and their zeros go into S by one more instruction, as 16 more
//           dimensions: the blocks' sums of q in two f16 parts times the zeros
//   values  zero + scale * code times a power of two that only grows, O rescaled when it does: no size of value leaves the f16 range
//   p       2^(x - ref), ref a past maximum: O and the sums are rescaled only when the maximum has grown by 8
//
// Accuracy.  q, p, the decoded keys (far zeros apart) and values are each rounded once to f16's 11 bits, the keys so by 1/64 of a
// scale at most; the products on the codes round q, p and p * scale.  With far zeros in the keys a log-sum over keys N(100, 0.3) was
// off by up to 3.5e-2, now by 3.8e-4.  float32 rows, which need more, stay with the codes.
//
// Layouts.  An eight-value group of dimensions is held in the order 0 4 1 5 2 6 3 7 that a code word gives, by Q and K
// alike; the positions of a tile in the order that gives a lane eight of them for one dimension: 32 positions 16 i + 8 j +
// 2 c + h at place 8 c + 4 i + 2 j + h, by K's rows, P's columns and V alike.  K is [place][d], V [d][place], both with
// 128-byte swizzled rows.  In writing a quarter of a warp covers all eight 16-byte units, so that it meets no bank twice.
//
// Codes arrive three tiles ahead by bulk copies.  While O += P V of tile t - 1 runs, the CTA decodes the keys of t + 1; while S
// of t runs, it looks for the largest parameters of t + 2 and decodes the values of t; then softmax and the one barrier of the
// tile.  A second CTA on the SM fills what is left idle.
//
// Bound by the instruction rate: decoding takes 17 for eight values and the softmax about five a score.  Measured: 2
// sequences' last 1000 of 6001 positions, 32 heads on 8 of dimension 128, 462 us, 0.39 PFLOP/s (the matrix pipe is busy for a
// fifth of it, an instruction issues in half of the cycles); the products on the codes take 1.1 ms there.
#pragma once

#include "nc_kv4_attention.cuh"

namespace nc {

constexpr int KVT_COLS = 128, KVT_STEP = 64, KVT_THREADS = 256, KVT_TMEM = 256;

__device__ unsigned int g_prompt_fault;        // set when a copy or a matrix instruction did not come to its end within the wait limit
constexpr unsigned int KVT_FAILED = 0x10000;   // added to a group's finish counter by a CTA whose part is not there

template <int D>
struct KvtShared {
    __align__(1024) char k[2][KVT_STEP * D * 2];   // [d / 64][64 places][128 bytes]
    __align__(1024) char v[KVT_STEP * D * 2];  // [d][128 bytes]
    __align__(1024) char kz[2][KVT_STEP * 32]; // [64 places][16 f16]: the far blocks' zeros, twice, then nothing
    __align__(1024) char qz[KVT_COLS * 32];    // [128 columns][16 f16]: the blocks' sums of q in two parts, then nothing
    __align__(16) char raw[3][4 * 20 * D];
    uint64_t s_done, o_done, raw_full[3];      // mbarriers
    float row_max[2][KVT_COLS], row_sum[2][KVT_COLS], block_sum[2][2][KVT_COLS];
    int2 row[KVT_COLS];                        // row, head
    uint32_t tmem, there[4], top[4][8];                  // there: the tile's cache tiles; top: its largest key scale, |key zero|, value scale, |value zero| (bits); whether there are far blocks
    unsigned int arrived;
};

__device__ __forceinline__ uint32_t kvt_smem(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void kvt_mbar_init(uint64_t *bar) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(kvt_smem(bar)) : "memory");
}
// Whether the phase is complete, or becomes so within `limit` cycles (g_wait_cycles where the kernel can stop, NC_DRAIN_CYCLES for
// what is in flight).  No clock is read for a phase that is: with it first, 476 us instead of 454 for the largest prompt below.
__device__ __forceinline__ bool kvt_mbar_wait(uint64_t *bar, unsigned parity, long long limit) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(kvt_smem(bar)), "r"(parity)
        : "memory");
    if (done) return true;
    const long long start = clock64();
    while (clock64() - start < limit) {                                // each try sleeps up to a millisecond
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done)
            : "r"(kvt_smem(bar)), "r"(parity), "r"(1000000u)
            : "memory");
        if (done) return true;
    }
    return false;
}
// A K-major operand of 128-byte swizzled rows: eight rows are 1024 bytes.
__device__ __forceinline__ uint64_t kvt_desc(uint32_t address) {
    return (uint64_t)((address & 0x3ffff) >> 4) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// The same of 32-byte swizzled rows: eight rows are 256 bytes, and bit 4 of an address is flipped by its bit 7.
__device__ __forceinline__ uint64_t kvt_desc32(uint32_t address) {
    return (uint64_t)((address & 0x3ffff) >> 4) | (uint64_t)1 << 16 | (uint64_t)(256 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)6 << 61;
}
// D[128 x N] = A[128 x 16] B[16 x N], both in shared memory, f16 with float32 sums.
__device__ __forceinline__ void kvt_mma_shared(uint32_t d, uint64_t a, uint64_t b, int n) {
    const uint32_t kind = 1u << 4 | (uint32_t)(n >> 3) << 17 | (uint32_t)(128 >> 4) << 24;
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(kind), "r"(0u)
        : "memory");
}
// D[128 x N] (+)= A[128 x 16] B[16 x N], A in tensor memory.
__device__ __forceinline__ void kvt_mma(uint32_t d, uint32_t a, uint64_t b, int n, bool add) {
    const uint32_t kind = 1u << 4 | (uint32_t)(n >> 3) << 17 | (uint32_t)(128 >> 4) << 24;
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(kind), "r"((uint32_t)add)
        : "memory");
}
__device__ __forceinline__ void kvt_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(kvt_smem(bar)) : "memory");
}
__device__ __forceinline__ void kvt_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void kvt_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void kvt_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void kvt_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void kvt_load32(uint32_t t, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(t));
}
__device__ __forceinline__ void kvt_load16(uint32_t t, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(t));
}
__device__ __forceinline__ void kvt_store16(uint32_t t, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(t),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void kvt_store8(uint32_t t, const uint32_t *r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(t), "r"(r[0]), "r"(r[1]), "r"(r[2]),
                 "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ uint32_t fma_f16x2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
__device__ __forceinline__ uint32_t max_nan_f16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// Whether either half of `a` is above that of `b`.
__device__ __forceinline__ bool any_above_f16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("{\n\t.reg .pred p, q;\n\tsetp.gt.f16x2 p|q, %1, %2;\n\tor.pred p, p, q;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r) : "r"(a), "r"(b));
    return r != 0;
}
// A block's parameters with a zero of 0 where it is far from nought: |zero| above 16 scales, 4 more in the exponent.
__device__ __forceinline__ uint32_t kvt_near(uint32_t w) { return (w >> 16 & 0x7fffu) > (w & 0xffffu) + 0x1000u ? w & 0xffffu : w; }
__device__ __forceinline__ uint32_t add_f16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// Pairs of codes as f16: nibbles `low` of each half-word (bits 0-3), or the next ones (4-7).
__device__ __forceinline__ uint32_t codes_low(uint32_t w) { return add_f16x2((w & 0x000f000fu) | 0x64006400u, 0xe400e400u); }
__device__ __forceinline__ uint32_t codes_high(uint32_t w) { return fma_f16x2((w & 0x00f000f0u) | 0x64006400u, 0x2c002c00u, 0xd400d400u); }
// 2^e as a pair of f16, -14 <= e <= 15.
__device__ __forceinline__ uint32_t pow2_f16x2(int e) { return (uint32_t)(e + 15) << 10 | (uint32_t)(e + 15) << 26; }
// The exponent that brings |zero| + 15 scale below 2^15 (and above 2^12): parameters are multiplied by 2^-e.  By the
// exponent fields of the largest of each, both f16 bits: 15 s < 2^(es - 10), |z| < 2^(ez - 14).  A NaN counts as the largest.
__device__ __forceinline__ int kvt_exponent(uint32_t scale, uint32_t zero) {
    return max(-14, min(14, max((int)(scale >> 10) + 4, (int)(zero >> 10)) - 28));
}
__device__ __forceinline__ void store16_shared(uint32_t address, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(address), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

template <int D>
__global__ void __launch_bounds__(KVT_THREADS, 2) kv4_prompt_kernel(const __grid_constant__ Kv4AttnArgs a) {
    constexpr int NB = D / 32, VB = kv4_vb(NB);
    static_assert(D == 64 || D == 128, "two blocks of a panel to a warp");
    extern __shared__ __align__(1024) char kvt_raw[];
    KvtShared<D> &sh = *reinterpret_cast<KvtShared<D> *>(kvt_raw + ((1024 - (kvt_smem(kvt_raw) & 1023)) & 1023));
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
    const int part = warp >> 2, col = 32 * (warp & 3) + lane;          // the thread's column and half of positions or dimensions

    wait_for_producer();
    const long long limit = g_wait_cycles;
    const int split = (int)(blockIdx.x % a.splits);
    const unsigned group = blockIdx.x / a.splits;
    const unsigned histories = (unsigned)(a.at.seqs * a.pool.kv), history = group % histories;
    const int cb = a.col_blocks - 1 - (int)(group / histories);        // the rows that see most first, of all sequences and heads: 479 -> 458 us, a 1024-row prompt 65 -> 58
    const int head = (int)(history % a.pool.kv), seq = (int)(history / a.pool.kv);
    const int length = a.at.lengths[seq];
    const int row0 = a.at.row_start ? a.at.row_start[seq] : seq;
    const int nr = a.at.row_start ? a.at.row_start[seq + 1] - row0 : 1;
    if (row0 < 0 || nr <= 0 || (int64_t)row0 + nr > a.at.rows) return;
    const int cols = min(nr, a.max_rows) * a.group, col0 = cb * KVT_COLS;
    if (col0 >= cols) return;
    const int ncol = min(cols - col0, KVT_COLS);
    const int last = length - nr + (col0 + ncol - 1) / a.group;
    const int first = a.cos_tab && last >= a.positions ? -1 : min(length - nr + col0 / a.group, a.max_length - 1);   // as there
    const int end = min(last < 0 ? 0 : last + 1, a.max_length);
    const int steps = (end + KVT_STEP - 1) / KVT_STEP;
    const int active = steps <= a.chunk ? 1 : (steps + a.chunk - 1) / a.chunk;
    if (split >= active) return;
    const int step0 = split * a.chunk, step_end = min(steps, step0 + a.chunk);

    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(kvt_smem(&sh.tmem)), "n"(KVT_TMEM) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid == 0) {
        kvt_mbar_init(&sh.s_done);
        kvt_mbar_init(&sh.o_done);
        kvt_mbar_init(&sh.raw_full[0]);
        kvt_mbar_init(&sh.raw_full[1]);
        kvt_mbar_init(&sh.raw_full[2]);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (tid < 32) sh.top[tid >> 3][tid & 7] = 0;

    // Lanes 0 .. 3 of the last warp: a cache tile each.  Its page is looked up a step before its copy is started.
    const int tiles_per_page = a.at.page / KV4_TILE;
    const int32_t *const table = a.at.table + (int64_t)seq * a.at.width;
    int page_next = -1;
    auto look_up = [&](int step) {                                     // nothing here waits for what is read
        const int tile = step * 4 + lane;
        page_next = -1;
        if (lane < 4 && step < step_end && tile * KV4_TILE < end) {
            const int j = (int)((uint64_t)tile * a.page_magic >> 37);
            if (j < a.at.width) page_next = table[j];
        }
    };
    auto issue = [&](int step) {                                       // by that warp, of a tile that exists, looked up before
        const int page = page_next;
        const int tile = step * 4 + lane, buffer = (step - step0) % 3;
        const bool wanted = lane < 4 && tile * KV4_TILE < end, there = wanted && page >= 0 && page < a.at.pages;
        const uint32_t mask = __ballot_sync(0xffffffffu, there);
        if (lane == 0) {
            sh.there[(step - step0) & 3] = mask;
            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(kvt_smem(&sh.raw_full[buffer])), "r"(__popc(mask) * 20 * D) : "memory");
        }
        __syncwarp();
        if (there) {
            const int j = (int)((uint64_t)tile * a.page_magic >> 37);
            const char *const src = a.pool.base + page * a.pool.page_bytes + ((int64_t)head * tiles_per_page + (tile - j * tiles_per_page)) * (20 * D);
            asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(kvt_smem(sh.raw[buffer] + lane * 20 * D)),
                         "l"(src), "n"(20 * D), "r"(kvt_smem(&sh.raw_full[buffer]))
                         : "memory");
        } else if (wanted && a.at.error) {
            atomicMin(a.at.error, (unsigned long long)seq);
        }
    };
    // The largest parameters of a tile that is here, for its exponents; warp: cache tile warp % 4, keys or values.
    auto look = [&](int step) {
        const int buffer = (step - step0) % 3, set = (step - step0) & 3, k = warp & 3;
        const bool there = sh.there[set] >> k & 1;
        uint32_t most = 0;
        bool far = false;                                              // a block further from nought than 16 scales, hence all on one side
        if (lane < 8 * NB) {
            uint2 *const at = (uint2 *)(sh.raw[buffer] + k * 20 * D + part * 10 * D + 8 * D) + lane;
            const int t = step * KVT_STEP + 16 * k + lane / NB;
            uint2 w = there ? *at : make_uint2(0, 0);
            if (!there || t + 8 >= end) {                              // past the end: whatever was there before
                if (t >= end) w.x = 0;
                if (t + 8 >= end) w.y = 0;
                *at = w;
            }
            most = max_nan_f16x2(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu);
            far = part == 0 && any_above_f16x2(__byte_perm(w.x, w.y, 0x7632) & 0x7fff7fffu, mul_f16x2(__byte_perm(w.x, w.y, 0x5410), 0x4c004c00u));
        }
        if (__any_sync(0xffffffffu, far) && lane == 0) sh.top[set][4] = 1;
        const uint32_t s = __reduce_max_sync(0xffffffffu, most & 0xffffu), z = __reduce_max_sync(0xffffffffu, most >> 16);
        if (lane == 0) {
            atomicMax(&sh.top[set][2 * part], s);
            atomicMax(&sh.top[set][2 * part + 1], z);
        }
    };
    kvt_before();
    __syncthreads();
    kvt_after();
    release_dependents();                      // not before this CTA has its tensor memory: a dependent may hold all the rest
    int issued = min(step_end, step0 + 3);                             // tiles whose copies are started
    constexpr int COPIER = KVT_THREADS / 32 - 1;
    if (warp == COPIER) {
        for (int s = step0; s < issued; ++s) {
            look_up(s);
            issue(s);
        }
        look_up(step0 + 3);
    }
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;          // the warp's quarter of tensor memory
    const uint32_t tq = sh.tmem, ts = tq + D / 2, to = ts + KVT_STEP;

    // The queries: dimensions i and i + d / 2 for a quarter of d, rotated, brought to [2^9, 2^10), that a block's sum stays in f16's
    // range, and put into tensor memory; the blocks' sums, of what is not rounded yet, go to shared memory.
    const bool have = col < ncol;
    const int r = have ? (col0 + col) / a.group : 0;
    const int qrow = row0 + r, qhead = head * a.group + (have ? col0 + col - r * a.group : 0);
    const int qpos = have ? length - nr + r : -1;
    const bool known = qpos >= 0 && (!a.cos_tab || qpos < a.positions);
    if (qpos >= 0 && !known && a.at.error) atomicMin(a.at.error, (unsigned long long)seq);
    const int pos = known ? min(qpos, a.max_length - 1) : -1;          // the last position that the row sees
    float f;                                                           // a score's factor, but for the tile's exponent
    {
        constexpr int Q = D / 4;
        float lo[Q], hi[Q];
        const int64_t at = qrow * a.q_stride + (int64_t)qhead * D + part * Q;
        float most = 0.0f;
        bool bad = false;
#pragma unroll
        for (int i = 0; i < Q; ++i) {
            const float x = known ? kv_load(a.q, at + i, KV_BF16) : 0.0f, y = known ? kv_load(a.q, at + i + D / 2, KV_BF16) : 0.0f;
            lo[i] = x;
            hi[i] = y;
            if (known && a.cos_tab) {
                const float cs = a.cos_tab[(int64_t)qpos * (D / 2) + part * Q + i], sn = a.sin_tab[(int64_t)qpos * (D / 2) + part * Q + i];
                lo[i] = fsub(fmul(x, cs), fmul(y, sn));
                hi[i] = fadd(fmul(y, cs), fmul(x, sn));
            }
            bad = bad || !(fabsf(lo[i]) < INFINITY) || !(fabsf(hi[i]) < INFINITY);
            most = fmaxf(most, fmaxf(fabsf(lo[i]), fabsf(hi[i])));
        }
        sh.row_max[part][col] = bad ? INFINITY : most;
        if (part == 0) sh.row[col] = make_int2(qrow, qhead);
        __syncthreads();
        most = fmaxf(sh.row_max[0][col], sh.row_max[1][col]);
        const uint32_t bits = __float_as_uint(most);
        int e = 0;
        if (bits != 0 && bits < 0x7f800000u) e = 9 - ((int)(bits >> 23) - 127);
        e = e < -100 ? -100 : e > 100 ? 100 : e;
        const float by = bits >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : pow2i(e);     // an infinity or a NaN: all of the row
        f = fmul(a.scale_log2e, pow2i(-e));
        uint32_t w[Q / 2];
        auto put = [&](const float (&x)[Q], uint32_t t) {
#pragma unroll
            for (int i = 0; i < Q / 8; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k) w[4 * i + k] = pack_f16(fmul(x[8 * i + k], by), fmul(x[8 * i + k + 4], by));
            if constexpr (Q == 32) kvt_store16(t, w);
            else kvt_store8(t, w);
        };
        put(lo, tq + lanes + part * (Q / 2));
        put(hi, tq + lanes + D / 4 + part * (Q / 2));
        kvt_wait_st();
        float first_half = 0.0f, second_half = 0.0f;                   // of blocks `part` and 2 + part, or halves of blocks 0 and 1 (d = 64)
#pragma unroll
        for (int i = 0; i < Q; ++i) {
            first_half = __fmaf_rn(lo[i], by, first_half);
            second_half = __fmaf_rn(hi[i], by, second_half);
        }
        sh.block_sum[part][0][col] = first_half;
        sh.block_sum[part][1][col] = second_half;
        __syncthreads();
        if (part == 0) {
            float sums[NB];
#pragma unroll
            for (int b = 0; b < NB; ++b) sums[b] = NB == 4 ? sh.block_sum[b & 1][b >> 1][col] : sh.block_sum[0][b][col] + sh.block_sum[1][b][col];
            uint32_t z[4] = {0, 0, 0, 0};
#pragma unroll
            for (int b = 0; b < NB; b += 2) {
                z[b / 2] = pack_f16(sums[b], sums[b + 1]);
                const float2 high = unpack_f16(z[b / 2]);
                z[(NB + b) / 2] = pack_f16(sums[b] - high.x, sums[b + 1] - high.y);
            }
            const uint32_t to_row = kvt_smem(sh.qz) + col * 32, flip = col >> 2 & 1;
            store16_shared(to_row + 16 * flip, z[0], z[1], z[2], z[3]);
            store16_shared(to_row + 16 * (flip ^ 1), 0, 0, 0, 0);
        } else {
            store16_shared(kvt_smem(sh.kz[0]) + col * 32, 0, 0, 0, 0);  // both buffers' 128 rows
            store16_shared(kvt_smem(sh.kz[0]) + col * 32 + 16, 0, 0, 0, 0);
        }
    }

    float ref = -INFINITY, sum = 0.0f;                                 // of the thread's half of the positions
    int ev = -14;                                                      // the values' exponent
    uint32_t poison = 0;                                               // blocks of dimensions that a NaN reached
    // Where the thread's first key and value units go; the others differ from them in bits 4-6 and by whole rows.
    const int key_place = 32 * (warp >> 1 & 1) + 8 * (g >> 1) + 4 * (warp & 1) + (g & 1);
    const uint32_t key_unit = kvt_smem(sh.k[0]) + (NB == 4 ? part : 0) * (KVT_STEP * 128) + key_place * 128 +
                              (((4 * ((NB == 4 ? 0 : part) ^ (g & 1)) + c) ^ (key_place & 7)) << 4);
    const uint32_t zero_row = kvt_smem(sh.kz[0]) + (key_place + 2 * c) * 32 + 16 * (key_place >> 2 & 1) + (NB == 4 ? 4 * part : 0);   // of lanes c < 2
    const int value_grp = NB == 4 ? part : warp >> 1 & 1, value_block = NB == 4 ? warp & 3 : warp & 1;
    const uint32_t value_unit = kvt_smem(sh.v) + (32 * value_block + 4 * g) * 128 + (((4 * value_grp + c) ^ (4 * (g & 1))) << 4);
    // Keys of a tile that is here: cache tile warp % 4, the blocks of panel `part` (d = 64: one of the panel's two for each half
    // of the lanes).
    auto decode_keys = [&](int step) {
        const int n = step - step0, k = warp & 3, pair = NB == 4 ? part : 0;      // the lane's words of both blocks are one load
        const char *const tile = sh.raw[n % 3] + k * 20 * D;
        const uint32_t unit = pow2_f16x2(-kvt_exponent(sh.top[n & 3][0], sh.top[n & 3][1])), to_unit = key_unit + (n & 1) * (KVT_STEP * D * 2);
        const uint4 codes = *(const uint4 *)((const uint32_t *)tile + kv4_code_word(VB, 2 * pair, lane, 0));
        uint4 params = *(const uint4 *)((const uint32_t *)(tile + 8 * D) + kv4_param_word(NB, 2 * pair, g));
        if (sh.top[n & 3][4]) {                                        // far blocks' zeros go apart
            const uint4 near = make_uint4(kvt_near(params.x), kvt_near(params.y), kvt_near(params.z), kvt_near(params.w));
            if (c < 2 && (NB == 4 || part == 0)) {                     // of position 8 c + g
                const uint32_t row = zero_row + (n & 1) * (KVT_STEP * 32);
                const uint32_t z = mul_f16x2(__byte_perm(c ? params.y ^ near.y : params.x ^ near.x, c ? params.w ^ near.w : params.z ^ near.z, 0x7632), unit);
                asm volatile("st.shared.b32 [%0], %1;\n\tst.shared.b32 [%0 + %2], %1;" ::"r"(row), "r"(z), "n"(2 * NB) : "memory");
            }
            params = near;
        }
#pragma unroll
        for (int n = 0; n < NB / 2; ++n) {
            const int v2 = (NB == 4 ? n : part) ^ (g & 1);             // odd rows take the other block first
            const uint2 w = v2 ? make_uint2(codes.z, codes.w) : make_uint2(codes.x, codes.y);
            const uint2 par = v2 ? make_uint2(params.z, params.w) : make_uint2(params.x, params.y);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint32_t x = j ? w.y : w.x, p = mul_f16x2(j ? par.y : par.x, unit);
                const uint32_t s = __byte_perm(p, p, 0x1010), z = __byte_perm(p, p, 0x3232);
                store16_shared((to_unit ^ (n << 6) ^ (j << 5)) + 256 * j, fma_f16x2(codes_low(x), s, z), fma_f16x2(codes_high(x), s, z),
                               fma_f16x2(codes_low(x >> 8), s, z), fma_f16x2(codes_high(x >> 8), s, z));
            }
        }
    };
    auto issue_scores = [&](int step) {                                // by one thread
        const uint32_t keys = kvt_smem(sh.k[(step - step0) & 1]);
        const bool far = sh.top[(step - step0) & 3][4] != 0;
        if (far) kvt_mma_shared(ts, kvt_desc32(kvt_smem(sh.qz)), kvt_desc32(kvt_smem(sh.kz[(step - step0) & 1])), KVT_STEP);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) kvt_mma(ts, tq + 8 * k, kvt_desc(keys + (k >> 2) * (KVT_STEP * 128) + (k & 3) * 32), KVT_STEP, k > 0 || far);
        kvt_commit(&sh.s_done);
    };
    auto look_at = [&](int step) {
        if (step >= step_end) return true;
        const bool here = kvt_mbar_wait(&sh.raw_full[(step - step0) % 3], (unsigned)((step - step0) / 3) & 1, limit);
        if (here) look(step);
        return here;
    };
    bool ok = look_at(step0);
    ok = look_at(step0 + 1) && ok;
    int step = step0;
    bool broken = __syncthreads_or(!ok);
    const bool begun = !broken && step0 < step_end;                    // scores have been asked for
    if (begun) {
        decode_keys(step0);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        kvt_before();
        __syncthreads();
        kvt_after();
        if (tid == 0) issue_scores(step0);
    }
    for (; step < step_end && !broken; ++step) {
        const int tile_no = step - step0, set = tile_no & 3;
        const bool edge = (step + 1) * KVT_STEP > first + 1;
        const char *const raw = sh.raw[tile_no % 3];
        const uint32_t there = sh.there[set];
        const int ek = kvt_exponent(sh.top[set][0], sh.top[set][1]);
        const int ev_now = max(ev, kvt_exponent(sh.top[set][2], sh.top[set][3]));
        const bool nan = sh.top[set][2] > 0x7c00u || sh.top[set][3] > 0x7c00u;
        if (tid < 8) sh.top[(set + 3) & 3][tid] = 0;                   // of the last tile, for the look at tile step + 3
        if (step + 1 < step_end) decode_keys(step + 1);
        // O += P V of the last tile is done: the values' buffer and O are free, and S, whose place P had.  The keys have been in
        // order since the last barrier.
        ok = true;
        if (step > step0) {
            ok = kvt_mbar_wait(&sh.o_done, (unsigned)(tile_no - 1) & 1, limit);
            kvt_after();
            if (tid == 0) issue_scores(step);
        }
        ok = look_at(step + 2) && ok;
        // Values: 32 positions `grp`, block b; (d = 64: two of its four dimensions of each lane).
        {
            const int grp = value_grp, b = value_block;
            const uint32_t unit = pow2_f16x2(-ev_now);
            uint32_t s[4], z[4], w[4];                                 // by (tile, j)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const char *const tile = raw + (2 * grp + k) * 20 * D + 10 * D;
                const uint2 x = *(const uint2 *)((const uint32_t *)tile + kv4_code_word(VB, b, lane, 0));
                uint2 even = *(const uint2 *)((const uint32_t *)(tile + 8 * D) + kv4_param_word(NB, b, 2 * c));
                uint2 odd = *(const uint2 *)((const uint32_t *)(tile + 8 * D) + kv4_param_word(NB, b, 2 * c + 1));
                if (nan) {                                             // dealt with row by row
                    if (nan_params(even.x)) even.x = 0;
                    if (nan_params(even.y)) even.y = 0;
                    if (nan_params(odd.x)) odd.x = 0;
                    if (nan_params(odd.y)) odd.y = 0;
                }
                w[2 * k] = x.x;
                w[2 * k + 1] = x.y;
                s[2 * k] = mul_f16x2(__byte_perm(even.x, odd.x, 0x5410), unit);
                s[2 * k + 1] = mul_f16x2(__byte_perm(even.y, odd.y, 0x5410), unit);
                z[2 * k] = mul_f16x2(__byte_perm(even.x, odd.x, 0x7632), unit);
                z[2 * k + 1] = mul_f16x2(__byte_perm(even.y, odd.y, 0x7632), unit);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (NB == 2 && (i >> 1) != (warp >> 2)) continue;
                uint32_t v[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint32_t x = i >> 1 ? w[k] >> 8 : w[k];
                    v[k] = fma_f16x2(i & 1 ? codes_high(x) : codes_low(x), s[k], z[k]);
                }
                store16_shared((value_unit ^ (i << 4)) + 128 * i, v[0], v[1], v[2], v[3]);
            }
        }
        if (nan) {                                                     // which of the thread's rows' positions have one
            for (int n = 0; n < KVT_STEP; ++n) {
                if (step * KVT_STEP + n > pos) break;
                const uint32_t *const par = (const uint32_t *)(raw + (n >> 4) * 20 * D + 18 * D);
                for (int b = 0; b < NB; ++b)
                    if (nan_params(par[kv4_param_word(NB, b, n & 15)])) poison |= 1u << b;
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        // Softmax of the thread's 32 positions.
        ok = kvt_mbar_wait(&sh.s_done, (unsigned)tile_no & 1, limit) && ok;
        kvt_after();
        uint32_t x[32];
        kvt_load32(ts + lanes + 32 * part, x);
        kvt_wait_ld();
        const float scale = fmul(f, pow2i(ek));
        float most = -INFINITY;
        if (edge) {
#pragma unroll
            for (int n = 0; n < 32; ++n) {
                const int t = step * KVT_STEP + 32 * part + 16 * (n >> 2 & 1) + 8 * (n >> 1 & 1) + 2 * (n >> 3) + (n & 1);
                if (t > pos) x[n] = 0xff800000u;
            }
        }
        if (there != 15u) {
#pragma unroll
            for (int n = 0; n < 32; ++n)
                if (!(there >> (2 * part + (n >> 2 & 1)) & 1)) x[n] = 0xff800000u;
        }
#pragma unroll
        for (int n = 0; n < 32; ++n) most = fmaxf(most, __uint_as_float(x[n]));
        sh.row_max[part][col] = most;
        asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp & 3)) : "memory");
        most = fmul(fmaxf(most, sh.row_max[part ^ 1][col]), scale);
        // A new reference when the maximum has grown by 8, or at the first position seen; the values' exponent with it.
        const float was = ref;
        if (most > ref + 8.0f) ref = most;
        const float shrink = was == ref ? 1.0f : was == -INFINITY ? 0.0f : fast_exp2(was - ref);
        const float by = fmul(shrink, pow2i(ev - ev_now));
        if (step > step0 && __any_sync(0xffffffffu, by != 1.0f)) {
#pragma unroll 1
            for (int k = 0; k < D / 32; ++k) {                         // few at a time: the scores are in registers
                uint32_t o[16];
                kvt_load16(to + lanes + part * (D / 2) + 16 * k, o);
                kvt_wait_ld();
#pragma unroll
                for (int n = 0; n < 16; ++n) o[n] = __float_as_uint(fmul(__uint_as_float(o[n]), by));
                kvt_store16(to + lanes + part * (D / 2) + 16 * k, o);
            }
        }
        ev = ev_now;
        sum = fmul(sum, shrink);
        const float base = ref == -INFINITY ? 0.0f : ref;
        uint32_t p[16];
        uint64_t total = 0;                                            // two sums
        const uint64_t scale2 = pack2(scale, scale), base2 = pack2(-base, -base);
#pragma unroll
        for (int n = 0; n < 16; ++n) {
            const float2 u = unpack2(fma2(pack2(__uint_as_float(x[2 * n]), __uint_as_float(x[2 * n + 1])), scale2, base2));
            const float2 v = make_float2(fast_exp2(u.x), fast_exp2(u.y));
            total = add2(total, pack2(v.x, v.y));
            p[n] = pack_f16(v.x, v.y);
        }
        sum += unpack2(total).x + unpack2(total).y;
        kvt_store16(ts + lanes + 16 * part, p);
        kvt_wait_st();
        kvt_before();
        broken = __syncthreads_or(!ok);                                // the tile's codes are read, too
        kvt_after();
        if (broken) break;
        if (tid == 0) {
#pragma unroll
            for (int k = 0; k < KVT_STEP / 16; ++k)
                kvt_mma(to, ts + 8 * k, kvt_desc(kvt_smem(sh.v) + k * 32), D, step > step0 || k > 0);
            kvt_commit(&sh.o_done);
        }
        if (issued < step_end) {
            if (warp == COPIER) {
                issue(step + 3);
                look_up(step + 4);
            }
            ++issued;
        }
    }
    // Nothing is left in flight. After a wait that ran out: the copies of the last three tiles, and the scores of the tile that was not
    // finished, behind which no matrix instruction has been issued; else the last O += P V.
    for (int s = max(step0, issued - 3); broken && s < issued; ++s)
        kvt_mbar_wait(&sh.raw_full[(s - step0) % 3], (unsigned)((s - step0) / 3) & 1, NC_DRAIN_CYCLES);
    const int done = step - step0;                                     // whole tiles, whose O += P V has been issued
    if (broken && begun) kvt_mbar_wait(&sh.s_done, (unsigned)done & 1, NC_DRAIN_CYCLES);
    if (!broken && done > 0) ok = kvt_mbar_wait(&sh.o_done, (unsigned)(done - 1) & 1, NC_DRAIN_CYCLES);
    const bool failed = __syncthreads_or(!ok || broken);
    kvt_after();

    // Half of the column's dimensions to a thread.
    const bool alone = active == 1;
    float *const parts = a.part + (int64_t)group * a.splits * (KVT_COLS * (D + 2)), *const mine = alone ? nullptr : parts + (int64_t)split * (KVT_COLS * (D + 2));
    if (!failed) {
        sh.row_sum[part][col] = sum;
        __syncthreads();
        sum += sh.row_sum[part ^ 1][col];
        const float by = pow2i(ev), inv = sum == 0.0f ? 0.0f : fdiv(by, sum);
        const int64_t at = qrow * a.out_stride + (int64_t)qhead * D + part * (D / 2);
#pragma unroll
        for (int k = 0; k < D / 64; ++k) {
            uint32_t o[32];
            if (done > 0) {
                kvt_load32(to + lanes + part * (D / 2) + 32 * k, o);
                kvt_wait_ld();
            } else {
#pragma unroll
                for (int n = 0; n < 32; ++n) o[n] = 0;
            }
            if (poison >> (part * (D / 64) + k) & 1) {
#pragma unroll
                for (int n = 0; n < 32; ++n) o[n] = 0x7fc00000u;
            }
            if (have && alone) {
                __nv_bfloat16 *const out = (__nv_bfloat16 *)a.out + at + 32 * k;
                const bool none = sum == 0.0f;
                if (((uintptr_t)out & 15) == 0) {
#pragma unroll
                    for (int n = 0; n < 32; n += 8) {
                        uint32_t w[4];
#pragma unroll
                        for (int m = 0; m < 4; ++m) {
                            const __nv_bfloat162 h = __floats2bfloat162_rn(none ? 0.0f : fmul(__uint_as_float(o[n + 2 * m]), inv),
                                                                           none ? 0.0f : fmul(__uint_as_float(o[n + 2 * m + 1]), inv));
                            w[m] = *reinterpret_cast<const uint32_t *>(&h);
                        }
                        *(uint4 *)(out + n) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                } else {
#pragma unroll
                    for (int n = 0; n < 32; ++n) out[n] = __float2bfloat16_rn(none ? 0.0f : fmul(__uint_as_float(o[n]), inv));
                }
            } else if (have) {
#pragma unroll
                for (int n = 0; n < 32; n += 4)
                    *(float4 *)(mine + col * D + part * (D / 2) + 32 * k + n) =
                        make_float4(fmul(__uint_as_float(o[n]), by), fmul(__uint_as_float(o[n + 1]), by),
                                    fmul(__uint_as_float(o[n + 2]), by), fmul(__uint_as_float(o[n + 3]), by));
            }
        }
        if (have && part == 0) {
            if (alone) {
                if (a.lse) a.lse[(int64_t)qrow * a.heads + qhead] = sum == 0.0f ? -INFINITY : fmul(ref + log2f(sum), 0.6931471805599453f);
            } else {
                *(float2 *)(mine + KVT_COLS * D + 2 * col) = make_float2(sum == 0.0f ? -INFINITY : ref, sum);
            }
        }
    } else if (tid == 0) {
        g_prompt_fault = 1;
    }
    if (!alone) {                                                      // a part that is not there counts too: the last one leaves the counter at zero
        __threadfence();
        __syncthreads();
        if (tid == 0) sh.arrived = atomicAdd(a.counter + group, failed ? 1u + KVT_FAILED : 1u);
        __syncthreads();
        if ((sh.arrived & (KVT_FAILED - 1)) == (unsigned)active - 1) {
            __threadfence();
            if (tid == 0) a.counter[group] = 0;
            if (!failed && sh.arrived < KVT_FAILED) kv4_join<KVT_COLS, D>(a, parts, active, ncol, sh.row);
        }
    }
    kvt_before();
    __syncthreads();
    if (warp == 0) {
        kvt_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(sh.tmem), "n"(KVT_TMEM) : "memory");
    }
}

}  // namespace nc
