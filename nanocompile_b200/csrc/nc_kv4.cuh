// nc_kv4.cuh -- a paged key/value cache held in 4 bits: its layout, the append and the read.
//
// Quantisation.  Blocks of 32 values along the head dimension, each with two f16 parameters:
//   zero = f16(min), scale = f16((max - min) * f32(1/15)), both kept within +-65504,
//   code = clamp(floor((x - zero) * (1 / scale) + 1/2), 0, 15), and 0 where the scale is 0;
// the block stands for zero + scale * code: 5 bits a value.  A zero per block, not codes around
// nought, because keys have channels that sit far from it.  The parameters are rounded to f16 before
// the codes are chosen, so the codes are nearest for the values that are read back.  A NaN makes its
// block's parameters, hence the whole block, NaN; infinities are held as the largest values the block
// can hold.
//
// Layout.  A page holds `page` positions (a multiple of 16) of one layer: [kv head][tile][20 d bytes],
// a tile being 16 positions of one head: key codes (8 d bytes), key parameters (2 d), value codes
// (8 d), value parameters (2 d).  Inside a tile the codes lie as the attention's matrix instruction
// (mma m16n8k16) wants its A operand: a lane's share of a tile is one vector load, and eight codes
// become four f16 pairs with one AND each (the masks below).  Position t = 8 j + g = 8 j + 2 c + h,
// block b, VB = 2 where the number of blocks is even, else 1, lane = 4 g + c:
//   key codes    u32 word [b / VB][lane][b % VB][j], (g, j) from t: nibble i is dimension 32 b + 8 c + i
//   value codes  u32 word [b / VB][lane][b % VB][j], (c, j, half-word h) from t: nibble i is dimension
//                32 b + 4 g + i
//   parameters   u32 word [g][b][j]: scale low, zero high
// Words and half-words belong to one position each, so positions are appended without reading.
//
// Both kernels read and write each byte once; memory's floor for 4 x 2048 rows of 8 heads of 128 (bfloat16 in, 44 MB for
// the append; float32 out, 78 MB for the read) is 6.7 and 11.9 us.  The append takes 21 us, bound by instructions and the latency
// between them (one issues in 61% of the cycles): a warp makes 236 for eight values a lane, of which rounding and rotation are about 90;
// the others find the rows' sequences, pages and tiles, once in every warp, and the angles, once for every head.  The read takes
// 17 us (4.5 TB/s), bound by the latency of the same chain (10 of a warp's 20 cycles an instruction wait for loads, issue 34%).
// One row of each of 256 sequences takes 5.3 and 5.8 us: the start and the chain from a row's sequence over its page to its bytes.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "nc_common.cuh"

namespace nc {

enum KvType : int { KV_F32 = 0, KV_F16 = 1, KV_BF16 = 2 };

constexpr int KV4_TILE = 16;       // positions of a tile

// Where a sequence's rows and pages are.  Row r of the call belongs to the sequence i with
// row_start[i] <= r < row_start[i + 1] (no row_start: to sequence r) and is at position
// lengths[i] - (row_start[i + 1] - r).
struct Kv4Rows {
    const int32_t *table;          // [seqs][width]
    const int32_t *lengths;        // [seqs], after the call's rows
    const int32_t *row_start;      // [seqs + 1] or null
    unsigned long long *error;     // null, or the smallest sequence with a page outside the pool
    int64_t rows;
    int seqs, width, page, pages;
};

struct Kv4Pool {
    char *base;                    // this layer's part of the first page
    int64_t page_bytes;            // from one page to the next
    int kv, d;
};

__device__ __forceinline__ float kv_load(const void *p, int64_t i, int type) {
    if (type == KV_F32) return ((const float *)p)[i];
    if (type == KV_F16) return __half2float(((const __half *)p)[i]);
    return __bfloat162float(((const __nv_bfloat16 *)p)[i]);
}
__device__ __forceinline__ void kv_store(void *p, int64_t i, int type, float v) {
    if (type == KV_F32) ((float *)p)[i] = v;
    else if (type == KV_F16) ((__half *)p)[i] = __float2half_rn(v);
    else ((__nv_bfloat16 *)p)[i] = __float2bfloat16_rn(v);
}

// The sequence of row r: the last one whose rows start at or before r.
__device__ __forceinline__ int kv4_sequence(const Kv4Rows &a, int64_t r) {
    if (!a.row_start) return (int)r;
    int low = 0, high = a.seqs;                          // row_start[low] <= r < row_start[high]
    while (high - low > 1) {
        const int mid = (low + high) >> 1;
        if (a.row_start[mid] <= r) low = mid;
        else high = mid;
    }
    return low;
}

// The page that holds `position` of sequence i, or -1 (recorded) where the table names none.
__device__ __forceinline__ int kv4_page(const Kv4Rows &a, int i, int position) {
    const int j = position / a.page;
    const int page = j < a.width ? a.table[(int64_t)i * a.width + j] : -1;
    if (page < 0 || page >= a.pages) {
        if (a.error) atomicMin(a.error, (unsigned long long)i);
        return -1;
    }
    return page;
}

__host__ __device__ constexpr int kv4_vb(int blocks) { return blocks % 2 == 0 ? 2 : 1; }

// Word indices inside a tile's codes and parameters.
__host__ __device__ __forceinline__ int kv4_code_word(int vb, int b, int lane, int j) {
    return ((b / vb * 32 + lane) * vb + b % vb) * 2 + j;
}
__host__ __device__ __forceinline__ int kv4_param_word(int blocks, int b, int t) {
    return ((t & 7) * blocks + b) * 2 + (t >> 3);
}

// Floats in the order of their values, as unsigned numbers (of numbers: a NaN is looked for by itself).
__device__ __forceinline__ uint32_t ordered_bits(float v) {
    const uint32_t u = __float_as_uint(v);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float from_ordered_bits(uint32_t u) {
    return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}

// The smaller and the larger of two, a NaN if either is one.
__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float min_nan(float a, float b, float c) {
    float r;
    asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// Two floats to an instruction.  A packed multiplication and a packed addition after it may become one FMA (seen, with
// -fmad=false and .rn too): where both roundings count, one of the two is not packed.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

__device__ __forceinline__ uint64_t add2_rz(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rz.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// A block of 32 values in four neighbouring lanes, eight each: the lane's eight codes in a word, the block's parameters.
__device__ __forceinline__ uint32_t kv4_quantise(const float (&x)[8], uint32_t *params) {
    float low = min_nan(x[0], x[1], x[2]), high = max_nan(x[0], x[1], x[2]);
    low = min_nan(low, x[3], x[4]), high = max_nan(high, x[3], x[4]);
    low = min_nan(low, x[5], x[6]), high = max_nan(high, x[5], x[6]);
    low = min_nan(low, x[7], __shfl_xor_sync(0xffffffffu, min_nan(low, x[7]), 1));
    high = max_nan(high, x[7], __shfl_xor_sync(0xffffffffu, max_nan(high, x[7]), 1));
    low = min_nan(low, __shfl_xor_sync(0xffffffffu, low, 2));
    high = max_nan(high, __shfl_xor_sync(0xffffffffu, high, 2));
    const float limit = 65504.0f;
    const float z = min_nan(max_nan(low, -limit), limit);
    // An infinite range, or none between infinities of one sign, counts as the largest; a NaN among the values stays one.
    const float w = low != low ? low : fminf(fmul(fsub(high, low), 1.0f / 15.0f), limit);
    const __half zero = __float2half_rn(z), scale = __float2half_rn(w);
    *params = (uint32_t)__half_as_ushort(scale) | (uint32_t)__half_as_ushort(zero) << 16;
    const float s = __half2float(scale), from = __half2float(zero);
    if (!(s > 0.0f)) return 0;
    const float inv = fdiv(1.0f, s);
    const uint64_t from2 = pack2(-from, -from), inv2 = pack2(inv, inv);
    uint64_t q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 v = unpack2(mul2(add2(pack2(x[2 * i], x[2 * i + 1]), from2), inv2));
        q[i] = pack2(fadd(v.x, 0.5f), fadd(v.y, 0.5f));
    }
    // The extremes' codes bound the others': seldom (a scale that f16 rounds far, infinities) is there anything to clamp.
    if (!(fadd(fmul(fsub(low, from), inv), 0.5f) >= 0.0f && fadd(fmul(fsub(high, from), inv), 0.5f) < 16.0f)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 v = unpack2(q[i]);
            q[i] = pack2(fminf(fmaxf(v.x, 0.0f), 15.0f), fminf(fmaxf(v.y, 0.0f), 15.0f));
        }
    }
    uint32_t word = 0;
#pragma unroll
    for (int i = 3; i >= 0; --i) {
        // 2^23 + the code, rounded towards zero: floor, as it is not negative.  The code is in the low bits.
        const float2 c = unpack2(add2_rz(q[i], pack2(8388608.0f, 8388608.0f)));
        word = (word * 16 + __float_as_uint(c.y)) * 16 + __float_as_uint(c.x);
    }
    return word - 0x4b000000u * 0x11111111u;       // what the eight 2^23 have added, modulo 2^32
}

struct Kv4AppendArgs {
    Kv4Rows at;
    Kv4Pool pool;
    const void *keys, *values;     // [rows][kv][d], rows apart by the strides
    const float *cos_tab, *sin_tab;   // [positions][d / 2] or null
    int64_t key_stride, value_stride, positions;
    int type;
};

// Eight values from element `at` (of 16-byte aligned memory where `vectors`).
__device__ __forceinline__ void kv_load8(const void *p, int64_t at, int type, bool vectors, float (&x)[8]) {
    if (!vectors) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = kv_load(p, at + i, type);
    } else if (type == KV_F32) {
        const float4 a = *(const float4 *)((const float *)p + at), b = *(const float4 *)((const float *)p + at + 4);
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
        x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
        const uint4 w = *(const uint4 *)((const uint16_t *)p + at);
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (type == KV_F16) {
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

// The append of many rows and the read go by tiles: the rows of a call that fall into one tile are one piece of work (two for
// the append) for a warp and head, keys or values, with lane 4 g + c at dimensions 32 b + 8 c .. of positions g and 8 + g: for keys the
// lane's words are the ones it writes, for values two shuffles turn them.  A CTA looks through `window` rows for
// the first rows of tiles.
struct Kv4TileRows {
    char *tile;                    // of the first head, or null: no page
    int64_t row, position;         // of the first row
    int count, t0;                 // rows of the tile, its first position in the tile
    int seq;
};

// Calls work(rows) for each tile whose first row is among the CTA's window, all threads of the CTA alike.
template <typename F>
__device__ __forceinline__ void kv4_tiles(const Kv4Rows &at, const Kv4Pool &pool, int window, F work) {
    const int lane = threadIdx.x & 31;
    const int64_t first = (int64_t)blockIdx.x * window, r = first + lane;
    int seq = 0, position = -1, count = 0;
    bool starts = false;
    if (lane < window && r < at.rows) {
        seq = kv4_sequence(at, r);
        const int64_t after = at.row_start ? at.row_start[seq + 1] - r : 1;      // rows to the sequence's end
        const int64_t begin = at.row_start ? at.row_start[seq] : r;
        position = (int)(at.lengths[seq] - after);
        if (after > 0 && position < 0) {                             // before position 0: a piece of one row
            starts = true;
            count = 1;
        } else if (after > 0) {
            starts = r == begin || position % KV4_TILE == 0;
            count = (int)min(min(after, at.rows - r), (int64_t)(KV4_TILE - position % KV4_TILE));   // row_start may end past the call's rows
        } else {                                                     // belongs to no sequence
            starts = true;
            count = 1;
            position = -1;
        }
    }
    for (uint32_t left = __ballot_sync(0xffffffffu, starts); left; left &= left - 1) {
        const int k = __ffs(left) - 1;
        Kv4TileRows t;
        t.seq = __shfl_sync(0xffffffffu, seq, k);
        t.row = first + k;
        t.position = __shfl_sync(0xffffffffu, position, k);
        t.count = __shfl_sync(0xffffffffu, count, k);
        t.t0 = (int)(t.position & (KV4_TILE - 1));
        t.tile = nullptr;
        if (t.position >= 0) {
            const int page = kv4_page(at, t.seq, (int)t.position);
            if (page >= 0) t.tile = pool.base + page * pool.page_bytes + (int64_t)((int)t.position % at.page / KV4_TILE) * (20 * pool.d);
        }
        work(t);
    }
}
constexpr int KV4_TILE_WARPS = 4;

// The append of few rows, or of one to a sequence: four lanes to a block of a row, eight blocks to a warp (six of d = 96).
template <int NB>
__global__ void __launch_bounds__(32 * KV4_TILE_WARPS) kv4_append_rows_kernel(const __grid_constant__ Kv4AppendArgs a, bool vectors) {
    constexpr int D = 32 * NB, VB = kv4_vb(NB), HALF = D / 2, SHARE = NB == 3 ? 4 : NB;
    release_dependents();
    wait_for_producer();
    const int lane = threadIdx.x & 31, c = lane & 3, b = (lane >> 2) % SHARE;
    const int64_t line = ((int64_t)blockIdx.x * (32 * KV4_TILE_WARPS) + threadIdx.x) / (4 * SHARE);   // row, 2 head + (0 keys, 1 values)
    const int64_t row = line / (2 * a.pool.kv);
    const int job = (int)(line % (2 * a.pool.kv)), head = job >> 1, which = job & 1;
    char *tile = nullptr;
    int t = 0;
    float x[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    if (row < a.at.rows && b < NB) {
        const void *const p = which ? a.values : a.keys;
        const int64_t from = row * (which ? a.value_stride : a.key_stride) + (int64_t)head * D;
        const int i0 = 32 * b + 8 * c, k = i0 < HALF ? i0 : i0 - HALF;
        const bool low = i0 < HALF, rotate = which == 0 && a.cos_tab;
        float y[8];
        kv_load8(p, from + i0, a.type, vectors, x);
        if (rotate) kv_load8(p, from + (low ? i0 + HALF : k), a.type, vectors, y);
        const int seq = kv4_sequence(a.at, row);
        const int64_t position = a.at.lengths[seq] - (a.at.row_start ? a.at.row_start[seq + 1] - row : 1);
        if (position >= 0 && position < a.at.lengths[seq]) {
            const int page = kv4_page(a.at, seq, (int)position);
            if (page >= 0 && a.cos_tab && position >= a.positions) {
                if (a.at.error) atomicMin(a.at.error, (unsigned long long)seq);
            } else if (page >= 0) {
                const int place = (int)position % a.at.page;
                t = place % KV4_TILE;
                tile = a.pool.base + page * a.pool.page_bytes + ((int64_t)head * (a.at.page / KV4_TILE) + place / KV4_TILE) * (20 * D) + which * 10 * D;
                if (rotate) {                          // the reference's t * cos + rot(t) * sin (nanocompile/nn.py:97-106), every step rounded
                    float cs[8], sn[8];
                    kv_load8(a.cos_tab, position * HALF + k, KV_F32, vectors, cs);
                    kv_load8(a.sin_tab, position * HALF + k, KV_F32, vectors, sn);
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        x[i] = low ? fsub(fmul(x[i], cs[i]), fmul(y[i], sn[i])) : fadd(fmul(x[i], cs[i]), fmul(y[i], sn[i]));
                }
            }
        }
    }
    uint32_t params;
    const uint32_t word = kv4_quantise(x, &params);
    if (!tile) return;
    const int g = t & 7, j = t >> 3;
    if (which) {
#pragma unroll
        for (int half = 0; half < 2; ++half)
            ((uint16_t *)tile)[2 * kv4_code_word(VB, b, 4 * (2 * c + half) + (g >> 1), j) + (g & 1)] = (uint16_t)(word >> (16 * half));
    } else {
        ((uint32_t *)tile)[kv4_code_word(VB, b, 4 * g + c, j)] = word;
    }
    if (c == 0) ((uint32_t *)(tile + 8 * D))[kv4_param_word(NB, b, t)] = params;
}

// A warp takes the positions 8 j .. 8 j + 7 of a tile: with both halves to a warp, 4 x 2048 rows took 22 us instead of 21, 2048 rows 8.9 instead of 7.2.
template <int NB>
__global__ void __launch_bounds__(32 * KV4_TILE_WARPS, NB == 3 ? 6 : 8) kv4_append_kernel(const __grid_constant__ Kv4AppendArgs a, bool vectors) {
    constexpr int D = 32 * NB, VB = kv4_vb(NB), HALF = D / 2, window = KV4_TILE;
    release_dependents();
    wait_for_producer();
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int job = blockIdx.y * KV4_TILE_WARPS + (threadIdx.x >> 5);     // 4 head + 2 (0 keys, 1 values) + j
    const int head = job >> 2, which = job >> 1 & 1, j = job & 1;
    if (head < a.pool.kv) {                                          // the rows are on their way while their tiles are looked up
        const int size = a.type == KV_F32 ? 4 : 2, lines = (D * size + 127) / 128;
        for (int i = lane; i < window / 2 * lines; i += 32) {
            const int64_t r = (int64_t)blockIdx.x * window + i / lines * 2 + j;
            if (r < a.at.rows)
                asm volatile("prefetch.global.L2 [%0];" ::"l"((const char *)(which ? a.values : a.keys) +
                             (r * (which ? a.value_stride : a.key_stride) + (int64_t)head * D) * size + min(i % lines * 128, D * size - 1)));
        }
    }
    kv4_tiles(a.at, a.pool, window, [&](const Kv4TileRows &rows) {
        if (!rows.tile || head >= a.pool.kv) return;
        int count = rows.count;
        if (a.cos_tab && rows.position + count > a.positions) {
            if (a.at.error && lane == 0) atomicMin(a.at.error, (unsigned long long)rows.seq);
            count = (int)(a.positions - rows.position);
        }
        if (rows.t0 >= 8 * j + 8 || rows.t0 + count <= 8 * j) return;
        char *const tile = rows.tile + (int64_t)head * (a.at.page / KV4_TILE) * (20 * D) + which * 10 * D;
        const void *const p = which ? a.values : a.keys;
        const int t = 8 * j + g;
        const bool in = t >= rows.t0 && t < rows.t0 + count, rotate = which == 0 && a.cos_tab;
        const int64_t at = (rows.row + t - rows.t0) * (which ? a.value_stride : a.key_stride) + (int64_t)head * D + 8 * c;
        float x[NB][8];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            if (in) kv_load8(p, at + 32 * b, a.type, vectors, x[b]);
            else
#pragma unroll
                for (int i = 0; i < 8; ++i) x[b][i] = 0.0f;
        }
        if (rotate && in) {                                           // as row by row
            const int64_t angle = (rows.position + t - rows.t0) * HALF;
            if constexpr (NB % 2 == 0) {                              // a lane has both of a pair
#pragma unroll
                for (int b = 0; b < NB / 2; ++b) {
                    float cs[8], sn[8];
                    kv_load8(a.cos_tab, angle + 32 * b + 8 * c, KV_F32, vectors, cs);
                    kv_load8(a.sin_tab, angle + 32 * b + 8 * c, KV_F32, vectors, sn);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float u = x[b][i], v = x[b + NB / 2][i];
                        x[b][i] = fsub(fmul(u, cs[i]), fmul(v, sn[i]));
                        x[b + NB / 2][i] = fadd(fmul(v, cs[i]), fmul(u, sn[i]));
                    }
                }
            } else {
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const int i0 = 32 * b + 8 * c;
                    const bool low = i0 < HALF;
                    const int k = low ? i0 : i0 - HALF;
                    float y[8], cs[8], sn[8];
                    kv_load8(p, at - 8 * c + (low ? i0 + HALF : k), a.type, vectors, y);
                    kv_load8(a.cos_tab, angle + k, KV_F32, vectors, cs);
                    kv_load8(a.sin_tab, angle + k, KV_F32, vectors, sn);
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        x[b][i] = low ? fsub(fmul(x[b][i], cs[i]), fmul(y[i], sn[i])) : fadd(fmul(x[b][i], cs[i]), fmul(y[i], sn[i]));
                }
            }
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            uint32_t params, word = kv4_quantise(x[b], &params);
            uint32_t *const code = (uint32_t *)tile + kv4_code_word(VB, b, lane, j);
            if (which) {
                // Value words: lane 4 g' + c' takes dimension group g' of positions 2 c' and 2 c' + 1.
                const uint32_t even = __shfl_sync(0xffffffffu, word, 8 * c + (g >> 1));
                const uint32_t odd = __shfl_sync(0xffffffffu, word, 8 * c + 4 + (g >> 1));
                word = __byte_perm(even, odd, g & 1 ? 0x7632 : 0x5410);
                const int t2 = 8 * j + 2 * c;
                const bool first = t2 >= rows.t0 && t2 < rows.t0 + count, second = t2 + 1 >= rows.t0 && t2 + 1 < rows.t0 + count;
                if (first && second) *code = word;
                else if (first) ((uint16_t *)code)[0] = (uint16_t)word;
                else if (second) ((uint16_t *)code)[1] = (uint16_t)(word >> 16);
            } else if (in) {
                *code = word;
            }
            if (in && c == (b & 3)) ((uint32_t *)(tile + 8 * D))[kv4_param_word(NB, b, t)] = params;
        }
    });
}

struct Kv4ReadArgs {
    Kv4Rows at;
    Kv4Pool pool;
    float *keys, *values;          // [rows][kv][d]
};

// The values the rows' positions stand for; zeros for a row without a position.
template <int NB>
__global__ void __launch_bounds__(32 * KV4_TILE_WARPS) kv4_read_kernel(const __grid_constant__ Kv4ReadArgs a, int window, bool vectors) {
    constexpr int D = 32 * NB, VB = kv4_vb(NB);
    release_dependents();
    wait_for_producer();
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int job = blockIdx.y * KV4_TILE_WARPS + (threadIdx.x >> 5);
    const int head = job >> 1, which = job & 1;
    kv4_tiles(a.at, a.pool, window, [&](const Kv4TileRows &rows) {
        if (head >= a.pool.kv) return;
        const char *const tile = rows.tile ? rows.tile + (int64_t)head * (a.at.page / KV4_TILE) * (20 * D) + which * 10 * D : nullptr;
        float *const out = which ? a.values : a.keys;
        uint2 codes[NB], params[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            codes[b] = tile ? *(const uint2 *)((const uint32_t *)tile + kv4_code_word(VB, b, lane, 0)) : make_uint2(0, 0);
            params[b] = tile ? *(const uint2 *)((const uint32_t *)(tile + 8 * D) + kv4_param_word(NB, b, g)) : make_uint2(0, 0);
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const uint2 w = codes[b];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                uint32_t word = j ? w.y : w.x;
                if (which) {
                    // Back to lane 4 g + c: groups 2 c (low half) and 2 c + 1 of position g, half-word g & 1 of lane 4 g' + g / 2.
                    const uint32_t low = __shfl_sync(0xffffffffu, word, 8 * c + (g >> 1));
                    const uint32_t high = __shfl_sync(0xffffffffu, word, 8 * c + 4 + (g >> 1));
                    word = __byte_perm(low, high, g & 1 ? 0x7632 : 0x5410);
                }
                const int t = 8 * j + g;
                if (t < rows.t0 || t >= rows.t0 + rows.count) continue;
                const float2 sz = __half22float2(*reinterpret_cast<const __half2 *>(j ? &params[b].y : &params[b].x));
                float x[8];
#pragma unroll
                for (int i = 0; i < 8; i += 2) {             // a code times an f16 is exact, so that the FMA rounds as the sum does
                    const uint64_t code = add2(pack2(__uint_as_float(0x4b000000u | (word >> (4 * i) & 15u)), __uint_as_float(0x4b000000u | (word >> (4 * i + 4) & 15u))),
                                               pack2(-8388608.0f, -8388608.0f));
                    const float2 v = unpack2(fma2(code, pack2(sz.x, sz.x), pack2(sz.y, sz.y)));
                    x[i] = v.x;
                    x[i + 1] = v.y;
                }
                float *const to = out + ((rows.row + t - rows.t0) * a.pool.kv + head) * D + 32 * b + 8 * c;
                if (vectors) {
                    *(float4 *)to = make_float4(x[0], x[1], x[2], x[3]);
                    *(float4 *)(to + 4) = make_float4(x[4], x[5], x[6], x[7]);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) to[i] = x[i];
                }
            }
        }
    });
}

}  // namespace nc
