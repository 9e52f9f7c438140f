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

// One block by one warp, lane = dimension in the block: the lane's code; the parameters' word in all lanes.
__device__ __forceinline__ uint32_t kv4_quantise(float x, uint32_t *params) {
    const uint32_t key = ordered_bits(x);
    const float low = from_ordered_bits(__reduce_min_sync(0xffffffffu, key));
    const float high = from_ordered_bits(__reduce_max_sync(0xffffffffu, key));
    const bool nan = __any_sync(0xffffffffu, x != x);   // the extremes are found as float maxima, which pass a NaN over
    const float limit = 65504.0f;
    const float z = fminf(fmaxf(low, -limit), limit);
    const float w = fminf(fmul(fsub(high, low), 1.0f / 15.0f), limit);
    const float bad = __uint_as_float(0x7fc00000u);
    const __half zero = __float2half_rn(nan ? bad : z), scale = __float2half_rn(nan ? bad : w);
    *params = (uint32_t)__half_as_ushort(scale) | (uint32_t)__half_as_ushort(zero) << 16;
    const float s = __half2float(scale);
    if (!(s > 0.0f)) return 0;
    const float q = floorf(fadd(fmul(fsub(x, __half2float(zero)), fdiv(1.0f, s)), 0.5f));
    return (uint32_t)fminf(fmaxf(q, 0.0f), 15.0f);
}

struct Kv4AppendArgs {
    Kv4Rows at;
    Kv4Pool pool;
    const void *keys, *values;     // [rows][kv][d], rows apart by the strides
    const float *cos_tab, *sin_tab;   // [positions][d / 2] or null
    int64_t key_stride, value_stride, positions;
    int type;
};

// The value of dimension i of a head's row, rotated where there is a table: the reference's
// t * cos + rot(t) * sin (nanocompile/nn.py:97-106), each product and sum rounded by itself.
__device__ __forceinline__ float kv4_rotated(const void *p, int64_t base, int i, int d, int type, const float *cos_tab,
                                             const float *sin_tab, int64_t position) {
    const float x = kv_load(p, base + i, type);
    if (!cos_tab) return x;
    const int half = d >> 1, k = i < half ? i : i - half;
    const float y = kv_load(p, base + (i < half ? i + half : i - half), type);
    const float c = cos_tab[position * half + k], s = sin_tab[position * half + k];
    return i < half ? fsub(fmul(x, c), fmul(y, s)) : fadd(fmul(x, c), fmul(y, s));
}

// A warp per (row, kv head, block, key or value).
__global__ void __launch_bounds__(256) kv4_append_kernel(Kv4AppendArgs a) {
    wait_for_producer();
    const int lane = threadIdx.x & 31, nb = a.pool.d / 32, vb = kv4_vb(nb), d = a.pool.d;
    const int64_t item = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
    if (item >= a.at.rows * a.pool.kv * nb * 2) return;
    const int which = (int)(item & 1);
    const int b = (int)((item >> 1) % nb), head = (int)((item >> 1) / nb % a.pool.kv);
    const int64_t row = (item >> 1) / nb / a.pool.kv;
    const int seq = kv4_sequence(a.at, row);
    const int64_t after = a.at.row_start ? a.at.row_start[seq + 1] - row : 1;
    const int64_t position = a.at.lengths[seq] - after;
    if (position < 0 || after <= 0) return;
    if (a.cos_tab && position >= a.positions) {
        if (a.at.error && lane == 0) atomicMin(a.at.error, (unsigned long long)seq);
        return;
    }
    const int page = kv4_page(a.at, seq, (int)position);
    if (page < 0) return;
    float x;
    if (which == 0)
        x = kv4_rotated(a.keys, row * a.key_stride + head * d, 32 * b + lane, d, a.type, a.cos_tab, a.sin_tab, position);
    else
        x = kv_load(a.values, row * a.value_stride + head * d + 32 * b + lane, a.type);
    uint32_t params;
    const uint32_t code = kv4_quantise(x, &params);
    const int inside = (int)(position % a.at.page), t = inside & 15, g = t & 7, c = (t & 7) >> 1, j = t >> 3, h = t & 1;
    char *tile = a.pool.base + page * a.pool.page_bytes +
                 ((int64_t)head * (a.at.page / KV4_TILE) + inside / KV4_TILE) * (20 * d) + which * 10 * d;
    uint32_t v = code << (4 * (lane & (which == 0 ? 7 : 3)));
    v |= __shfl_xor_sync(0xffffffffu, v, 1);
    v |= __shfl_xor_sync(0xffffffffu, v, 2);
    if (which == 0) {
        v |= __shfl_xor_sync(0xffffffffu, v, 4);
        if ((lane & 7) == 0) ((uint32_t *)tile)[kv4_code_word(vb, b, 4 * g + (lane >> 3), j)] = v;
    } else if ((lane & 3) == 0) {
        ((uint16_t *)tile)[kv4_code_word(vb, b, 4 * (lane >> 2) + c, j) * 2 + h] = (uint16_t)v;
    }
    if (lane == 0) ((uint32_t *)(tile + 8 * d))[kv4_param_word(nb, b, t)] = params;
}

struct Kv4ReadArgs {
    Kv4Rows at;
    Kv4Pool pool;
    float *keys, *values;          // [rows][kv][d]
};

// The values the rows' positions stand for; zeros for a row without a position.  A warp per
// (row, kv head, key or value).
__global__ void __launch_bounds__(256) kv4_read_kernel(Kv4ReadArgs a) {
    wait_for_producer();
    const int lane = threadIdx.x & 31, nb = a.pool.d / 32, vb = kv4_vb(nb), d = a.pool.d;
    const int64_t item = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
    if (item >= a.at.rows * a.pool.kv * 2) return;
    const int which = (int)(item & 1), head = (int)((item >> 1) % a.pool.kv);
    const int64_t row = (item >> 1) / a.pool.kv;
    const int seq = kv4_sequence(a.at, row);
    const int64_t after = a.at.row_start ? a.at.row_start[seq + 1] - row : 1;
    const int64_t position = a.at.lengths[seq] - after;
    const int page = position >= 0 && after > 0 ? kv4_page(a.at, seq, (int)position) : -1;
    float *out = (which == 0 ? a.keys : a.values) + (row * a.pool.kv + head) * d;
    if (page < 0) {
        for (int b = 0; b < nb; ++b) out[32 * b + lane] = 0.0f;
        return;
    }
    const int inside = (int)(position % a.at.page), t = inside & 15, g = t & 7, c = (t & 7) >> 1, j = t >> 3, h = t & 1;
    const char *tile = a.pool.base + page * a.pool.page_bytes +
                       ((int64_t)head * (a.at.page / KV4_TILE) + inside / KV4_TILE) * (20 * d) + which * 10 * d;
    for (int b = 0; b < nb; ++b) {
        uint32_t code;
        if (which == 0)
            code = ((const uint32_t *)tile)[kv4_code_word(vb, b, 4 * g + (lane >> 3), j)] >> (4 * (lane & 7)) & 15u;
        else
            code = ((const uint16_t *)tile)[kv4_code_word(vb, b, 4 * (lane >> 2) + c, j) * 2 + h] >> (4 * (lane & 3)) & 15u;
        const uint32_t par = ((const uint32_t *)(tile + 8 * d))[kv4_param_word(nb, b, t)];
        const float s = __half2float(__ushort_as_half((unsigned short)(par & 0xffff)));
        const float z = __half2float(__ushort_as_half((unsigned short)(par >> 16)));
        out[32 * b + lane] = fadd(z, fmul(s, (float)code));
    }
}

}  // namespace nc
