// nc_kv_pages.cuh -- the pages of a cache: forking, growing, cutting and freeing sequences, and compaction.
//
// A cache is a pool of pages and, for each of its sequences, a length and a row of the page table.
// Which pages are in use, and by how many sequences, is what the table says and nothing else: there is
// no free list and no stored count that could fall out of step with it.
//
// Update: new sequence i continues old sequence parent[i] (-1: none, the sequence is freed) with
// length n_i = clamp(length + grow[i], 0, width * page).  Its first pages are the parent's.  A page may be
// shared by any number of sequences while none of them writes to it; the last page of a sequence, where
// it is not full, is written to next and so has to be its own.  Sequence i keeps it if all sequences that
// refer to that page end in it and i is the first of them; the others, and all of them where another
// sequence reads on past it, get a copy.  Copies and further pages take the lowest free page ids, in the order
// of the new table's entries, so the result does not depend on the schedule.
// Compaction: of the n pages in use, those with ids n and above move to the free ids below n, in order.
// Both write a new table beside the old one (every entry past a sequence's pages is -1) and touch no page
// that the new table shares with the old one's other readers, so a call can be repeated.
//
// The bookkeeping is one CTA: it reads the live table entries once, counts in global memory (atomics on
// integers, whose order does not matter), and finds free pages by prefix sums.  The page copies are a second
// kernel over the list that the first one leaves, bound by memory.
#pragma once

#include <climits>

#include "nc_common.cuh"

namespace nc {

constexpr int KVP_THREADS = 1024;
constexpr int KVP_COPY_CTAS = 148 * 4, KVP_COPY_THREADS = 256;
constexpr int KVP_COPY_CHUNK = 16384;          // bytes of a page that a CTA copies at a time

struct KvPagesArgs {
    int32_t *new_table, *new_lengths;          // [seqs][width], [seqs]
    const int32_t *table, *lengths, *parent, *grow;   // parent, grow: null for identity, 0
    int64_t *status;                           // [4]: pages missing (-1: bad table), pages in use, pages copied, highest id + 1
    int32_t *refs, *tails, *owner;             // [pages]
    int32_t *fresh;                            // [pages]: the free pages that are taken
    int32_t *first, *need, *offset;            // [seqs]: first fresh entry, how many, where they start in `fresh`
    int32_t *list, *copies;                    // list [2 * max(seqs, pages)]: (from, to); copies [1]
    int seqs, width, pages, page;
};

// Exclusive prefix sum over the block's threads; *total gets the sum.  `buf`: 33 ints.
__device__ __forceinline__ int block_exclusive_sum(int v, int *buf, int *total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();                            // the last call's readers are done with buf
    if (lane == 31) buf[warp] = x;
    __syncthreads();
    if (warp == 0) {
        int w = lane < KVP_THREADS / 32 ? buf[lane] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += y;
        }
        buf[lane] = w;
    }
    __syncthreads();
    *total = buf[31];
    return x - v + (warp ? buf[warp - 1] : 0);
}

__device__ __forceinline__ int pages_of(int length, int page) { return (int)(((int64_t)length + page - 1) / page); }

struct KvPageSpan {
    int source, kept, after;                   // the parent (or -1), the positions taken over, the new length
};
__device__ __forceinline__ KvPageSpan kvp_span(const KvPagesArgs &a, int i) {
    KvPageSpan s{a.parent ? a.parent[i] : i, 0, 0};
    if (s.source < 0 || s.source >= a.seqs) {
        s.source = -1;
        return s;
    }
    const int64_t most = (int64_t)a.width * a.page;
    const int64_t before = max(0, a.lengths[s.source]);
    int64_t after = before + (a.grow ? a.grow[i] : 0);
    after = after < 0 ? 0 : after > most ? most : after;
    s.after = (int)after;
    s.kept = (int)(before < after ? before : after);
    return s;
}

// The new table is the old one, and nothing is copied.
__device__ __forceinline__ void kvp_refuse(const KvPagesArgs &a, int short_of, int used) {
    const int64_t n = (int64_t)a.seqs * a.width;
    for (int64_t i = threadIdx.x; i < n; i += KVP_THREADS) a.new_table[i] = a.table[i];
    for (int i = threadIdx.x; i < a.seqs; i += KVP_THREADS)
        if (a.new_lengths) a.new_lengths[i] = a.lengths[i];
    if (threadIdx.x == 0) {
        a.status[0] = short_of;
        a.status[1] = used;
        a.status[2] = a.status[3] = 0;
        *a.copies = 0;
    }
}

__global__ void __launch_bounds__(KVP_THREADS) kv_pages_update_kernel(const __grid_constant__ KvPagesArgs a) {
    __shared__ int buf[33], bad, highest;
    wait_for_producer();
    const int tid = threadIdx.x;
    if (tid == 0) bad = highest = 0;
    for (int i = tid; i < a.pages; i += KVP_THREADS) {
        a.refs[i] = a.tails[i] = 0;
        a.owner[i] = INT_MAX;
    }
    __syncthreads();
    // Every reference that the new table keeps.
    const int64_t entries = (int64_t)a.seqs * a.width;
    for (int64_t at = tid; at < entries; at += KVP_THREADS) {
        const int i = (int)(at / a.width), j = (int)(at % a.width);
        const KvPageSpan s = kvp_span(a, i);
        if (j >= pages_of(s.kept, a.page)) continue;
        const int id = a.table[(int64_t)s.source * a.width + j];
        if (id < 0 || id >= a.pages) {
            bad = 1;
            continue;
        }
        atomicAdd(a.refs + id, 1);
        if (s.kept % a.page && j == s.kept / a.page) {
            atomicAdd(a.tails + id, 1);
            atomicMin(a.owner + id, i);
        }
    }
    __syncthreads();
    if (bad) {
        kvp_refuse(a, -1, 0);
        return;
    }
    // What each sequence needs, and where its fresh pages start.
    int wanted = 0, copied = 0;
    for (int base = 0; base < a.seqs; base += KVP_THREADS) {
        const int i = base + tid;
        int need = 0, copy = 0;
        if (i < a.seqs) {
            const KvPageSpan s = kvp_span(a, i);
            int first = pages_of(s.kept, a.page);
            if (s.kept % a.page) {
                const int id = __ldcg(a.table + (int64_t)s.source * a.width + first - 1);
                if (__ldcg(a.refs + id) != __ldcg(a.tails + id) || __ldcg(a.owner + id) != i) {
                    --first;
                    copy = 1;
                }
            }
            need = pages_of(s.after, a.page) - first;
            a.first[i] = first;
            a.need[i] = need;
        }
        int total, copies;
        const int at = block_exclusive_sum(need, buf, &total);
        const int place = block_exclusive_sum(copy, buf, &copies);
        if (i < a.seqs) {
            a.offset[i] = wanted + at;
            if (copy) {
                const KvPageSpan s = kvp_span(a, i);
                a.list[2 * (copied + place)] = a.table[(int64_t)s.source * a.width + a.first[i]];
                a.list[2 * (copied + place) + 1] = wanted + at;        // becomes the page id below
            }
        }
        wanted += total;
        copied += copies;
    }
    // The free pages, lowest first, and the pages in use.
    int found = 0, kept = 0;
    for (int base = 0; base < a.pages; base += KVP_THREADS) {
        const int id = base + tid;
        const bool in = id < a.pages, free = in && __ldcg(a.refs + id) == 0;
        int total;
        const int at = found + block_exclusive_sum(free, buf, &total);
        if (free && at < wanted) a.fresh[at] = id;
        found += total;
        kept += min(KVP_THREADS, a.pages - base) - total;
    }
    __syncthreads();
    if (found < wanted) {
        // The pages that the old table uses, for the caller to see.
        for (int i = tid; i < a.pages; i += KVP_THREADS) a.tails[i] = 0;
        __syncthreads();
        int used = 0;
        for (int64_t at = tid; at < entries; at += KVP_THREADS) {
            const int i = (int)(at / a.width), j = (int)(at % a.width);
            const int id = a.table[at];
            if (j < pages_of(max(0, a.lengths[i]), a.page) && id >= 0 && id < a.pages) used += atomicExch(a.tails + id, 1) == 0;
        }
        int total;
        block_exclusive_sum(used, buf, &total);
        kvp_refuse(a, wanted - found, total);
        return;
    }
    int top = 0;
    for (int64_t at = tid; at < entries; at += KVP_THREADS) {
        const int i = (int)(at / a.width), j = (int)(at % a.width);
        const KvPageSpan s = kvp_span(a, i);
        const int first = __ldcg(a.first + i);
        int id = -1;
        if (j < first) id = a.table[(int64_t)s.source * a.width + j];
        else if (j - first < __ldcg(a.need + i)) id = __ldcg(a.fresh + __ldcg(a.offset + i) + j - first);
        a.new_table[at] = id;
        top = max(top, id + 1);
    }
    for (int i = tid; i < a.seqs; i += KVP_THREADS) a.new_lengths[i] = kvp_span(a, i).after;
    for (int i = tid; i < copied; i += KVP_THREADS) a.list[2 * i + 1] = __ldcg(a.fresh + __ldcg(a.list + 2 * i + 1));
    atomicMax(&highest, top);
    __syncthreads();
    if (tid == 0) {
        a.status[0] = 0;
        a.status[1] = kept + wanted;
        a.status[2] = copied;
        a.status[3] = highest;
        *a.copies = copied;
    }
}

__global__ void __launch_bounds__(KVP_THREADS) kv_pages_compact_kernel(const __grid_constant__ KvPagesArgs a) {
    __shared__ int buf[33], bad;
    wait_for_producer();
    const int tid = threadIdx.x;
    if (tid == 0) bad = 0;
    for (int i = tid; i < a.pages; i += KVP_THREADS) a.refs[i] = 0;
    __syncthreads();
    const int64_t entries = (int64_t)a.seqs * a.width;
    for (int64_t at = tid; at < entries; at += KVP_THREADS) {
        const int i = (int)(at / a.width), j = (int)(at % a.width);
        if (j >= pages_of(max(0, a.lengths[i]), a.page)) continue;
        const int id = a.table[at];
        if (id < 0 || id >= a.pages) bad = 1;
        else a.refs[id] = 1;
    }
    __syncthreads();
    if (bad) {
        kvp_refuse(a, -1, 0);
        return;
    }
    int used = 0;
    for (int base = 0; base < a.pages; base += KVP_THREADS) {
        int total;
        block_exclusive_sum(base + tid < a.pages && __ldcg(a.refs + base + tid) != 0, buf, &total);
        used += total;
    }
    // The k-th hole below `used` takes the k-th page in use from `used` on.
    int holes = 0, high = 0;
    for (int base = 0; base < a.pages; base += KVP_THREADS) {
        const int id = base + tid;
        const bool in = id < a.pages, live = in && __ldcg(a.refs + id) != 0;
        const bool hole = in && !live && id < used, move = live && id >= used;
        int total, moves;
        const int at = holes + block_exclusive_sum(hole, buf, &total);
        const int from = high + block_exclusive_sum(move, buf, &moves);
        if (hole) a.list[2 * at + 1] = id;
        if (move) {
            a.list[2 * from] = id;
            a.tails[id] = from;
        }
        holes += total;
        high += moves;
    }
    __syncthreads();
    for (int64_t at = tid; at < entries; at += KVP_THREADS) {
        const int i = (int)(at / a.width), j = (int)(at % a.width);
        int id = -1;
        if (j < pages_of(max(0, a.lengths[i]), a.page)) {
            id = a.table[at];
            if (id >= used) id = __ldcg(a.list + 2 * __ldcg(a.tails + id) + 1);
        }
        a.new_table[at] = id;
    }
    if (tid == 0) {
        a.status[0] = 0;
        a.status[1] = used;
        a.status[2] = holes;
        a.status[3] = used;
        *a.copies = holes;
    }
}

// The listed pages, in chunks; no page is both read and written.
__global__ void __launch_bounds__(KVP_COPY_THREADS) kv_pages_copy_kernel(char *pool, int64_t page_bytes, const int32_t *list,
                                                                        const int32_t *copies) {
    wait_for_producer();
    const int64_t chunks = (page_bytes + KVP_COPY_CHUNK - 1) / KVP_COPY_CHUNK;
    const int64_t items = *copies * chunks;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int64_t k = item / chunks, at = item % chunks * KVP_COPY_CHUNK;
        const int64_t n = page_bytes - at < KVP_COPY_CHUNK ? page_bytes - at : KVP_COPY_CHUNK;
        const uint4 *const from = (const uint4 *)(pool + list[2 * k] * page_bytes + at);
        uint4 *const to = (uint4 *)(pool + list[2 * k + 1] * page_bytes + at);
#pragma unroll 4
        for (int64_t i = threadIdx.x; i < n / 16; i += KVP_COPY_THREADS) to[i] = __ldcs(from + i);
    }
}

}  // namespace nc
