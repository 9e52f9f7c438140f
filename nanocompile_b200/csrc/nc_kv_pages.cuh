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
// The bookkeeping is one CTA, or a cluster of eight where there is much of it: warps read the live table entries
// once and count in global memory (atomics on integers, whose order does not matter), prefix sums over the cluster find
// the free pages.  It is bound by the latency of its few dependent steps.  The page copies are a second kernel over
// the list that the first one leaves, bound by memory.
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
    int32_t *words;                            // [KVP_WORDS]: what the cluster's CTAs tell one another
    int seqs, width, pages, page;
};
constexpr int KVP_CLUSTER = 8;
enum KvpWord : int { KVP_BAD = 0, KVP_HIGHEST = 1, KVP_LOW = 2, KVP_SUMS = 4, KVP_WORDS = KVP_SUMS + 2 * KVP_CLUSTER };
constexpr int KVP_UNIT = 256;                  // table entries of a sequence that a warp takes

// The kernel's threads: of one CTA or of a cluster.
struct KvpTeam {
    int rank, size;                            // CTAs
    int thread, threads;
    int parity;                                // of the prefix sums: they use two sets of words in turn
    __device__ __forceinline__ KvpTeam() {
        uint32_t r, n;
        asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
        asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(n));
        rank = (int)r;
        size = (int)n;
        thread = rank * KVP_THREADS + (int)threadIdx.x;
        threads = size * KVP_THREADS;
        parity = 0;
    }
    // A barrier that orders global memory; what another CTA wrote is read past L1.
    __device__ __forceinline__ void sync() const {
        if (size == 1) {
            __syncthreads();
        } else {
            __threadfence();
            asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
            asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        }
    }
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
// The same over the team.
__device__ __forceinline__ int team_exclusive_sum(KvpTeam &team, int32_t *words, int v, int *buf, int *total) {
    int mine = block_exclusive_sum(v, buf, total);
    if (team.size == 1) return mine;
    int32_t *const sums = words + KVP_SUMS + team.parity * KVP_CLUSTER;
    team.parity ^= 1;
    if (threadIdx.x == 0) sums[team.rank] = *total;
    team.sync();
    *total = 0;
#pragma unroll
    for (int r = 0; r < KVP_CLUSTER; ++r) {
        const int x = __ldcg(sums + r);
        if (r < team.rank) mine += x;
        *total += x;
    }
    return mine;
}

__device__ __forceinline__ int pages_of(int length, int page) { return (int)(((int64_t)length + page - 1) / page); }

struct KvPageSpan {
    int source, kept, after;                   // the parent (or -1), the positions taken over, the new length
};
__device__ __forceinline__ KvPageSpan kvp_span(const KvPagesArgs &a, int i) {
    KvPageSpan s{a.parent ? a.parent[i] : i, 0, 0};
    const int grow = a.grow ? a.grow[i] : 0;
    if (s.source < 0 || s.source >= a.seqs) {
        s.source = -1;
        return s;
    }
    const int64_t most = (int64_t)a.width * a.page;
    const int64_t before = max(0, a.lengths[s.source]);
    int64_t after = before + grow;
    after = after < 0 ? 0 : after > most ? most : after;
    s.after = (int)after;
    s.kept = (int)(before < after ? before : after);
    return s;
}

// Calls work(i, j0) for units of KVP_UNIT entries from j0 of sequence i, in each lane of the unit's warp.
template <typename F>
__device__ __forceinline__ void kvp_units(const KvpTeam &team, const KvPagesArgs &a, F work) {
    const unsigned chunks = (a.width + KVP_UNIT - 1) / KVP_UNIT, units = chunks * a.seqs;
    for (unsigned u = team.thread >> 5; u < units; u += team.threads >> 5) work((int)(u / chunks), (int)(u % chunks) * KVP_UNIT);
}

// The new table is the old one, and nothing is copied.
__device__ __forceinline__ void kvp_refuse(const KvpTeam &team, const KvPagesArgs &a, int short_of, int used) {
    const int64_t n = (int64_t)a.seqs * a.width;
    for (int64_t i = team.thread; i < n; i += team.threads) a.new_table[i] = a.table[i];
    for (int i = team.thread; i < a.seqs; i += team.threads)
        if (a.new_lengths) a.new_lengths[i] = a.lengths[i];
    if (team.thread == 0) {
        a.status[0] = short_of;
        a.status[1] = used;
        a.status[2] = a.status[3] = 0;
        *a.copies = 0;
    }
}

__global__ void __launch_bounds__(KVP_THREADS) kv_pages_update_kernel(const __grid_constant__ KvPagesArgs a) {
    __shared__ int buf[33];
    release_dependents();
    wait_for_producer();
    KvpTeam team;
    const int lane = threadIdx.x & 31;
    for (int i = team.thread; i < a.pages; i += team.threads) {
        a.refs[i] = a.tails[i] = 0;
        a.owner[i] = INT_MAX;
    }
    if (team.thread < KVP_SUMS) a.words[team.thread] = 0;
    team.sync();
    // Every reference that the new table keeps.
    kvp_units(team, a, [&](int i, int j0) {
        const KvPageSpan s = kvp_span(a, i);
        const int n = pages_of(s.kept, a.page), tail = s.kept % a.page ? n - 1 : -1;
#pragma unroll
        for (int k = 0; k < KVP_UNIT / 32; ++k) {
            const int j = j0 + 32 * k + lane;
            if (j >= n) break;
            const int id = a.table[(int64_t)s.source * a.width + j];
            if (id < 0 || id >= a.pages) {
                atomicOr(a.words + KVP_BAD, 1);
                continue;
            }
            atomicAdd(a.refs + id, 1);
            if (j == tail) {
                atomicAdd(a.tails + id, 1);
                atomicMin(a.owner + id, i);
            }
        }
    });
    team.sync();
    if (__ldcg(a.words + KVP_BAD)) {
        kvp_refuse(team, a, -1, 0);
        return;
    }
    // What each sequence needs, and where its fresh pages start.
    int wanted = 0, copied = 0;
    for (int base = 0; base < a.seqs; base += team.threads) {
        const int i = base + team.thread;
        int need = 0, copy = 0, first = 0, source = -1;
        if (i < a.seqs) {
            const KvPageSpan s = kvp_span(a, i);
            first = pages_of(s.kept, a.page);
            if (s.kept % a.page) {
                source = a.table[(int64_t)s.source * a.width + first - 1];
                if (__ldcg(a.refs + source) != __ldcg(a.tails + source) || __ldcg(a.owner + source) != i) {
                    --first;
                    copy = 1;
                }
            }
            need = pages_of(s.after, a.page) - first;
            a.first[i] = first;
            a.need[i] = need;
            a.new_lengths[i] = s.after;
        }
        int total, copies;
        const int at = team_exclusive_sum(team, a.words, need, buf, &total);
        const int place = team_exclusive_sum(team, a.words, copy, buf, &copies);
        if (i < a.seqs) {
            a.offset[i] = wanted + at;
            if (copy) {
                a.list[2 * (copied + place)] = source;
                a.list[2 * (copied + place) + 1] = wanted + at;        // becomes the page id below
            }
        }
        wanted += total;
        copied += copies;
    }
    // The free pages, lowest first, and the pages in use.
    int found = 0;
    for (int base = 0; base < a.pages; base += team.threads) {
        const int id = base + team.thread;
        const bool free = id < a.pages && __ldcg(a.refs + id) == 0;
        int total;
        const int at = found + team_exclusive_sum(team, a.words, free, buf, &total);
        if (free && at < wanted) a.fresh[at] = id;
        found += total;
    }
    const int kept = a.pages - found;
    team.sync();
    if (found < wanted) {
        // The pages that the old table uses, for the caller to see.
        for (int i = team.thread; i < a.pages; i += team.threads) a.tails[i] = 0;
        team.sync();
        int used = 0;
        kvp_units(team, a, [&](int i, int j0) {
            const int n = min(a.width, pages_of(max(0, a.lengths[i]), a.page));
            for (int j = j0 + lane; j < min(n, j0 + KVP_UNIT); j += 32) {
                const int id = a.table[(int64_t)i * a.width + j];
                if (id >= 0 && id < a.pages) used += atomicExch(a.tails + id, 1) == 0;
            }
        });
        int total;
        team_exclusive_sum(team, a.words, used, buf, &total);
        kvp_refuse(team, a, wanted - found, total);
        return;
    }
    int top = 0;
    kvp_units(team, a, [&](int i, int j0) {
        const int first = __ldcg(a.first + i), need = __ldcg(a.need + i), offset = __ldcg(a.offset + i);
        const int source = a.parent ? a.parent[i] : i;
#pragma unroll
        for (int k = 0; k < KVP_UNIT / 32; ++k) {
            const int j = j0 + 32 * k + lane;
            if (j >= a.width) break;
            int id = -1;
            if (j < first) id = a.table[(int64_t)source * a.width + j];
            else if (j - first < need) id = __ldcg(a.fresh + offset + j - first);
            a.new_table[(int64_t)i * a.width + j] = id;
            top = max(top, id + 1);
        }
    });
    for (int i = team.thread; i < copied; i += team.threads) a.list[2 * i + 1] = __ldcg(a.fresh + __ldcg(a.list + 2 * i + 1));
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0 && top) atomicMax(a.words + KVP_HIGHEST, top);
    team.sync();
    if (team.thread == 0) {
        a.status[0] = 0;
        a.status[1] = kept + wanted;
        a.status[2] = copied;
        a.status[3] = __ldcg(a.words + KVP_HIGHEST);
        *a.copies = copied;
    }
}

__global__ void __launch_bounds__(KVP_THREADS) kv_pages_compact_kernel(const __grid_constant__ KvPagesArgs a) {
    __shared__ int buf[33];
    release_dependents();
    wait_for_producer();
    KvpTeam team;
    const int lane = threadIdx.x & 31;
    for (int i = team.thread; i < a.pages; i += team.threads) a.refs[i] = 0;
    if (team.thread < KVP_SUMS) a.words[team.thread] = 0;
    team.sync();
    kvp_units(team, a, [&](int i, int j0) {
        const int n = pages_of(max(0, a.lengths[i]), a.page);
        if (n > a.width && lane == 0) atomicOr(a.words + KVP_BAD, 1);
#pragma unroll
        for (int k = 0; k < KVP_UNIT / 32; ++k) {
            const int j = j0 + 32 * k + lane;
            if (j >= min(n, a.width)) break;
            const int id = a.table[(int64_t)i * a.width + j];
            if (id < 0 || id >= a.pages) atomicOr(a.words + KVP_BAD, 1);
            else a.refs[id] = 1;
        }
    });
    team.sync();
    if (__ldcg(a.words + KVP_BAD)) {
        kvp_refuse(team, a, -1, 0);
        return;
    }
    // owner[id]: the pages in use below id.
    int used = 0;
    for (int base = 0; base < a.pages; base += team.threads) {
        const int id = base + team.thread;
        int total;
        const int below = used + team_exclusive_sum(team, a.words, id < a.pages && __ldcg(a.refs + id), buf, &total);
        if (id < a.pages) a.owner[id] = below;
        used += total;
    }
    team.sync();
    // The k-th hole below `used` takes the k-th page in use from `used` on.
    const int low = used < a.pages ? __ldcg(a.owner + used) : used, holes = used - low;
    for (int id = team.thread; id < a.pages; id += team.threads) {
        const int below = __ldcg(a.owner + id);
        const bool live = __ldcg(a.refs + id) != 0;
        if (id < used && !live) a.list[2 * (id - below) + 1] = id;
        if (id >= used && live) a.list[2 * (below - low)] = id;
    }
    team.sync();
    kvp_units(team, a, [&](int i, int j0) {
        const int n = min(a.width, pages_of(max(0, a.lengths[i]), a.page));
#pragma unroll
        for (int k = 0; k < KVP_UNIT / 32; ++k) {
            const int j = j0 + 32 * k + lane;
            if (j >= a.width) break;
            int id = -1;
            if (j < n) {
                id = a.table[(int64_t)i * a.width + j];
                if (id >= used) id = __ldcg(a.list + 2 * (__ldcg(a.owner + id) - low) + 1);
            }
            a.new_table[(int64_t)i * a.width + j] = id;
        }
    });
    if (team.thread == 0) {
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
    release_dependents();
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
