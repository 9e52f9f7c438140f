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
// the free pages.  It is bound by the latency of its few dependent steps, so it leaves the rest to a second kernel of
// many CTAs: the page copies, bound by memory, and the new table.  Measured: a step of 8 beams 13.5 us (both launches; the
// host takes as long), 256 sequences of 64 prompts of 4096 positions forked 24 us, of which the copies of 47 MB
// need 14.5; half of 64 sequences of 4000 gone and the rest packed (234 MB moved) 112 us, 4.2 TB/s read and written where a plain
// copy does 6.5: a CTA loads a chunk, stores it and only then looks for the next one, so that nothing of the next is on its way while
// it stores.  With one CTA for the bookkeeping that fork took 65 us, the packing 144.
#pragma once

#include <climits>

#include "nc_common.cuh"

namespace nc {

constexpr int KVP_THREADS = 1024;
constexpr int KVP_COPY_CTAS = 148 * 5, KVP_COPY_THREADS = 256;
constexpr int KVP_TABLE_CTAS = 64;             // of them also write the new table, first
constexpr int KVP_COPY_CHUNK = 16384;          // bytes of a page that a CTA copies at a time

struct KvPagesArgs {
    int32_t *new_table, *new_lengths;          // [seqs][width], [seqs]
    const int32_t *table, *lengths, *parent, *grow;   // parent, grow: null for identity, 0
    int64_t *status;                           // [4]: pages missing (-1: bad table), pages in use, pages copied, highest id + 1
    int32_t *refs, *tails, *owner;             // [pages]
    int32_t *fresh;                            // [pages]: the free pages that are taken
    int32_t *first, *need, *offset;            // [seqs]: first fresh entry, how many, where they start in `fresh`
    int32_t *list;                             // [2 * max(seqs, pages)]: (from, to), `to` by its place in `fresh` for an update
    int32_t *words;                            // [KVP_WORDS]: what the cluster's CTAs tell one another
    int seqs, width, pages, page;
};
constexpr int KVP_CLUSTER = 8;
// KVP_STATE: 0 the new table as planned, 1 the old one again.
enum KvpWord : int { KVP_BAD = 0, KVP_STATE = 1, KVP_COPIES = 2, KVP_USED = 3, KVP_LOW = 4, KVP_SUMS = 8, KVP_WORDS = KVP_SUMS + 4 * KVP_CLUSTER };
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
    // A barrier that orders global memory (release and acquire for the cluster); what another CTA wrote is read past L1.
    __device__ __forceinline__ void sync() const {
        if (size == 1) {
            __syncthreads();
        } else {
            asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
            asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        }
    }
};

// Exclusive prefix sums of two counts (packed into 64 bits: neither passes 32) over the team; *total gets their sums.
struct KvpCounts {
    int a, b;
};
__device__ __forceinline__ KvpCounts team_exclusive_sum(KvpTeam &team, int32_t *words, KvpCounts v, unsigned long long *buf, KvpCounts *total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned long long mine = (unsigned long long)(unsigned)v.b << 32 | (unsigned)v.a;
    unsigned long long x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();                            // the last call's readers are done with buf
    if (lane == 31) buf[warp] = x;
    __syncthreads();
    unsigned long long w = buf[lane];           // KVP_THREADS / 32 = 32 warps: every warp sums them for itself
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long y = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += y;
    }
    const unsigned long long before = __shfl_sync(0xffffffffu, w, warp > 0 ? warp - 1 : 0);
    unsigned long long all = __shfl_sync(0xffffffffu, w, 31), at = x - mine + (warp ? before : 0);
    if (team.size > 1) {
        unsigned long long *const sums = (unsigned long long *)(words + KVP_SUMS) + team.parity * KVP_CLUSTER;
        team.parity ^= 1;
        if (threadIdx.x == 0) sums[team.rank] = all;
        team.sync();
        all = 0;
#pragma unroll
        for (int r = 0; r < KVP_CLUSTER; ++r) {
            const unsigned long long y = __ldcg(sums + r);
            if (r < team.rank) at += y;
            all += y;
        }
    }
    *total = KvpCounts{(int)(unsigned)all, (int)(all >> 32)};
    return KvpCounts{(int)(unsigned)at, (int)(at >> 32)};
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
    for (int i = team.thread; i < a.seqs; i += team.threads)
        if (a.new_lengths) a.new_lengths[i] = a.lengths[i];
    if (team.thread == 0) {
        a.status[0] = short_of;
        a.status[1] = used;
        a.status[2] = a.status[3] = 0;
        a.words[KVP_STATE] = 1;
        a.words[KVP_COPIES] = 0;
    }
}

__global__ void __launch_bounds__(KVP_THREADS) kv_pages_update_kernel(const __grid_constant__ KvPagesArgs a) {
    __shared__ unsigned long long buf[32];
    release_dependents();
    wait_for_producer();
    KvpTeam team;
    const int lane = threadIdx.x & 31;
    for (int i = team.thread; i < a.pages; i += team.threads) {
        a.refs[i] = a.tails[i] = 0;
        a.owner[i] = INT_MAX;
    }
    if (team.thread < KVP_SUMS) a.words[team.thread] = 0;          // KVP_STATE among them
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
        KvpCounts total;
        const KvpCounts at = team_exclusive_sum(team, a.words, KvpCounts{need, copy}, buf, &total);
        if (i < a.seqs) {
            a.offset[i] = wanted + at.a;
            if (copy) {
                a.list[2 * (copied + at.b)] = source;
                a.list[2 * (copied + at.b) + 1] = wanted + at.a;
            }
        }
        wanted += total.a;
        copied += total.b;
    }
    // The free pages, lowest first, and the pages in use.
    int found = 0;
    for (int base = 0; base < a.pages; base += team.threads) {
        const int id = base + team.thread;
        const bool free = id < a.pages && __ldcg(a.refs + id) == 0;
        KvpCounts total;
        const int at = found + team_exclusive_sum(team, a.words, KvpCounts{free, 0}, buf, &total).a;
        if (free && at < wanted) a.fresh[at] = id;
        found += total.a;
    }
    if (found < wanted) {
        // The pages that the old table uses, for the caller to see.
        team.sync();
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
        KvpCounts total;
        team_exclusive_sum(team, a.words, KvpCounts{used, 0}, buf, &total);
        kvp_refuse(team, a, wanted - found, total.a);
        return;
    }
    if (team.thread == 0) {
        a.status[0] = 0;
        a.status[1] = a.pages - found + wanted;
        a.status[2] = copied;
        a.status[3] = 0;                                           // raised as the table is written
        a.words[KVP_COPIES] = copied;
    }
}

__global__ void __launch_bounds__(KVP_THREADS) kv_pages_compact_kernel(const __grid_constant__ KvPagesArgs a) {
    __shared__ unsigned long long buf[32];
    release_dependents();
    wait_for_producer();
    KvpTeam team;
    const int lane = threadIdx.x & 31;
    for (int i = team.thread; i < a.pages; i += team.threads) a.refs[i] = 0;
    if (team.thread < KVP_SUMS) a.words[team.thread] = 0;          // KVP_STATE among them
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
        KvpCounts total;
        const int live = id < a.pages && __ldcg(a.refs + id);
        const int below = used + team_exclusive_sum(team, a.words, KvpCounts{live, 0}, buf, &total).a;
        if (id < a.pages) a.owner[id] = below;
        used += total.a;
    }
    team.sync();
    // The k-th hole below `used` takes the k-th page in use from `used` on.
    const int low = used < a.pages ? __ldcg(a.owner + used) : used;
    for (int id = team.thread; id < a.pages; id += team.threads) {
        const int below = __ldcg(a.owner + id);
        const bool live = __ldcg(a.refs + id) != 0;
        if (id < used && !live) a.list[2 * (id - below) + 1] = id;
        if (id >= used && live) a.list[2 * (below - low)] = id;
    }
    if (team.thread == 0) {
        a.status[0] = 0;
        a.status[1] = a.status[3] = used;
        a.status[2] = a.words[KVP_COPIES] = used - low;
        a.words[KVP_USED] = used;
        a.words[KVP_LOW] = low;
    }
}

// The new table, by the first CTAs, and the listed pages, in chunks; no page is both read and written.
template <bool UPDATE>
__global__ void __launch_bounds__(KVP_COPY_THREADS) kv_pages_write_kernel(const __grid_constant__ KvPagesArgs a, char *pool, int64_t page_bytes) {
    release_dependents();
    wait_for_producer();
    const int lane = threadIdx.x & 31;
    if (blockIdx.x < KVP_TABLE_CTAS) {
        const bool refused = a.words[KVP_STATE] != 0;
        const unsigned chunks = (a.width + KVP_UNIT - 1) / KVP_UNIT, units = chunks * a.seqs;
        int top = 0;
        for (unsigned u = (blockIdx.x * KVP_COPY_THREADS + threadIdx.x) >> 5; u < units; u += KVP_TABLE_CTAS * KVP_COPY_THREADS / 32) {
            const int i = (int)(u / chunks), j0 = (int)(u % chunks) * KVP_UNIT;
            int first, end, offset = 0, source = i, used = 0, low = 0;      // entries before `first` are old, before `end` fresh
            if (refused) {
                first = end = a.width;
            } else if (UPDATE) {
                first = a.first[i];
                end = first + a.need[i];
                offset = a.offset[i];
                source = a.parent ? a.parent[i] : i;
            } else {
                first = end = min(a.width, pages_of(max(0, a.lengths[i]), a.page));
                used = a.words[KVP_USED];
                low = a.words[KVP_LOW];
            }
#pragma unroll
            for (int k = 0; k < KVP_UNIT / 32; ++k) {
                const int j = j0 + 32 * k + lane;
                if (j >= a.width) break;
                int id = -1;
                if (j < first) {
                    id = a.table[(int64_t)source * a.width + j];
                    if (!UPDATE && !refused && id >= used) id = a.list[2 * (a.owner[id] - low) + 1];
                } else if (j < end) {
                    id = a.fresh[offset + j - first];
                }
                a.new_table[(int64_t)i * a.width + j] = id;
                top = max(top, id + 1);
            }
        }
        if (UPDATE && !refused) {
            top = __reduce_max_sync(0xffffffffu, top);
            if (lane == 0 && top) atomicMax((long long *)a.status + 3, (long long)top);
        }
    }
    const int64_t chunks = (page_bytes + KVP_COPY_CHUNK - 1) / KVP_COPY_CHUNK;
    const int64_t items = a.words[KVP_COPIES] * chunks;
    // From the last CTA on, as the first ones have the table.
    for (int64_t item = gridDim.x - 1 - blockIdx.x; item < items; item += gridDim.x) {
        const int64_t k = item / chunks, at = item % chunks * KVP_COPY_CHUNK;
        const int64_t n = page_bytes - at < KVP_COPY_CHUNK ? page_bytes - at : KVP_COPY_CHUNK;
        const int32_t to_page = UPDATE ? a.fresh[a.list[2 * k + 1]] : a.list[2 * k + 1];
        const uint4 *const from = (const uint4 *)(pool + a.list[2 * k] * page_bytes + at);
        uint4 *const to = (uint4 *)(pool + to_page * page_bytes + at);
        if (n == KVP_COPY_CHUNK) {
            uint4 v[KVP_COPY_CHUNK / 16 / KVP_COPY_THREADS];
#pragma unroll
            for (int i = 0; i < KVP_COPY_CHUNK / 16 / KVP_COPY_THREADS; ++i) v[i] = __ldcs(from + i * KVP_COPY_THREADS + threadIdx.x);
#pragma unroll
            for (int i = 0; i < KVP_COPY_CHUNK / 16 / KVP_COPY_THREADS; ++i) __stcs(to + i * KVP_COPY_THREADS + threadIdx.x, v[i]);
        } else {
            for (int64_t i = threadIdx.x; i < n / 16; i += KVP_COPY_THREADS) to[i] = __ldcs(from + i);
        }
    }
}

}  // namespace nc
