// nc_serving.cu -- the serving entry points of include/nc_cuda.h: the paged 4-bit key/value cache
// (append, read, attention, page updates) and token log probabilities.
//
// nanocompile keeps its history as float32 arrays that a step returns and takes back
// (nanocompile/models/qwen2.py:232-271) and chooses tokens by argmax on the host
// (nanocompile/models/qwen2.py:348-368); these operators have no counterpart there.
#include "nc_api.cuh"
#include "nc_kv4_prompt.cuh"
#include "nc_kv_pages.cuh"
#include "nc_logprobs.cuh"

#include <algorithm>
#include <atomic>
#include <cstring>

using namespace nc;

namespace {

constexpr int64_t I32 = (int64_t(1) << 31) - 1;

bool misaligned(const void *p, int64_t n) { return ((uintptr_t)p & (uintptr_t)(n - 1)) != 0; }

int32_t check_type(int64_t type) {
    if (type < KV_F32 || type > KV_BF16) return fail(NC_ERR_ARGUMENT, "element type %lld: 0 float32, 1 float16, 2 bfloat16", (long long)type);
    return NC_OK;
}

// Raises a kernel's limit of shared memory, once on each device (`allowed`: a bit for each).
template <typename K>
int32_t allow_smem_once(K kernel, size_t bytes, std::atomic<uint64_t> *allowed) {
    int device = 0;
    CUDA_TRY(cudaGetDevice(&device));
    if (device < 64 && (allowed->load(std::memory_order_relaxed) >> device & 1)) return NC_OK;
    CUDA_TRY(allow_smem(kernel, bytes));
    if (device < 64) allowed->fetch_or(uint64_t(1) << device, std::memory_order_relaxed);
    return NC_OK;
}

// The sizes that append, read and attention share.
int32_t kv4_common(Kv4Rows *at, Kv4Pool *pool, void *base, const void *table, const void *lengths, const void *row_start,
                   void *error, int64_t rows, int64_t seqs, int64_t kv, int64_t d, int64_t page, int64_t pages,
                   int64_t page_bytes, int64_t offset, int64_t width) {
    if (rows < 0 || seqs < 0 || rows > I32 || seqs > I32 || kv <= 0 || kv > 32768)
        return fail(NC_ERR_ARGUMENT, "bad sizes: %lld rows, %lld sequences, %lld kv heads", (long long)rows, (long long)seqs, (long long)kv);
    if (d != 32 && d != 64 && d != 96 && d != 128)
        return fail(NC_ERR_ARGUMENT, "head dimension %lld: the 4-bit cache serves 32, 64, 96 and 128", (long long)d);
    if (page <= 0 || page % KV4_TILE || page > 1024) return fail(NC_ERR_ARGUMENT, "page size %lld: a multiple of 16 positions, 1024 at most", (long long)page);
    if (pages < 0 || pages > I32 || width < 0 || width * page > I32)
        return fail(NC_ERR_ARGUMENT, "bad cache extent: %lld pages, %lld of a sequence", (long long)pages, (long long)width);
    const int64_t layer = kv * page * d * 5 / 4;
    if (offset < 0 || offset % 16 || page_bytes % 16 || offset + layer > page_bytes || misaligned(base, 16))
        return fail(NC_ERR_ARGUMENT, "a layer takes %lld bytes of a page at a 16-byte boundary; offset %lld in pages of %lld bytes",
                    (long long)layer, (long long)offset, (long long)page_bytes);
    if (rows && !seqs) return fail(NC_ERR_ARGUMENT, "%lld rows of no sequence", (long long)rows);
    if (!row_start && rows != seqs) return fail(NC_ERR_ARGUMENT, "%lld rows of %lld sequences need row_start", (long long)rows, (long long)seqs);
    if (rows && (!base || !table || !lengths)) return fail(NC_ERR_ARGUMENT, "null pool, table or lengths");
    if (misaligned(error, 8)) return fail(NC_ERR_ARGUMENT, "the error word is not at an 8-byte boundary");
    at->table = (const int32_t *)table;
    at->lengths = (const int32_t *)lengths;
    at->row_start = (const int32_t *)row_start;
    at->error = (unsigned long long *)error;
    at->rows = rows;
    at->seqs = (int)seqs;
    at->width = (int)width;
    at->page = (int)page;
    at->pages = (int)pages;
    pool->base = (char *)base + offset;
    pool->page_bytes = page_bytes;
    pool->kv = (int)kv;
    pool->d = (int)d;
    return NC_OK;
}

// Rows that a CTA looks through for tiles: a tile's worth, or one where tiles have few.  Measured, the read of 8 heads of 128 with
// sixteen / one: 4 x 2048 rows 17 / 37 us, 1 x 1024 4.8 / 6.9, 1 x 256 3.2 / 4.6, one of each of 256 sequences 20 / 5.8.
int kv4_window(const Kv4Rows &at) { return at.row_start && at.rows >= 16 * (int64_t)at.seqs ? KV4_TILE : 1; }
dim3 kv4_tile_grid(const Kv4Rows &at, const Kv4Pool &pool, int window, int jobs) {       // jobs: warps to a tile and head
    return dim3((unsigned)((at.rows + window - 1) / window), (unsigned)((jobs * pool.kv + KV4_TILE_WARPS - 1) / KV4_TILE_WARPS));
}

// Many rows of each sequence go by tiles, the others row by row.  Measured (us, by rows / by tiles), bfloat16 keys and values of
// 8 heads of 128: one sequence's 512 rows 4.7 / 5.3, 1024 6.7 / 6.6, 2048 10.3 / 7.2, 4 of 2048 36 / 21 (96: 36 / 23), one of
// each of 256 sequences 5.3 / 12.7; of 2 heads of 64 1024 rows 3.4 / 3.9, 2048 4.1 / 4.1, 8 of 1024 7.1 / 5.6.
template <int NB>
int32_t launch_kv4_append(cudaStream_t st, const Kv4AppendArgs &a, bool vectors) {
    if (!a.at.row_start || a.at.rows < 16 * (int64_t)a.at.seqs || a.at.rows < 2048) {
        const int64_t threads = a.at.rows * 2 * a.pool.kv * 4 * (NB == 3 ? 4 : NB), cta = 32 * KV4_TILE_WARPS;
        CUDA_TRY(launch_k(kv4_append_rows_kernel<NB>, (unsigned)((threads + cta - 1) / cta), (unsigned)cta, 0, st, a, vectors));
        return check_launch("kv4_append_rows_kernel");
    }
    CUDA_TRY(launch_k(kv4_append_kernel<NB>, kv4_tile_grid(a.at, a.pool, KV4_TILE, 4), 32 * KV4_TILE_WARPS, 0, st, a, vectors));
    return check_launch("kv4_append_kernel");
}

float bits_to_f32(int64_t bits) {
    const uint32_t u = (uint32_t)bits;
    float f;
    std::memcpy(&f, &u, 4);
    return f;
}

// Ways to cut that the plans weigh: every call makes its plan, so there are few of them.
constexpr int CUTS[] = {1, 2, 3, 4, 5, 6, 7, 8, 10, 12, 14, 16, 20, 24, 28, 32, 40, 48, 56, 64, 80, 96, 112, 128, 160, 192, 224, 256};

// How a call's work is cut: 8 nt columns and `chunk` steps of positions to a CTA.
struct AttnPlan {
    int nt, warps, col_blocks, splits, chunk;
    int64_t groups;
};
constexpr int64_t KV4_COUNTERS = 4096;         // groups that can be split: their finish counters lead the scratch
constexpr int64_t KV4_PARTS = 1 << 17;         // columns of all parts of a split call at most: bounds the scratch of every smaller call
constexpr int64_t KV4_SPLITS = 64, KVT_PLACES = 148 * 2;
constexpr int KV4_STAGES = 2;
// bfloat16 rows of this many columns of a sequence and more may go to the tensor cores' kernel: half of its 128 are idle then.
constexpr int64_t KV4_PROMPT_COLS = 64;

// Its splits, and what they take by a model of the measured times, in us: the start with the queries, a chunk of tiles (128 columns by
// 64 positions) in a CTA that has an SM to itself or shares it, more of both in rounds of CTAs, the join of split histories.  The call
// goes there where this is less than what the products on the codes take by their model.  Both timed for 546 calls (1 to 128
// sequences, 1 to 2,000 rows, histories to 16,000, fourteen layouts of heads; 250 of them drawn after the model was fitted), the choice
// costs 1% against the better of the two in the mean, 40% at most (16 heads of 64, 2 sequences of 256 rows over 756: 43 us, 31 by
// the codes).  In us, there and by the codes: 14 heads on 2 of 64, 4 sequences of 480 rows 27 and 61, one of 1024 38 and 47; 32 on 8 of
// 128, 480 rows 31 and 53, 128 rows over 3128 59 (in four splits; 108 whole, 99 in ten) and 94; 128 rows alone 20 and 14.
struct PromptPlan {
    int splits, chunk;
    float cost;
};
PromptPlan kv4_prompt_plan(int64_t groups, int64_t group, int64_t d, int64_t max_rows, int64_t max_length) {
    const bool wide = d == 128;
    const float start = wide ? 16.0f : 10.5f, alone = wide ? 1.8f : 1.7f, shared = wide ? 2.8f : 2.7f, round = wide ? 30.0f : 20.0f;
    const float join = wide ? 19.0f : 9.0f, part = wide ? 1.7f : 0.6f;
    const int64_t steps = std::max<int64_t>(1, (max_length + KVT_STEP - 1) / KVT_STEP);
    const int64_t block_rows = std::min(max_rows, std::max<int64_t>(1, KVT_COLS / group));       // the first block's last row sees `first` tiles
    const int64_t first = std::max<int64_t>(1, (max_length - max_rows + block_rows + KVT_STEP - 1) / KVT_STEP);
    const float mean = 0.5f * (float)(std::min(first, steps) + steps);
    PromptPlan best{};
    for (int splits : CUTS) {
        if (splits > 1 && (splits > std::min(KV4_SPLITS, steps) || groups * splits > KVT_PLACES)) break;
        const int64_t chunk = (steps + splits - 1) / splits;
        if ((steps + chunk - 1) / chunk != splits) continue;            // as good as fewer
        const float ctas = (float)groups * (splits == 1 ? 1.0f : std::min((float)splits, mean / (float)chunk + 0.5f));
        float cost = start + (splits > 1 ? join + part * (float)splits : 0.0f);
        if (ctas <= (float)KVT_PLACES) cost += (ctas <= (float)(KVT_PLACES / 2) ? alone : shared) * (float)chunk;
        else cost += shared * (float)groups * mean / (float)KVT_PLACES + 1.2f * (float)chunk + round * (ctas / (float)KVT_PLACES - 1.0f);
        if (best.splits == 0 || cost < best.cost) best = PromptPlan{splits, (int)chunk, cost};
    }
    return best;
}

// Columns and warps of a CTA, and splits of the histories: the cheapest by a model of the measured times, in units of a step on
// an SM that is full (3.3 us; 16 warps of 8 columns fill it, or 8 of 16, which share the codes' way to operands): a CTA
// starts in about half a step, the join of splits takes another half in every round, wide CTAs lose a little to their
// barriers.  Few rounds of CTAs count as whole ones, as equal histories take them; for long histories the last CTA's half
// counts instead, as lengths differ, and for prompts the mean over their rows.  Measured: 64 sequences of 2048 positions and
// two heads 12.3 us in 128 CTAs of 16 warps, 14.9 in 512 of four; 128 sequences of 512 8.5 us in 256 CTAs of eight, 11.3 of
// four, 12.0 of sixteen; 32 of 2048 and 16 heads 33 us in 512 of four, 45 of sixteen; a float32 prompt of 512 rows of 7 heads a
// key head 17.8 us by 8 columns and four warps, 23 of eight, 21 by 16 columns and four; of 1024 rows 41.6 by 8, 44.7 by 16;
// bfloat16, 8 sequences of 16 rows of 4 heads over 2000 41 us by 16, 48 by 8.
AttnPlan kv4_plan(int64_t seqs, int64_t heads, int64_t kv, int64_t d, int64_t max_rows, int64_t max_length, bool bf16) {
    AttnPlan p{};
    const int64_t cols = heads / kv * max_rows;
    const int64_t step = kv4_step_tiles((int)d) * KV4_TILE, steps = std::max<int64_t>(1, (max_length + step - 1) / step);
    const int64_t first = std::max<int64_t>(1, (max_length - max_rows + step) / step);       // of the first row
    float best = 0.0f;
    for (int nt = 1; nt <= (cols <= 8 ? 1 : 2); ++nt) {
        const int64_t col_blocks = (cols + 8 * nt - 1) / (8 * nt), groups = seqs * kv * col_blocks;
        const int64_t most = groups > KV4_COUNTERS ? 1 : std::min({KV4_SPLITS, steps, std::max<int64_t>(1, KV4_PARTS / (groups * 8 * nt))});
        for (int warps = nt == 1 ? 16 : 8; warps >= 4; warps /= 2) {
            const int64_t places = 148 * (nt == 1 ? 16 : 8) / warps;
            for (int splits : CUTS) {
                if (splits > most) break;
                const int64_t chunk = (steps + splits - 1) / splits, active = (steps + chunk - 1) / chunk;
                if (active != splits) continue;                          // as good as fewer
                const int64_t mine = (chunk + warps - 1) / warps;        // steps of a warp
                const float rounds = (float)(groups * active) / (float)places, whole = (float)((groups * active + places - 1) / places);
                const bool few = whole * (float)mine <= 16.0f, grows = steps - first >= warps && rounds > 1.0f;
                const float turns = rounds > 1.0f ? rounds : 1.0f;
                float mean = (float)mine;                                // of a warp's steps, over a prompt's rows
                if (grows) {
                    mean = 0.0f;
                    for (int i = 1; i < 8; i += 2) {
                        const int64_t sees = first + (steps - first) * i / 8, rest = sees % chunk;
                        mean += 0.25f / (float)active * (float)(sees / chunk * mine + (rest + warps - 1) / warps);
                    }
                }
                float work = few && !grows ? whole * (float)mine : turns * mean + 0.5f * (float)mine;
                if (nt > 1) work *= 0.98f;
                const float start = 0.25f + 0.125f * (float)(4 * nt) / (float)warps;   // the more queries a warp has to bring
                const float cost = work * (1.0f + (few ? 0.0025f : 0.01f) * (float)warps) + start * (grows ? turns + 0.5f : whole) +
                                   (active > 1 ? (0.5f + 0.015f * (float)active) * turns : 0.0f);
                if (p.warps == 0 || cost < best) {
                    best = cost;
                    p.nt = nt;
                    p.col_blocks = (int)col_blocks;
                    p.groups = groups;
                    p.warps = warps;
                    p.chunk = (int)chunk;
                    p.splits = (int)active;
                }
                if (groups * splits > 16 * places) break;
            }
        }
    }
    if (bf16 && (d == 64 || d == 128) && cols >= KV4_PROMPT_COLS) {
        const int64_t blocks = (cols + KVT_COLS - 1) / KVT_COLS, groups = seqs * kv * blocks;
        const PromptPlan t = kv4_prompt_plan(groups, heads / kv, d, max_rows, max_length);
        if (t.cost < (p.nt == 1 ? 3.7f + 4.2f * best : 6.8f + 2.6f * best)) {     // the model's units as us, fitted to the same calls
            p.nt = KVT_COLS / 8;                                         // 128 columns, two CTAs to an SM
            p.col_blocks = (int)blocks;
            p.groups = groups;
            p.splits = t.splits;
            p.chunk = t.chunk;
        }
    }
    return p;
}

int64_t kv4_scratch(const AttnPlan &p, int64_t d) {
    return p.splits == 1 ? 256 : 4 * KV4_COUNTERS + p.groups * p.splits * 8 * p.nt * (d + 2) * 4;
}

template <int D, int NT, bool HL, int W>
int32_t launch_kv4_attention_t(cudaStream_t st, const Kv4AttnArgs &a, int64_t ctas) {
    using S = Kv4AttnShape<D, NT, HL, W, KV4_STAGES>;
    auto kernel = kv4_attention_kernel<D, NT, HL, W, KV4_STAGES>;
    static std::atomic<uint64_t> allowed{0};
    NC_TRY(allow_smem_once(kernel, S::SMEM, &allowed));
    CUDA_TRY(launch_k(kernel, (unsigned)ctas, 32 * W, S::SMEM, st, a));
    return check_launch("kv4_attention_kernel");
}

template <int D, bool HL>
int32_t launch_kv4_attention_n(cudaStream_t st, const Kv4AttnArgs &a, const AttnPlan &p, int64_t ctas) {
    if (p.nt == 1) {
        if (p.warps == 4) return launch_kv4_attention_t<D, 1, HL, 4>(st, a, ctas);
        if (p.warps == 8) return launch_kv4_attention_t<D, 1, HL, 8>(st, a, ctas);
        return launch_kv4_attention_t<D, 1, HL, 16>(st, a, ctas);
    }
    return p.warps == 4 ? launch_kv4_attention_t<D, 2, HL, 4>(st, a, ctas) : launch_kv4_attention_t<D, 2, HL, 8>(st, a, ctas);
}

template <int D>
int32_t launch_kv4_prompt(cudaStream_t st, const Kv4AttnArgs &a, int64_t ctas) {
    constexpr size_t bytes = sizeof(KvtShared<D>) + 1024;
    static std::atomic<uint64_t> allowed{0};
    NC_TRY(allow_smem_once(kv4_prompt_kernel<D>, bytes, &allowed));
    CUDA_TRY(launch_k(kv4_prompt_kernel<D>, (unsigned)ctas, KVT_THREADS, bytes, st, a));
    return check_launch("kv4_prompt_kernel");
}

template <int D>
int32_t launch_kv4_attention_d(cudaStream_t st, const Kv4AttnArgs &a, const AttnPlan &p, int64_t ctas) {
    if constexpr (D == 64 || D == 128)
        if (p.nt == KVT_COLS / 8) return launch_kv4_prompt<D>(st, a, ctas);
    return a.type != KV_BF16 ? launch_kv4_attention_n<D, true>(st, a, p, ctas) : launch_kv4_attention_n<D, false>(st, a, p, ctas);
}

}  // namespace

int32_t nc::set_prompt_wait_limit(long long cycles) {
    CUDA_TRY(cudaMemcpyToSymbol(g_wait_cycles, &cycles, sizeof(cycles)));
    return NC_OK;
}

// Whether a wait has run out since the last call; clears it.
int32_t nc::prompt_fault(bool *fault) {
    unsigned int word = 0;
    CUDA_TRY(cudaMemcpyFromSymbol(&word, g_prompt_fault, sizeof(word)));
    *fault = word != 0;
    word = 0;
    if (*fault) CUDA_TRY(cudaMemcpyToSymbol(g_prompt_fault, &word, sizeof(word)));
    return NC_OK;
}

extern "C" int32_t nc_kv4_append(void **p, const int64_t *s, void *stream) {
    Kv4AppendArgs a{};
    NC_TRY(kv4_common(&a.at, &a.pool, p[0], p[3], p[4], p[5], p[8], s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], s[8]));
    NC_TRY(check_type(s[11]));
    if (a.at.rows == 0) return NC_OK;
    a.keys = p[1];
    a.values = p[2];
    a.cos_tab = (const float *)p[6];
    a.sin_tab = (const float *)p[7];
    a.key_stride = s[9];
    a.value_stride = s[10];
    a.type = (int)s[11];
    a.positions = s[12];
    const int64_t line = (int64_t)a.pool.kv * a.pool.d;
    if (!a.keys || !a.values || !a.cos_tab != !a.sin_tab) return fail(NC_ERR_ARGUMENT, "null keys or values, or half a rotation table");
    if (a.key_stride < line || a.value_stride < line) return fail(NC_ERR_ARGUMENT, "rows of %lld values overlap", (long long)line);
    const int64_t bytes = a.type == KV_F32 ? 4 : 2;
    const bool vectors = !misaligned(a.keys, 16) && !misaligned(a.values, 16) && a.key_stride * bytes % 16 == 0 &&
                         a.value_stride * bytes % 16 == 0 && !misaligned(a.cos_tab, 16) && !misaligned(a.sin_tab, 16);
    const cudaStream_t st = (cudaStream_t)stream;
    switch (a.pool.d) {
        case 32: return launch_kv4_append<1>(st, a, vectors);
        case 64: return launch_kv4_append<2>(st, a, vectors);
        case 96: return launch_kv4_append<3>(st, a, vectors);
        default: return launch_kv4_append<4>(st, a, vectors);
    }
}

extern "C" int32_t nc_kv4_read(void **p, const int64_t *s, void *stream) {
    Kv4ReadArgs a{};
    NC_TRY(kv4_common(&a.at, &a.pool, p[2], p[3], p[4], p[5], p[6], s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], s[8]));
    if (a.at.rows == 0) return NC_OK;
    a.keys = (float *)p[0];
    a.values = (float *)p[1];
    if (!a.keys || !a.values) return fail(NC_ERR_ARGUMENT, "null keys or values");
    const bool vectors = !misaligned(a.keys, 16) && !misaligned(a.values, 16);
    const int window = kv4_window(a.at);
    const dim3 grid = kv4_tile_grid(a.at, a.pool, window, 2);
    const cudaStream_t st = (cudaStream_t)stream;
    switch (a.pool.d) {
        case 32: CUDA_TRY(launch_k(kv4_read_kernel<1>, grid, 32 * KV4_TILE_WARPS, 0, st, a, window, vectors)); break;
        case 64: CUDA_TRY(launch_k(kv4_read_kernel<2>, grid, 32 * KV4_TILE_WARPS, 0, st, a, window, vectors)); break;
        case 96: CUDA_TRY(launch_k(kv4_read_kernel<3>, grid, 32 * KV4_TILE_WARPS, 0, st, a, window, vectors)); break;
        default: CUDA_TRY(launch_k(kv4_read_kernel<4>, grid, 32 * KV4_TILE_WARPS, 0, st, a, window, vectors)); break;
    }
    return check_launch("kv4_read_kernel");
}

extern "C" int64_t nc_kv4_attention_scratch_bytes(int64_t seqs, int64_t heads, int64_t kv_heads, int64_t d, int64_t max_rows,
                                                  int64_t max_length) {
    if (seqs <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || d <= 0 || max_rows <= 0 || max_length < 0) return 256;
    // Not what the plan for these sizes needs, which may be nothing where one for fewer sequences or rows has splits, but a bound
    // that grows with each of them: the columns of all groups times the most splits, within what the plans keep to.
    const int64_t cols = heads / kv_heads * std::min(max_rows, I32), histories = std::min(KV4_PARTS, std::min(seqs, I32) * std::min(kv_heads, KV4_PARTS));
    auto padded = [&](int64_t n) { return std::min(KV4_PARTS, (cols + n - 1) / n * n); };
    const int64_t step = kv4_step_tiles((int)d) * KV4_TILE, splits = std::min(KV4_SPLITS, (max_length + step - 1) / step);
    int64_t most = 0;
    if (splits > 1) most = std::min(KV4_PARTS, histories * padded(cols <= 8 ? 8 : 16) * splits);
    if (const int64_t prompt = std::min(KV4_SPLITS, (max_length + KVT_STEP - 1) / KVT_STEP); prompt > 1 && cols >= KV4_PROMPT_COLS)
        most = std::max(most, std::min(KVT_PLACES * KVT_COLS, histories * padded(KVT_COLS) * prompt));
    return most == 0 ? 256 : 4 * KV4_COUNTERS + most * (d + 2) * 4;
}

extern "C" int32_t nc_kv4_attention(void **p, const int64_t *s, void *stream) {
    Kv4AttnArgs a{};
    NC_TRY(kv4_common(&a.at, &a.pool, p[2], p[3], p[4], p[5], p[10], s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], s[8]));
    NC_TRY(check_type(s[12]));
    const int64_t heads = s[9], max_length = s[16], scratch = s[17];
    int64_t max_rows = s[15];
    if (heads <= 0 || heads % a.pool.kv) return fail(NC_ERR_ARGUMENT, "%lld query heads do not share %d KV heads evenly", (long long)heads, a.pool.kv);
    if (a.at.rows == 0) return NC_OK;
    a.out = p[0];
    a.q = p[1];
    a.cos_tab = (const float *)p[6];
    a.sin_tab = (const float *)p[7];
    a.lse = (float *)p[8];
    a.q_stride = s[10];
    a.out_stride = s[11];
    a.type = (int)s[12];
    a.positions = s[13];
    const float scale = bits_to_f32(s[14]);
    if (!(scale > 0.0f) || scale > 1e30f) return fail(NC_ERR_ARGUMENT, "a score scale of %g: positive", scale);
    a.scale_log2e = scale * 1.4426950408889634f;
    const uint64_t tiles = (uint64_t)a.at.page / KV4_TILE;
    a.page_magic = ((uint64_t(1) << 37) + tiles - 1) / tiles;
    a.heads = (int)heads;
    a.group = (int)(heads / a.pool.kv);
    if (!a.out || !a.q || !a.cos_tab != !a.sin_tab) return fail(NC_ERR_ARGUMENT, "null output or queries, or half a rotation table");
    if (a.q_stride < heads * a.pool.d || a.out_stride < heads * a.pool.d) return fail(NC_ERR_ARGUMENT, "rows of %lld values overlap", (long long)(heads * a.pool.d));
    if (max_rows <= 0 || max_length < 0 || max_length > I32 || (!a.at.row_start && max_rows != 1))
        return fail(NC_ERR_ARGUMENT, "at most %lld rows and %lld positions of a sequence", (long long)max_rows, (long long)max_length);
    max_rows = std::min(max_rows, a.at.rows);
    const AttnPlan plan = kv4_plan(a.at.seqs, heads, a.pool.kv, a.pool.d, max_rows, max_length, a.type == KV_BF16);
    a.col_blocks = plan.col_blocks;
    a.splits = plan.splits;
    a.chunk = plan.chunk;
    a.max_rows = (int)max_rows;
    a.max_length = (int)max_length;
    if (plan.splits > 1) {
        if (!p[9] || misaligned(p[9], 16) || scratch < kv4_scratch(plan, a.pool.d))
            return fail(NC_ERR_ARGUMENT, "scratch of %lld bytes, %lld needed", (long long)scratch, (long long)kv4_scratch(plan, a.pool.d));
        a.counter = (unsigned int *)p[9];
        a.part = (float *)((char *)p[9] + 4 * KV4_COUNTERS);
    }
    const int64_t ctas = plan.groups * plan.splits;
    if (ctas > I32 || a.at.rows * a.group > I32) return fail(NC_ERR_ARGUMENT, "%lld rows in one call", (long long)a.at.rows);
    const cudaStream_t st = (cudaStream_t)stream;
    switch (a.pool.d) {
        case 32: return launch_kv4_attention_d<32>(st, a, plan, ctas);
        case 64: return launch_kv4_attention_d<64>(st, a, plan, ctas);
        case 96: return launch_kv4_attention_d<96>(st, a, plan, ctas);
        default: return launch_kv4_attention_d<128>(st, a, plan, ctas);
    }
}

// ---- pages --------------------------------------------------------------------------------------

namespace {

// refs, tails, owner and fresh by page; first, need, offset by sequence; the copy list; its length.
int64_t kvp_list(int64_t seqs, int64_t pages) { return 2 * std::max(seqs, pages); }

int32_t kvp_args(KvPagesArgs *a, void **p, const int64_t *s, int table, int status, int scratch) {
    const int64_t seqs = s[0], width = s[1], pages = s[2], page = s[3], page_bytes = s[4];
    if (seqs < 0 || width < 0 || pages < 0 || page <= 0 || seqs > I32 || pages > I32 / 2 || width * page > I32 || seqs * width > I32)
        return fail(NC_ERR_ARGUMENT, "bad cache extent: %lld sequences of %lld pages of %lld positions, %lld pages", (long long)seqs,
                    (long long)width, (long long)page, (long long)pages);
    if (page_bytes <= 0 || page_bytes % 16 || misaligned(p[5], 16)) return fail(NC_ERR_ARGUMENT, "pages of %lld bytes: a multiple of 16 at a 16-byte boundary", (long long)page_bytes);
    if (seqs && (!p[0] || !p[table] || !p[table + 1] || !p[5] || !p[status] || !p[scratch] || misaligned(p[scratch], 16)))
        return fail(NC_ERR_ARGUMENT, "null table, lengths, pool, status or scratch");
    if (p[0] == p[table] && seqs) return fail(NC_ERR_ARGUMENT, "the new table is the old one");
    if (s[5] < nc_kv_pages_scratch_bytes(seqs, width, pages))
        return fail(NC_ERR_ARGUMENT, "scratch of %lld bytes, %lld needed", (long long)s[5], (long long)nc_kv_pages_scratch_bytes(seqs, width, pages));
    a->new_table = (int32_t *)p[0];
    a->table = (const int32_t *)p[table];
    a->lengths = (const int32_t *)p[table + 1];
    a->status = (int64_t *)p[status];
    int32_t *w = (int32_t *)p[scratch];
    a->words = w;                              // pairs of them are 64-bit sums
    w += KVP_WORDS;
    for (int32_t **x : {&a->refs, &a->tails, &a->owner, &a->fresh}) *x = w, w += pages;
    for (int32_t **x : {&a->first, &a->need, &a->offset}) *x = w, w += seqs;
    a->list = w;
    a->seqs = (int)seqs;
    a->width = (int)width;
    a->pages = (int)pages;
    a->page = (int)page;
    return NC_OK;
}

// One CTA for up to four pages or table entries to a thread (its barriers are cheaper), else a cluster.
cudaError_t launch_pages(void (*kernel)(KvPagesArgs), cudaStream_t st, const KvPagesArgs &a) {
    const bool many = (int64_t)a.seqs * a.width + a.pages > 4 * KVP_THREADS;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = many ? KVP_CLUSTER : 1;
    cfg.blockDim = KVP_THREADS;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = many ? KVP_CLUSTER : 1;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <bool UPDATE>
int32_t launch_pages_write(cudaStream_t st, const KvPagesArgs &a, void *pool, int64_t page_bytes) {
    CUDA_TRY(launch_k(kv_pages_write_kernel<UPDATE>, KVP_COPY_CTAS, KVP_COPY_THREADS, 0, st, a, (char *)pool, page_bytes));
    return check_launch("kv_pages_write_kernel");
}

}  // namespace

extern "C" int64_t nc_kv_pages_scratch_bytes(int64_t seqs, int64_t width, int64_t pages) {
    (void)width;
    if (seqs < 0 || pages < 0) return 0;
    return 4 * (KVP_WORDS + 4 * pages + 3 * seqs + kvp_list(seqs, pages));
}

// p: [0] new table [1] new lengths [2] table [3] lengths [4] status [5] pool [6] scratch [7] parent [8] grow
extern "C" int32_t nc_kv_pages_update(void **p, const int64_t *s, void *stream) {
    KvPagesArgs a{};
    NC_TRY(kvp_args(&a, p, s, 2, 4, 6));
    if (a.seqs == 0) return NC_OK;
    if (!p[1] || p[1] == p[3]) return fail(NC_ERR_ARGUMENT, "the new lengths are null or the old ones");
    a.new_lengths = (int32_t *)p[1];
    a.parent = (const int32_t *)p[7];
    a.grow = (const int32_t *)p[8];
    CUDA_TRY(launch_pages(kv_pages_update_kernel, (cudaStream_t)stream, a));
    NC_TRY(check_launch("kv_pages_update_kernel"));
    return launch_pages_write<true>((cudaStream_t)stream, a, p[5], s[4]);
}

extern "C" int32_t nc_kv_pages_compact(void **p, const int64_t *s, void *stream) {
    KvPagesArgs a{};
    NC_TRY(kvp_args(&a, p, s, 2, 4, 6));
    if (a.seqs == 0) return NC_OK;
    CUDA_TRY(launch_pages(kv_pages_compact_kernel, (cudaStream_t)stream, a));
    NC_TRY(check_launch("kv_pages_compact_kernel"));
    return launch_pages_write<false>((cudaStream_t)stream, a, p[5], s[4]);
}

// ---- token log probabilities ----------------------------------------------------------------------

namespace {

struct LogprobPlan {
    int segs;
    int64_t seg_vecs;
};

constexpr int64_t LP_PARTS = 1 << 14;          // segments of a launch at most, where rows are cut for speed: bounds the scratch

int64_t logprob_vecs(int64_t vocab, int64_t type) {               // of a row at any alignment
    const int n = type == KV_F32 ? 4 : 8;
    return (vocab + 2 * (n - 1)) / n;
}
// As many segments as a row has to have.
int64_t logprob_fewest(int64_t vocab, int64_t type) {
    constexpr int64_t longest = (int64_t)LP_BATCHES * LP_THREADS * LP_VECS;
    return (logprob_vecs(vocab, type) + longest - 1) / longest;
}

// Segments to a row: the fewest elements' time over the waves of CTAs that the card holds at once, a segment's
// start and end counted as 4096 elements and its share of the join as 16.
LogprobPlan logprob_plan(int64_t rows, int64_t vocab, int64_t type) {
    const int n = type == KV_F32 ? 4 : 8;
    const int64_t vecs = logprob_vecs(vocab, type), slots = 148 * LP_CTAS, fewest = logprob_fewest(vocab, type);
    int64_t best = -1;
    LogprobPlan p{0, 0};
    for (int cut : CUTS) {
        const int64_t segs = std::max<int64_t>(cut, fewest);
        if (segs > LP_SEGS || (segs > fewest && (vecs / segs < LP_THREADS || rows * segs > LP_PARTS))) break;
        const int64_t waves = (rows * segs + slots - 1) / slots, cost = waves * (vecs * n / segs + 4096) + 16 * segs;
        if (best >= 0 && cost >= best) continue;
        best = cost;
        p.seg_vecs = (vecs + segs - 1) / segs;
        p.segs = (int)((vecs + p.seg_vecs - 1) / p.seg_vecs);
    }
    return p;
}

template <int TYPE>
int32_t launch_logprobs(cudaStream_t st, const LogprobArgs &a, int64_t rows) {
    CUDA_TRY(launch_k(logprobs_kernel<TYPE>, (unsigned)(rows * a.segs), LP_THREADS, 0, st, a));
    return check_launch("logprobs_kernel");
}

}  // namespace

extern "C" int64_t nc_token_logprobs_scratch_bytes(int64_t rows, int64_t vocab, int64_t k) {
    if (rows <= 0 || vocab <= 0 || k < 0) return 4 * LP_ROWS;
    // A bound that grows with the rows: fewer of them are cut into more segments.
    int64_t most = 0;
    rows = std::min<int64_t>(rows, LP_ROWS);
    for (int type : {KV_F32, KV_F16}) {
        const int64_t fewest = logprob_fewest(vocab, type), cut = std::min<int64_t>(LP_SEGS, logprob_vecs(vocab, type) / LP_THREADS);
        most = std::max({most, rows * fewest, std::min(LP_PARTS, rows * cut)});
    }
    return 4 * LP_ROWS + most * (16 + 8 * k);
}

extern "C" int32_t nc_token_logprobs(void **p, const int64_t *s, void *stream) {
    const int64_t rows = s[0], vocab = s[1], type = s[3], ntargets = s[4], k = s[5], scratch = s[6];
    LogprobArgs a{};
    NC_TRY(check_type(type));
    if (rows < 0 || vocab <= 0 || vocab >= (int64_t(1) << 32) - 1 || ntargets < 0 || ntargets > I32)
        return fail(NC_ERR_ARGUMENT, "bad sizes: %lld rows of %lld logits, %lld targets", (long long)rows, (long long)vocab, (long long)ntargets);
    if (k < 0 || k > LP_MAX_TOP || k > vocab)
        return fail(NC_ERR_ARGUMENT, "%lld alternatives: at most %d, and no more than the vocabulary's %lld", (long long)k, LP_MAX_TOP, (long long)vocab);
    if (s[2] < vocab) return fail(NC_ERR_ARGUMENT, "rows of %lld logits overlap at a stride of %lld", (long long)vocab, (long long)s[2]);
    if (rows == 0) return NC_OK;
    const LogprobPlan plan = logprob_plan(std::min<int64_t>(rows, LP_ROWS), vocab, type);
    if (plan.segs == 0) return fail(NC_ERR_ARGUMENT, "a vocabulary of %lld is beyond %d segments", (long long)vocab, LP_SEGS);
    if (!p[5] || (ntargets && (!p[0] || !p[6])) || (k && (!p[3] || !p[4])) || misaligned(p[5], type == KV_F32 ? 4 : 2))
        return fail(NC_ERR_ARGUMENT, "null or misaligned logits, targets or outputs");
    if (misaligned(p[8], 8)) return fail(NC_ERR_ARGUMENT, "the error word is not at an 8-byte boundary");
    if (plan.segs > 1 && (!p[7] || misaligned(p[7], 16) || scratch < 4 * LP_ROWS + std::min<int64_t>(rows, LP_ROWS) * plan.segs * (16 + 8 * k)))
        return fail(NC_ERR_ARGUMENT, "scratch of %lld bytes, %lld needed", (long long)scratch,
                    (long long)nc_token_logprobs_scratch_bytes(rows, vocab, k));
    a.out = (float *)p[0];
    a.entropy = (float *)p[1];
    a.lse = (float *)p[2];
    a.top = (int64_t *)p[3];
    a.top_logprobs = (float *)p[4];
    a.logits = (const char *)p[5];
    a.targets = (const int64_t *)p[6];
    a.error = (unsigned long long *)p[8];
    a.stride = s[2];
    a.vocab = vocab;
    a.ntargets = (int)ntargets;
    a.k = (int)k;
    a.segs = plan.segs;
    a.seg_vecs = plan.seg_vecs;
    if (plan.segs > 1) {
        a.counter = (unsigned int *)p[7];
        a.part = (float4 *)((char *)p[7] + 4 * LP_ROWS);
        a.part_top = (unsigned long long *)(a.part + std::min<int64_t>(rows, LP_ROWS) * plan.segs);
    }
    const cudaStream_t st = (cudaStream_t)stream;
    for (int64_t first = 0; first < rows; first += LP_ROWS) {
        const int64_t n = std::min<int64_t>(rows - first, LP_ROWS);
        a.row_first = first;
        NC_TRY(type == KV_F32 ? launch_logprobs<KV_F32>(st, a, n) : type == KV_F16 ? launch_logprobs<KV_F16>(st, a, n)
                                                                                  : launch_logprobs<KV_BF16>(st, a, n));
    }
    return NC_OK;
}
