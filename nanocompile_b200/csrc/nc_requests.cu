// nc_requests.cu -- entry points of what the requests of a batch have of their own: low-rank adapters beside the shared
// projections, and beam search's selection and reordering of states.
//
// nanocompile runs one sequence with one set of weights and chooses its tokens by argmax on the host
// (nanocompile/models/qwen2.py:348-368); these operators have no counterpart there.
#include "nc_api.cuh"
#include "nc_beams.cuh"
#include "nc_lora_stream.cuh"

#include <algorithm>

using namespace nc;

namespace {

int32_t check_type(int64_t type) {
    if (type < KV_F32 || type > KV_BF16) return fail(NC_ERR_ARGUMENT, "element type %lld: 0 float32, 1 float16, 2 bfloat16", (long long)type);
    return NC_OK;
}
int64_t type_bytes(int64_t type) { return type == KV_F32 ? 4 : 2; }

// ---- adapters -----------------------------------------------------------------------------------

int32_t lora_batch(int64_t rows, int64_t seqs, int64_t slots) {
    if (rows < 0 || rows > I32 / 2 || seqs < 0 || seqs > LORA_SEQS || slots <= 0 || slots > I32 / 2)
        return fail(NC_ERR_ARGUMENT, "bad sizes: %lld rows of %lld sequences (%d at most), %lld adapters", (long long)rows, (long long)seqs,
                    LORA_SEQS, (long long)slots);
    if (rows && !seqs) return fail(NC_ERR_ARGUMENT, "%lld rows of no sequence", (long long)rows);
    return NC_OK;
}
int64_t lora_groups(int64_t seqs, int64_t slots) { return std::min(seqs, slots + 1); }
// Rows of an item: by the mean of the largest number of groups, as only the device knows how many there are.
int64_t lora_tile(int64_t rows, int64_t seqs, int64_t slots) {
    const int64_t mean = rows / std::max<int64_t>(1, lora_groups(seqs, slots));
    // The few items of an adapter by eights read it from L2.  Us by eights and by 128: adapters of 45 KB beside float32 rows, 64 of them for 16 rows
    // each 18 and 37, for 48 55 and 39; of 1 MB beside bfloat16 rows, 64 of them for 16 rows each 64 and 68, for 24 93 and 69, 8 of them 17 and 25.
    return mean <= 16 ? 8 : 128;
}
// Items at most: a group that has any has a row.
int64_t lora_places(int64_t rows, int64_t seqs, int64_t slots) {
    const int64_t groups = std::min(rows, lora_groups(seqs, slots));
    return groups + (rows - groups) / lora_tile(rows, seqs, slots);
}
// Items that are to be expected of them: one to a group, or half an item for the end of each.
int lora_items(int64_t rows, int64_t seqs, int64_t slots) {
    const int64_t groups = std::min(rows, lora_groups(seqs, slots)), tile = lora_tile(rows, seqs, slots);
    return (int)std::min(lora_places(rows, seqs, slots), std::max(groups, (2 * rows + tile * groups + 2 * tile - 1) / (2 * tile)));
}
// Clusters of 1 to 8 CTAs that a B200 holds at once, with one CTA on an SM and with two: fewer than its SMs would hold, as a cluster lies
// within one of its processing clusters, and for two twice as many, as they come to lie (32 clusters of 8: 26 us, 24 of them 16).  A
// device with other processing clusters only has a rule that fits it less well.
constexpr int CLUSTERS_ALONE[8] = {148, 74, 45, 33, 26, 22, 15, 15}, CLUSTERS_TWO[8] = {296, 148, 90, 66, 52, 44, 30, 30};
// Rounds in which `clusters` of `n` CTAs run.
int lora_rounds(int64_t clusters, int n, bool two) {
    const int at_once = (two ? CLUSTERS_TWO : CLUSTERS_ALONE)[n - 1];
    return (int)((clusters + at_once - 1) / at_once);
}

template <int TX, int TW, int NT>
int32_t launch_lora(cudaStream_t st, const LoraArgs &a, int passes) {
    auto kernel = lora_rows_kernel<TX, TW, NT>;
    constexpr size_t bytes = LoraShape<NT>::SMEM;
    static std::atomic<uint64_t> allowed{0};
    NC_TRY(allow_smem_once(kernel, bytes, &allowed));
    const int64_t subs = (a.tile + 8 * NT - 1) / (8 * NT), clusters = (int64_t)a.items * passes * subs;
    int ctas = 8;                              // as many CTAs to an item as leave room for all items at once, two on an SM
    while (ctas > 1 && clusters * ctas > 2 * 148) ctas /= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.items * ctas), (unsigned)passes, (unsigned)subs);
    cfg.blockDim = LORA_THREADS;
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ctas;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, a));
    return check_launch("lora_rows_kernel");
}
// For items of eight rows.  False where a CTA's share of the inputs is too long, or its part of an adapter so small that the ring
// takes longer than it saves.  With the ring and without, us a call, adapters cold: 15 KB a CTA (896 -> 1152 at rank 16) one row 10.0 and 9.6, 64
// rows of 8 adapters 12.4 and 10.6; 28 KB (896 -> 896 at 64) 9.5 and 8.8, 13.0 and 10.1; 30 KB (896 -> 1152 at 32) 11.4 and 11.8, 15.5 and
// 13.2; 32 KB (4096 -> 4096 at 16) 10.3 and 11.2, 12.5 and 12.9; 64 KB (4096 -> 4096 at 32) 9.6 and 11.6, 12.9 and 13.5.  Most is saved where
// outputs are many (896 -> 9728 at 16: 12.4 and 17.7); with few of them the ring may take up to a fifth longer (4864 -> 896 at 64: one row 11.7 and
// 11.5, 64 rows of 8 bfloat16 adapters 15.3 and 12.5, 32 of 32 adapters 15.1 and 16.7).  With one CTA or two to many items it pays earlier:
// 28 KB (128 adapters of 896 -> 896 at 16) 11.8 and 12.5.
template <int TX, int TW>
bool lora_stream_shape(const LoraArgs &a, int passes, int items, int *ctas, LoraStreamPlan *plan) {
    using S = LoraStream<TX, TW>;
    const int units = (a.inputs + 31) / 32;
    const double bytes = 2.0 * a.rank * ((double)a.targets * a.inputs + a.outputs) / passes;
    // CTAs of a cluster, by rounds: 10 us to start and to add up, then bytes at 22 a ns for each of two on an SM, 30 alone.  Measured:
    // 64 adapters of 1 MB 24 us by 4 CTAs, 44 by 8; 128 of them 46 by 4 with two on an SM, 58 by 2 alone.
    double best = 0.0;
    *ctas = 0;
    for (int n = 8; n >= 1; --n) {
        const LoraStreamPlan p = lora_stream_plan(a.pass_targets, a.rank, (units + n - 1) / n * 32, S::PX, S::PH);
        if (!p.fits) break;
        const bool two = p.bytes <= LS_BYTES;
        const int rounds = lora_rounds((int64_t)items * passes, n, two);
        if (rounds > 1 && (n & (n - 1))) continue; // clusters of odd sizes do not take each other's places: 200 adapters of 1 MB 97 us by 3, 79 by 4
        const double cost = rounds * (10.0 + 1e-3 * bytes / n / (two ? 22.0 : 30.0));
        if (*ctas != 0 && cost >= best) continue;
        best = cost;
        *ctas = n;
        *plan = p;
    }
    return *ctas != 0 && bytes / *ctas > (*ctas > 2 ? 28 : 24) * 1024;
}
template <int TX, int TW>
int32_t launch_lora_stream(cudaStream_t st, const LoraArgs &a, int passes, int ctas, const LoraStreamPlan &plan) {
    auto kernel = lora_stream_kernel<TX, TW>;
    static std::atomic<uint64_t> allowed{0};
    NC_TRY(allow_smem_once(kernel, LS_BYTES_ALONE, &allowed));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.items * ctas), (unsigned)passes);
    cfg.blockDim = LS_THREADS;
    cfg.dynamicSmemBytes = plan.bytes;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ctas;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, a, plan));
    return check_launch("lora_stream_kernel");
}
// For items of 128 rows.  False where shared memory is too small for the rank (float16 adapters above 96 beside float32 rows).
template <int TX, int TW>
bool lora_tiles_shape(LoraArgs *a, LoraTilesPlan *plan) {
    using S = LoraTiles<TX, TW>;
    a->pass_targets = std::min(a->targets, std::max(1, LORA_PASS / ((a->rank + 15) / 16 * 16)));
    *plan = lora_tiles_plan<S>(a->pass_targets, a->rank);
    while ((plan->slots < 2 || plan->stages < 2) && a->pass_targets > 1) *plan = lora_tiles_plan<S>(--a->pass_targets, a->rank);
    return plan->slots >= 2 && plan->stages >= 2;
}
template <int TX, int TW>
int32_t launch_lora_tiles(cudaStream_t st, const LoraArgs &a, int items, const LoraTilesPlan &plan) {
    auto kernel = lora_tiles_kernel<TX, TW>;
    static std::atomic<uint64_t> allowed{0};
    NC_TRY(allow_smem_once(kernel, LT_BYTES + 1024, &allowed));
    const int passes = (a.targets + a.pass_targets - 1) / a.pass_targets;
    const size_t bytes = (size_t)plan.bytes + 1024;
    // CTAs of a cluster, one on an SM, by rounds: 14 us for what does not depend on an item's size, then its bytes.
    const double size = TX == KV_F32 ? 4 : 2, rate = TX == KV_F32 ? 20.0 : 33.0;
    const double moved = LT_ROWS * size * ((double)a.inputs + (a.base ? 2.0 : 1.0) * a.outputs / passes);
    double best = 0.0;
    int ctas = 0;
    for (int n = 8; n >= 1; --n) {
        const double cost = lora_rounds((int64_t)items * passes, n, false) * (14.0 + 1e-3 * moved / n / rate);
        if (ctas != 0 && cost >= best) continue;
        best = cost;
        ctas = n;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.items * ctas), (unsigned)passes);
    cfg.blockDim = LT_THREADS;
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ctas;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, a, plan));
    return check_launch("lora_tiles_kernel");
}
template <int TX, int TW>
int32_t launch_lora_n(cudaStream_t st, const LoraArgs &a, int passes, int items, bool tiles) {
    if constexpr (TX == TW || TX == KV_F32)
        if (tiles) {
            LoraArgs t = a;
            LoraTilesPlan plan;
            if (lora_tiles_shape<TX, TW>(&t, &plan)) return launch_lora_tiles<TX, TW>(st, t, items, plan);
        }
    if (a.tile == 8) {
        int ctas;
        LoraStreamPlan plan;
        if (lora_stream_shape<TX, TW>(a, passes, items, &ctas, &plan)) return launch_lora_stream<TX, TW>(st, a, passes, ctas, plan);
    }
    return a.tile == 8 ? launch_lora<TX, TW, 1>(st, a, passes) : launch_lora<TX, TW, 4>(st, a, passes);
}
template <int TX>
int32_t launch_lora_w(cudaStream_t st, const LoraArgs &a, int passes, int items, bool tiles) {
    return a.wtype == KV_F16 ? launch_lora_n<TX, KV_F16>(st, a, passes, items, tiles) : launch_lora_n<TX, KV_BF16>(st, a, passes, items, tiles);
}

}  // namespace

int32_t nc::set_requests_wait_limit(long long cycles) {
    CUDA_TRY(cudaMemcpyToSymbol(g_wait_cycles, &cycles, sizeof(cycles)));
    return NC_OK;
}

// What went wrong in the adapters' kernels since the last call, or null; clears it.
int32_t nc::requests_fault(const char **what) {
    unsigned int word = 0;
    CUDA_TRY(cudaMemcpyFromSymbol(&word, g_lora_fault, sizeof(word)));
    *what = word & LORA_LATE    ? "a copy or a matrix instruction did not complete within its wait limit"
            : word & LORA_OTHER ? "a plan was made for other rows, sequences or slots than the projection's"
                                : nullptr;
    word = 0;
    if (*what) CUDA_TRY(cudaMemcpyToSymbol(g_lora_fault, &word, sizeof(word)));
    return NC_OK;
}

extern "C" int64_t nc_lora_plan_bytes(int64_t rows, int64_t seqs, int64_t slots) {
    if (rows < 0 || rows > I32 / 2 || seqs < 0 || seqs > LORA_SEQS || slots <= 0 || slots > I32 / 2) return 0;
    return 4 * (LORA_HEAD + 4 * lora_places(rows, seqs, slots) + rows);
}

extern "C" int32_t nc_lora_plan(void **p, const int64_t *s, void *stream) {
    const int64_t rows = s[0], seqs = s[1], slots = s[2];
    NC_TRY(lora_batch(rows, seqs, slots));
    if (!p[2] && rows != seqs) return fail(NC_ERR_ARGUMENT, "%lld rows of %lld sequences need row_start", (long long)rows, (long long)seqs);
    if (!p[0] || misaligned(p[0], 16) || s[3] < nc_lora_plan_bytes(rows, seqs, slots))
        return fail(NC_ERR_ARGUMENT, "a plan of %lld bytes, %lld needed at a 16-byte boundary", (long long)s[3], (long long)nc_lora_plan_bytes(rows, seqs, slots));
    if (seqs && !p[1]) return fail(NC_ERR_ARGUMENT, "null adapters");
    if (misaligned(p[3], 8)) return fail(NC_ERR_ARGUMENT, "the error word is not at an 8-byte boundary");
    LoraPlanArgs a{};
    a.plan = (int32_t *)p[0];
    a.adapters = (const int32_t *)p[1];
    a.row_start = (const int32_t *)p[2];
    a.error = (unsigned long long *)p[3];
    a.rows = (int)rows;
    a.seqs = (int)seqs;
    a.slots = (int)slots;
    a.tile = (int)lora_tile(rows, seqs, slots);
    a.items = (int)lora_places(rows, seqs, slots);
    a.size = 2;
    while (a.size < a.seqs) a.size *= 2;
    // Threads for the longer of the sort's pairs, the items and the rows, as barriers of fewer warps are cheaper.
    const int64_t work = std::max<int64_t>({a.size / 2, a.items, rows / 4});
    const unsigned threads = work <= 128 ? 128 : work <= 256 ? 256 : work <= 512 ? 512 : 1024;
    const size_t bytes = (size_t)a.size * 8 + (size_t)4 * 4 * (a.size + 1);
    static std::atomic<uint64_t> allowed{0};
    NC_TRY(allow_smem_once(lora_plan_kernel, (size_t)LORA_SEQS * 8 + (size_t)4 * 4 * (LORA_SEQS + 1), &allowed));
    CUDA_TRY(launch_k(lora_plan_kernel, 1, threads, bytes, (cudaStream_t)stream, a));
    return check_launch("lora_plan_kernel");
}

extern "C" int32_t nc_lora_project(void **p, const int64_t *s, void *stream) {
    LoraArgs a{};
    const int64_t rows = s[0], seqs = s[1], slots = s[2], inputs = s[3], rank = s[4], targets = s[5], type = s[6], wtype = s[7];
    NC_TRY(lora_batch(rows, seqs, slots));
    NC_TRY(check_type(type));
    if (wtype != KV_F16 && wtype != KV_BF16) return fail(NC_ERR_ARGUMENT, "adapters of element type %lld: 1 float16 or 2 bfloat16", (long long)wtype);
    if (inputs <= 0 || inputs % 8 || inputs > LORA_LINE || rank <= 0 || rank % 8 || rank > LORA_RANK)
        return fail(NC_ERR_ARGUMENT, "%lld inputs (%d at most), rank %lld: multiples of 8, the rank %d at most", (long long)inputs, LORA_LINE, (long long)rank,
                    LORA_RANK);
    if (targets <= 0 || targets > LORA_TARGETS) return fail(NC_ERR_ARGUMENT, "%lld targets: 1 to %d", (long long)targets, LORA_TARGETS);
    int64_t outputs = 0;
    bool even = true;
    for (int t = 0; t < targets; ++t) {
        const int64_t width = s[12 + t];
        if (width <= 0 || width > LORA_LINE - outputs)
            return fail(NC_ERR_ARGUMENT, "a target of %lld outputs after %lld: %d at most", (long long)width, (long long)outputs, LORA_LINE);
        even = even && outputs % 2 == 0;
        a.width[t] = (int)width;
        outputs += width;
    }
    if (s[8] < nc_lora_plan_bytes(rows, seqs, slots) || !p[5] || misaligned(p[5], 16))
        return fail(NC_ERR_ARGUMENT, "a plan of %lld bytes, %lld needed at a 16-byte boundary", (long long)s[8], (long long)nc_lora_plan_bytes(rows, seqs, slots));
    if (rows == 0) return NC_OK;
    const int64_t bytes = type_bytes(type);
    a.out = p[0];
    a.x = p[1];
    a.base = p[2];
    a.a = p[3];
    a.b = p[4];
    a.plan = (const int32_t *)p[5];
    a.ranks = (const int32_t *)p[6];
    a.scales = (const float *)p[7];
    a.x_stride = s[9];
    a.base_stride = s[10];
    a.out_stride = s[11];
    if (!a.out || !a.x || !a.a || !a.b) return fail(NC_ERR_ARGUMENT, "null output, rows or adapters");
    if (misaligned(a.a, 16) || misaligned(a.b, 16)) return fail(NC_ERR_ARGUMENT, "adapters are not at a 16-byte boundary");
    if (misaligned(a.x, bytes) || misaligned(a.out, bytes) || misaligned(a.base, bytes)) return fail(NC_ERR_ARGUMENT, "misaligned rows");
    if (a.x_stride < inputs || a.out_stride < outputs || (a.base && a.base_stride < outputs))
        return fail(NC_ERR_ARGUMENT, "rows of %lld inputs or %lld outputs overlap", (long long)inputs, (long long)outputs);
    if (a.out == a.x) return fail(NC_ERR_ARGUMENT, "the outputs are the inputs");
    if (a.out == a.base && a.out_stride != a.base_stride)
        return fail(NC_ERR_ARGUMENT, "outputs in place of base at a stride of %lld, base's is %lld", (long long)a.out_stride, (long long)a.base_stride);
    a.rows = (int)rows;
    a.seqs = (int)seqs;
    a.items = (int)lora_places(rows, seqs, slots);
    a.tile = (int)lora_tile(rows, seqs, slots);
    a.inputs = (int)inputs;
    a.outputs = (int)outputs;
    a.rank = (int)rank;
    a.slots = (int)slots;
    a.targets = (int)targets;
    a.wtype = (int)wtype;
    a.x_vectors = !misaligned(a.x, 16) && !misaligned(a.x_stride * bytes, 16);
    a.pairs = even && !misaligned(a.out, 2 * bytes) && !misaligned(a.base, 2 * bytes) && a.out_stride % 2 == 0 && (!a.base || a.base_stride % 2 == 0);
    bool wide = !misaligned(a.out, 16) && !misaligned(a.base, 16) && !misaligned(a.out_stride * bytes, 16) && (!a.base || !misaligned(a.base_stride * bytes, 16));
    for (int t = 0; t + 1 < targets; ++t) wide = wide && !misaligned(a.width[t] * bytes, 16);
    a.wide = wide;
    a.pass_targets = (int)std::min<int64_t>(targets, std::max<int64_t>(1, LORA_PASS / ((rank + 31) / 32 * 32)));
    const int passes = (int)((targets + a.pass_targets - 1) / a.pass_targets);
    const cudaStream_t st = (cudaStream_t)stream;
    const bool tiles = a.tile == LT_ROWS && a.x_vectors && targets * rank * inputs <= I32;
    const int items = lora_items(rows, seqs, slots);
    return type == KV_F32 ? launch_lora_w<KV_F32>(st, a, passes, items, tiles) : type == KV_F16 ? launch_lora_w<KV_F16>(st, a, passes, items, tiles)
                                                                                                : launch_lora_w<KV_BF16>(st, a, passes, items, tiles);
}

// ---- beams --------------------------------------------------------------------------------------

namespace {

constexpr int64_t BEAM_COUNTERS = BEAM_ROWS;

int64_t beam_batches(int64_t vocab, int64_t type) {               // of a row at any alignment
    const int64_t n = 16 / type_bytes(type), vecs = (vocab + 2 * (n - 1)) / n;
    return (vecs + BEAM_BATCH - 1) / BEAM_BATCH;
}
// Batches of a CTA's share at least, that a request has no more than BEAM_LISTS segments (0: it has more), and segments of a row at most:
// it is cut where shares end, and after every 16 batches.
struct BeamPlan {
    int64_t least, lists;
};
BeamPlan beam_plan(int64_t batches, int64_t beams) {
    auto lists = [&](int64_t least) { return std::min(batches, (std::max<int64_t>(batches - 2, 0)) / least + 2 + batches / BEAM_BATCHES); };
    if (lists(batches) * beams > BEAM_LISTS) return BeamPlan{0, 0};
    int64_t least = std::max<int64_t>(1, batches * beams / BEAM_LISTS);
    // Two batches where that leaves half of the candidates that are taken at once: 4 beams of 151936 float32 logits 13.2 us, 14.7 with one.
    if (least == 1 && batches > 1 && lists(1) * beams * beams > 512 && lists(2) * beams * beams <= 512) least = 2;
    while (lists(least) * beams > BEAM_LISTS) ++least;
    return BeamPlan{least, lists(least)};
}
int64_t beam_launch_rows(int64_t rows, int64_t beams) { return std::min<int64_t>(rows, BEAM_ROWS / beams * beams); }

template <int TYPE>
int32_t launch_beams(cudaStream_t st, const BeamArgs &a, int64_t rows) {
    CUDA_TRY(launch_k(beam_select_kernel<TYPE>, (unsigned)std::min<int64_t>(rows * a.batches, BEAM_CTAS), LP_THREADS, 0, st, a));
    return check_launch("beam_select_kernel");
}

}  // namespace

extern "C" int64_t nc_beam_select_scratch_bytes(int64_t rows, int64_t vocab, int64_t beams) {
    if (rows <= 0 || vocab <= 0 || beams <= 0 || beams > LP_MAX_TOP) return 4 * BEAM_COUNTERS;
    // Of the most segments that any smaller vocabulary and number of beams may have (smaller ones can have more: 64 batches of 8 beams are
    // cut into 64 segments, 65 into 37): a batch each, and BEAM_LISTS of a request.
    int64_t row = 0;
    for (int64_t n = 1; n <= beams; ++n) row = std::max(row, std::min<int64_t>(beam_batches(vocab, KV_F32), BEAM_LISTS / n) * 8 * (1 + n));
    return 4 * BEAM_COUNTERS + std::min<int64_t>(rows, BEAM_ROWS) * row;
}

extern "C" int32_t nc_beam_select(void **p, const int64_t *s, void *stream) {
    const int64_t rows = s[0], vocab = s[1], type = s[3], beams = s[4], scratch = s[6];
    BeamArgs a{};
    NC_TRY(check_type(type));
    if (rows < 0 || rows > I32 || vocab <= 0 || vocab >= (int64_t(1) << 32) - 1)
        return fail(NC_ERR_ARGUMENT, "bad sizes: %lld rows of %lld logits", (long long)rows, (long long)vocab);
    if (beams <= 0 || beams > LP_MAX_TOP || rows % beams)
        return fail(NC_ERR_ARGUMENT, "%lld beams: at most %d, and the %lld rows are those of whole requests", (long long)beams, LP_MAX_TOP, (long long)rows);
    if (s[2] < vocab) return fail(NC_ERR_ARGUMENT, "rows of %lld logits overlap at a stride of %lld", (long long)vocab, (long long)s[2]);
    if (s[5] >= vocab) return fail(NC_ERR_ARGUMENT, "the end token %lld is outside the vocabulary", (long long)s[5]);
    if (s[5] < 0 && p[8]) return fail(NC_ERR_ARGUMENT, "finished beams without an end token");
    if (rows == 0) return NC_OK;
    const int64_t at_once = beam_launch_rows(rows, beams), k = std::min(beams, vocab);
    const BeamPlan plan = beam_plan(beam_batches(vocab, type), beams);
    if (plan.least == 0) return fail(NC_ERR_ARGUMENT, "a vocabulary of %lld is too large for %lld beams", (long long)vocab, (long long)beams);
    if (!p[0] || !p[1] || !p[2] || !p[6] || !p[7] || misaligned(p[6], type_bytes(type)))
        return fail(NC_ERR_ARGUMENT, "null or misaligned logits, scores or outputs");
    if (p[7] == p[2] || (p[8] && p[8] == p[3])) return fail(NC_ERR_ARGUMENT, "the new scores or flags are the old ones");
    if (misaligned(p[11], 8)) return fail(NC_ERR_ARGUMENT, "the error word is not at an 8-byte boundary");
    const int64_t need = 4 * BEAM_COUNTERS + at_once * plan.lists * (8 + 8 * k);
    if (!p[10] || misaligned(p[10], 16) || scratch < need)
        return fail(NC_ERR_ARGUMENT, "scratch of %lld bytes, %lld needed", (long long)scratch, (long long)nc_beam_select_scratch_bytes(rows, vocab, beams));
    a.parent = (int32_t *)p[0];
    a.tokens = (int64_t *)p[1];
    a.new_scores = (float *)p[2];
    a.new_finished = (int32_t *)p[3];
    a.grow = (int32_t *)p[4];
    a.history = (int32_t *)p[5];
    a.logits = (const char *)p[6];
    a.scores = (const float *)p[7];
    a.finished = (const int32_t *)p[8];
    a.norms = (const float *)p[9];
    a.error = (unsigned long long *)p[11];
    a.stride = s[2];
    a.vocab = vocab;
    a.beams = (int)beams;
    a.end = s[5];
    a.k = (int)k;
    a.batches = (int)beam_batches(vocab, type);
    a.least = (int)plan.least;
    a.lists = (int)plan.lists;
    a.counter = (unsigned int *)p[10];
    a.part_top = (unsigned long long *)((char *)p[10] + 4 * BEAM_COUNTERS);
    a.part = (float2 *)(a.part_top + at_once * plan.lists * k);
    const cudaStream_t st = (cudaStream_t)stream;
    for (int64_t first = 0; first < rows; first += at_once) {
        const int64_t n = std::min(rows - first, at_once);
        a.row_first = first;
        a.rows = (int)n;
        NC_TRY(type == KV_F32 ? launch_beams<KV_F32>(st, a, n) : type == KV_F16 ? launch_beams<KV_F16>(st, a, n) : launch_beams<KV_BF16>(st, a, n));
    }
    return NC_OK;
}

namespace {

template <typename V>
int32_t launch_reorder(cudaStream_t st, ReorderArgs a) {
    const int64_t chunk = (int64_t)sizeof(V) * BEAM_COPY_THREADS * BEAM_COPY_VECS;
    a.chunks = std::max<int64_t>(1, (a.capacity * a.line + chunk - 1) / chunk);
    const int64_t ctas = (int64_t)a.rows * a.planes <= I32 / a.chunks ? a.rows * a.planes * a.chunks : 0;
    if (ctas == 0) return fail(NC_ERR_ARGUMENT, "%d rows of %d planes of %lld bytes in one call", a.rows, a.planes, (long long)(a.capacity * a.line));
    CUDA_TRY(launch_k(beam_reorder_kernel<V>, (unsigned)ctas, BEAM_COPY_THREADS, 0, st, a));
    return check_launch("beam_reorder_kernel");
}

}  // namespace

extern "C" int32_t nc_beam_reorder(void **p, const int64_t *s, void *stream) {
    const int64_t rows = s[0], planes = s[1], capacity = s[2], line = s[3], to_stride = s[4], from_stride = s[5];
    if (rows < 0 || rows > I32 || planes <= 0 || planes > I32 || capacity < 0 || capacity >= I32 || line <= 0 || line > (int64_t(1) << 40) / std::max<int64_t>(1, capacity))
        return fail(NC_ERR_ARGUMENT, "bad sizes: %lld rows of %lld planes of %lld lines of %lld bytes", (long long)rows, (long long)planes, (long long)capacity,
                    (long long)line);
    if (planes * (long double)capacity * line > 4e18L || to_stride < planes * capacity * line || from_stride < planes * capacity * line)
        return fail(NC_ERR_ARGUMENT, "rows of %lld planes of %lld lines of %lld bytes overlap", (long long)planes, (long long)capacity, (long long)line);
    if (rows == 0) return NC_OK;
    if (!p[2] || (capacity && (!p[0] || !p[1]))) return fail(NC_ERR_ARGUMENT, "null states or parents");
    if (p[0] == p[1] && capacity) return fail(NC_ERR_ARGUMENT, "the new states are the old ones");
    if (p[3] && p[3] == p[4]) return fail(NC_ERR_ARGUMENT, "the new lengths are the old ones");
    if (!p[3] && (p[4] || p[5] || p[6])) return fail(NC_ERR_ARGUMENT, "new lengths, a line to append or grow without lengths");
    if (p[6] && !p[5]) return fail(NC_ERR_ARGUMENT, "grow without a line to append");
    ReorderArgs a{};
    a.to = (char *)p[0];
    a.from = (const char *)p[1];
    a.parent = (const int32_t *)p[2];
    a.lengths = (const int32_t *)p[3];
    a.new_lengths = (int32_t *)p[4];
    a.append = (const char *)p[5];
    a.grow = (const int32_t *)p[6];
    a.to_stride = to_stride;
    a.from_stride = from_stride;
    a.line = line;
    a.rows = (int)rows;
    a.planes = (int)planes;
    a.capacity = (int)capacity;
    // The widest vectors that every plane of every row begins at.
    const int64_t at = (int64_t)(uintptr_t)p[0] | (int64_t)(uintptr_t)p[1] | to_stride | from_stride | capacity * line;
    const cudaStream_t st = (cudaStream_t)stream;
    if (!misaligned(at, 16)) return launch_reorder<uint4>(st, a);
    if (!misaligned(at, 8)) return launch_reorder<uint2>(st, a);
    if (!misaligned(at, 4)) return launch_reorder<uint32_t>(st, a);
    return !misaligned(at, 2) ? launch_reorder<uint16_t>(st, a) : launch_reorder<uint8_t>(st, a);
}
