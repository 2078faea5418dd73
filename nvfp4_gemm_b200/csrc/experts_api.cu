// C ABI of the mixture-of-experts operators (declared in include/nvfp4_b200.h): argument checks, kernel selection, launch.
// Nothing is allocated and nothing is kept between calls.
#include "api_internal.h"
#include "expert_gemm_sm100.cuh"
#include "route_kernels.cuh"

namespace {

using namespace nvfp4;
using namespace nvfp4::host;

// Rows of an expert that the grouped product takes at a time: the form with two CTAs per SM (32) where experts have
// few rows, CTA pairs (256) where they have more.  Measured (us, 32 / 256; weights E x n x k): 16 rows per expert on average, 32 x 7168 x 2048
// 39.7 / 43.4, 32 x 4096 x 4096 46.9 / 49.7, 256 x 2048 x 2048 94.6 / 90.6; 24 rows, 32 x 4096 x 4096 51.1 / 50.9; 42 rows 63.3 / 54.1; 32 rows,
// 256 x 2048 x 2048 104.5 / 99.6.  (64 rows at a time with a shallower ring: 36.3 instead of 34.7 at 2 rows, 48.5 at 16, 59.1 at 42.)
constexpr int kTileFew = 32, kTileMany = 256;   // (powers of two: PlanParams::tile_shift)
constexpr int kManyFrom = 20;   // rows per expert, on average

struct PlanSizes {
    int tile_tokens, tile_sf_rows, chunk_tokens, chunks;
    long long max_tiles, count_words, words, sf_rows;
};

int plan_sizes(int tokens, int top_k, int experts, PlanSizes* s) {
    if (tokens < 0 || top_k < 1 || experts < 1)
        return fail(NVFP4_ERR_INVALID_ARGUMENT, "tokens must not be negative, top_k and experts must be positive (got %d, %d, %d)", tokens, top_k, experts);
    if (experts > kMaxExperts || top_k > kMaxTopK)
        return fail(NVFP4_ERR_INVALID_ARGUMENT, "at most %d experts and top_k %d (got %d, %d)", kMaxExperts, kMaxTopK, experts, top_k);
    const long long pairs = static_cast<long long>(tokens) * top_k;
    s->tile_tokens = pairs < static_cast<long long>(kManyFrom) * experts ? kTileFew : kTileMany;
    s->tile_sf_rows = (s->tile_tokens + 127) / 128 * 128;
    // sum over the experts that have rows of ceil(rows / tile)
    s->max_tiles = pairs / s->tile_tokens + (pairs < experts ? pairs : experts);
    s->sf_rows = s->max_tiles * s->tile_sf_rows;
    if (pairs > 0x7fffffffll || s->sf_rows > 0x7fffffffll) return fail(NVFP4_ERR_INVALID_ARGUMENT, "problem too large: %lld pairs", pairs);
    // Chunks of the tokens: one CTA each, 148 at most (more only where a chunk's pairs would not be counted in 16 bits), or a single one, which
    // takes one launch for choice and order.  Router, one chunk / more (us): 160 x 8 of 64 experts 6.4 / 7.7, of 256 9.3 / 10.3; 256 x 4 of 32
    // 6.8 / 7.5; 300 x 2 of 32 7.3 / 7.3; 200 x 6 of 256 11.0 / 10.1 (the pairs of 256 experts are ranked 1152 at a time); 340 x 3 of 64 8.0 / 7.8; 512 x 2 of 64
    // 8.9 / 7.8; 256 x 8 of 64 9.0 / 7.7.
    constexpr int kUnit = 8, kMostChunks = 148, kOneChunk = 256;
    const bool one = tokens <= kOneChunk && pairs <= (experts <= 128 ? 1280 : 1024);
    int chunk_tokens = one ? kOneChunk : kUnit * ((tokens + kUnit * kMostChunks - 1) / (kUnit * kMostChunks));
    if (chunk_tokens < 32) chunk_tokens = 32;
    if (chunk_tokens > kMaxChunkPairs / top_k) chunk_tokens = kMaxChunkPairs / top_k;
    s->chunk_tokens = chunk_tokens;
    s->chunks = (tokens + chunk_tokens - 1) / chunk_tokens;
    s->count_words = static_cast<long long>(s->chunks) * counts_row(experts) / 2;
    s->words = 4 + 4 * s->max_tiles + s->count_words + pairs;
    return NVFP4_OK;
}

int check_routing(const nvfp4_routing* r, PlanSizes* s) {
    if (!r) return fail(NVFP4_ERR_INVALID_ARGUMENT, "routing is NULL");
    if (int rc = plan_sizes(r->tokens, r->top_k, r->experts, s)) return rc;
    if (!r->plan || !aligned(r->plan, 16)) return fail(NVFP4_ERR_INVALID_ARGUMENT, "routing.plan must be a 16-byte aligned pointer");
    return NVFP4_OK;
}

// (bits, by which a chunk's pairs are ranked: all of them at once where 36 KB allow it)
void set_chunks(PlanParams* q, int chunk_tokens, int chunks) {
    q->chunk_tokens = chunk_tokens;
    q->chunks = chunks;
    const int in_chunk = q->tokens < chunk_tokens ? q->tokens : chunk_tokens;
    const long long needed = (static_cast<long long>(in_chunk) * q->top_k + 31) / 32, most = 9216 / q->experts;
    q->bit_words = static_cast<int>(needed < most ? needed : most);
}

PlanParams plan_params(const nvfp4_routing* r, const PlanSizes& s) {
    PlanParams q;
    q.tokens = r->tokens; q.top_k = r->top_k; q.experts = r->experts;
    q.tile_tokens = s.tile_tokens; q.tile_sf_rows = s.tile_sf_rows;
    q.tile_shift = s.tile_tokens == kTileFew ? 5 : 8;
    set_chunks(&q, s.chunk_tokens, s.chunks);
    q.expert = r->expert; q.row = r->row; q.offset = r->offset;
    int* words = static_cast<int*>(r->plan);
    q.tile_count = words;
    q.tiles = reinterpret_cast<int4*>(words + 4);
    q.counts = reinterpret_cast<uint16_t*>(words + 4 + 4 * s.max_tiles);
    q.sf_row = words + 4 + 4 * s.max_tiles + s.count_words;
    return q;
}

// A launch whose set-up may overlap the end of the kernel before it in the stream (the kernels wait before their first access).
template <class... Params, class... Args>
int launch(void (*kernel)(Params...), unsigned grid, unsigned block, size_t smem, unsigned cluster, cudaStream_t stream, const char* name, const Args&... args) {
    cudaLaunchConfig_t cfg;
    std::memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(grid, 1, 1);
    cfg.blockDim = dim3(block, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, args...));
    g_launches.fetch_add(1);
    t_last_kernel = name;
    return NVFP4_OK;
}

int check_device(DeviceCtx** c) {
    if (int rc = get_ctx(c)) return rc;
    if (!(*c)->sm100) return fail(NVFP4_ERR_UNSUPPORTED, "device %d is not sm_100", (*c)->device);
    return NVFP4_OK;
}

// No tokens: no rows and no tiles.
int empty_plan(const PlanParams& q, cudaStream_t stream) {
    CUDA_TRY(cudaMemsetAsync(q.offset, 0, (q.experts + 1) * sizeof(int), stream));
    CUDA_TRY(cudaMemsetAsync(q.tile_count, 0, sizeof(int), stream));
    return NVFP4_OK;
}

// More than half of an SM's shared memory: one CTA of the plan's kernels on an SM.  (Two of them, as they come to stand where the kernel ahead leaves
// SMs free early, share its instructions: 2000 tokens x 8 of 256 18.7 us instead of 17.4, plan of 65536 x 8 of 256 28.8 instead of 21.0.)
constexpr size_t kPlaceSmem = 116 * 1024;
constexpr int kPlaceMostCtas = 120;    // as many as 148 SMs hold in clusters of eight
size_t plan_smem(const PlanParams& q) {
    const int per_expert = (q.bit_words | 1) < 3 ? 3 : (q.bit_words | 1);     // (the place kernel keeps three sums there)
    return (plan_head_words(q.experts) + static_cast<size_t>(q.experts) * per_expert) * sizeof(int);
}

// Raises a kernel's limit of dynamic shared memory once per device.
int allow_smem(DeviceCtx* c, int variant, const void* kernel, size_t bytes) {
    if (bytes > 48 * 1024 && !c->smem_attr_set[variant]) {
        CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
        c->smem_attr_set[variant] = true;
    }
    return NVFP4_OK;
}

template <int CHUNKS>
int place(DeviceCtx* c, int variant, const PlanParams& q, cudaStream_t stream, const char* name) {
    constexpr int kChunks = kPlaceCluster * CHUNKS;
    const size_t smem = plan_smem(q) > kPlaceSmem ? plan_smem(q) : kPlaceSmem;
    if (int rc = allow_smem(c, variant, reinterpret_cast<const void*>(place_kernel<CHUNKS>), smem)) return rc;
    return launch(place_kernel<CHUNKS>, (q.chunks + kChunks - 1) / kChunks * kPlaceCluster, kPlaceThreads, smem, kPlaceCluster, stream, name, q);
}
int place(DeviceCtx* c, const PlanParams& q, cudaStream_t stream, const char* name) {
    if (q.chunks <= 1) return NVFP4_OK;
    return q.chunks > kPlaceMostCtas ? place<2>(c, 74, q, stream, name) : place<1>(c, 88, q, stream, name);
}

template <bool BY_LOGIT, int VPL>
int launch_route(DeviceCtx* c, int variant, RouteParams p, const PlanParams& q, cudaStream_t stream, const char* name) {
    // A warp per token.  Each has 128 words for candidates; with groups room for all keys, in 64 bits: at most 64 KB.
    constexpr int kMost = route_threads(VPL) / 32;
    const int per = q.experts / p.groups, lanes = per / VPL;
    p.direct_lanes = per % VPL == 0 && (lanes & (lanes - 1)) == 0 ? lanes : 0;
    const size_t size = p.logit_type == kLogitFp32 ? 4 : 2, piece = VPL * size < 16 ? VPL * size : 16;
    p.vector = aligned(p.logits, piece) && p.logits_row_stride * size % piece == 0;
    p.key_words = p.groups > 1 && 2 * q.experts > 128 ? (2 * q.experts + 3) & ~3 : 128;
    const int in_chunk = q.tokens < q.chunk_tokens ? q.tokens : q.chunk_tokens;
    // One chunk: up to eight CTAs, so that a scheduler has few tokens to issue for (32 tokens of 256 experts: 7.4 us, in one CTA 11.3).
    const int most_ctas = q.chunks == 1 ? 8 : 1;
    p.chunk_ctas = (in_chunk + 3) / 4 < most_ctas ? (in_chunk + 3) / 4 : most_ctas;
    int warps = (in_chunk + p.chunk_ctas - 1) / p.chunk_ctas;
    warps = warps < 8 ? 8 : warps > kMost ? kMost : warps;
    const size_t key_bytes = (plan_head_words(q.experts) + static_cast<size_t>(warps) * p.key_words) * sizeof(int);
    const size_t smem = plan_smem(q) > key_bytes ? plan_smem(q) : key_bytes;
    auto kernel = route_kernel<BY_LOGIT, VPL>;
    if (int rc = allow_smem(c, variant, reinterpret_cast<const void*>(kernel), smem)) return rc;
    return launch(kernel, q.chunks * p.chunk_ctas, 32 * warps, smem, p.chunk_ctas, stream, name, p, q);
}

template <bool BY_LOGIT>
int launch_route(DeviceCtx* c, const RouteParams& p, const PlanParams& q, cudaStream_t stream, const char* name) {
    constexpr int kFirst = BY_LOGIT ? 76 : 82;
    if (q.experts <= 32) return launch_route<BY_LOGIT, 1>(c, kFirst, p, q, stream, name);
    if (q.experts <= 64) return launch_route<BY_LOGIT, 2>(c, kFirst + 1, p, q, stream, name);
    if (q.experts <= 128) return launch_route<BY_LOGIT, 4>(c, kFirst + 2, p, q, stream, name);
    if (q.experts <= 256) return launch_route<BY_LOGIT, 8>(c, kFirst + 3, p, q, stream, name);
    if (q.experts <= 512) return launch_route<BY_LOGIT, 16>(c, kFirst + 4, p, q, stream, name);
    return launch_route<BY_LOGIT, 32>(c, kFirst + 5, p, q, stream, name);
}

template <int CG, int BT, int STAGES, int EPI_WARPS, int CTAS_PER_SM>
int launch_expert_gemm(DeviceCtx* c, int variant, const ExpertGemmParams& g, long long most_tiles, cudaStream_t stream, const char* name) {
    using S = ExpertSmem<CG, BT, STAGES, EPI_WARPS>;
    auto kernel = expert_gemm_kernel<CG, BT, STAGES, EPI_WARPS, CTAS_PER_SM>;
    if (!c->smem_attr_set[variant]) {
        CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kDynamicBytes));
        c->smem_attr_set[variant] = true;
    }
    long long workers = static_cast<long long>(c->num_sms) * CTAS_PER_SM;
    if (CG == 2) {
        if (c->expert_pairs < 0) {     // pairs that fit the device at once
            cudaLaunchConfig_t cfg;
            std::memset(&cfg, 0, sizeof(cfg));
            cfg.gridDim = dim3(c->num_sms & ~1, 1, 1);
            cfg.blockDim = dim3(S::kThreads, 1, 1);
            cfg.dynamicSmemBytes = S::kDynamicBytes;
            cudaLaunchAttribute attr;
            attr.id = cudaLaunchAttributeClusterDimension;
            attr.val.clusterDim.x = 2;
            attr.val.clusterDim.y = 1;
            attr.val.clusterDim.z = 1;
            cfg.attrs = &attr;
            cfg.numAttrs = 1;
            int n = 0;
            CUDA_TRY(cudaOccupancyMaxActiveClusters(&n, kernel, &cfg));
            c->expert_pairs = n > 0 ? n : 1;
        }
        workers = c->expert_pairs;
    }
    const long long tiles = most_tiles * g.tiles_n;
    if (tiles > 0x7fffffffll) return fail(NVFP4_ERR_INVALID_ARGUMENT, "problem too large: %lld tiles", tiles);
    if (workers > tiles) workers = tiles;
    return launch(kernel, static_cast<unsigned>(workers * CG), S::kThreads, S::kDynamicBytes, CG, stream, name, g);
}

}  // namespace

extern "C" {

int nvfp4_routing_plan(int32_t tokens, int32_t top_k, int32_t experts, int32_t* tile_tokens, int64_t* plan_bytes, int64_t* sf_rows) {
    PlanSizes s;
    if (int rc = plan_sizes(tokens, top_k, experts, &s)) return rc;
    if (tile_tokens) *tile_tokens = s.tile_tokens;
    if (plan_bytes) *plan_bytes = 4 * s.words;
    if (sf_rows) *sf_rows = s.sf_rows;
    return NVFP4_OK;
}

int nvfp4_route(const nvfp4_router* o, const nvfp4_routing* r, void* stream_v) {
    if (!o) return fail(NVFP4_ERR_INVALID_ARGUMENT, "router is NULL");
    PlanSizes s;
    if (int rc = check_routing(r, &s)) return rc;
    if (r->top_k > r->experts) return fail(NVFP4_ERR_INVALID_ARGUMENT, "top_k = %d of %d experts", r->top_k, r->experts);
    if (!r->offset || (r->tokens > 0 && (!r->expert || !r->row || !o->logits || !o->weights)))
        return fail(NVFP4_ERR_INVALID_ARGUMENT, "logits, weights, expert, row and offset must not be NULL");
    if (o->logits_type < NVFP4_LOGITS_FP16 || o->logits_type > NVFP4_LOGITS_FP32)
        return fail(NVFP4_ERR_INVALID_ARGUMENT, "logits_type must be NVFP4_LOGITS_FP16, NVFP4_LOGITS_BF16 or NVFP4_LOGITS_FP32");
    const size_t size = o->logits_type == NVFP4_LOGITS_FP32 ? 4 : 2;
    if (!aligned(o->logits, size) || !aligned(o->bias, 4) || o->logits_row_stride < 0)
        return fail(NVFP4_ERR_INVALID_ARGUMENT, "logits and bias must be aligned to their elements, the row stride must not be negative");
    if (o->scoring != NVFP4_SCORE_SOFTMAX && o->scoring != NVFP4_SCORE_SIGMOID)
        return fail(NVFP4_ERR_INVALID_ARGUMENT, "scoring must be NVFP4_SCORE_SOFTMAX or NVFP4_SCORE_SIGMOID");
    if (o->groups < 1 || o->groups > kMaxGroups || r->experts % o->groups || o->top_groups < 1 || o->top_groups > o->groups)
        return fail(NVFP4_ERR_INVALID_ARGUMENT, "groups must divide the experts and not exceed %d, top_groups must be 1 to groups (got %d of %d groups, %d experts)",
                    kMaxGroups, o->top_groups, o->groups, r->experts);
    if (o->group_top != 1 && o->group_top != 2) return fail(NVFP4_ERR_INVALID_ARGUMENT, "group_top must be 1 or 2");
    if (static_cast<long long>(o->top_groups) * (r->experts / o->groups) < r->top_k)
        return fail(NVFP4_ERR_INVALID_ARGUMENT, "top_k = %d of the %d experts in %d groups", r->top_k, o->top_groups * (r->experts / o->groups), o->top_groups);
    cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
    DeviceCtx* c = nullptr;
    if (int rc = check_device(&c)) return rc;
    const PlanParams q = plan_params(r, s);
    if (r->tokens == 0) return empty_plan(q, stream);
    RouteParams p;
    p.logits = o->logits;
    p.logit_type = o->logits_type;
    p.logits_row_stride = o->logits_row_stride;
    p.bias = o->bias;
    p.scoring = o->scoring;
    p.groups = o->groups; p.top_groups = o->top_groups; p.group_top = o->group_top;
    p.renormalize = o->renormalize ? 1 : 0;
    p.scale = o->scale;
    p.weights = o->weights;
    const int per = r->experts / o->groups;
    p.per_magic = ((1 << 20) + per - 1) / per;
    p.group_lanes = 32;
    while (p.group_lanes * o->groups > 32) p.group_lanes /= 2;
    // the order of the logits is that of the scores where nothing is added to them
    const bool by_logit = !o->bias && (o->groups == 1 || o->group_top == 1);
    if (int rc = by_logit ? launch_route<true>(c, p, q, stream, "route_by_logits") : launch_route<false>(c, p, q, stream, "route_by_scores")) return rc;
    return place(c, q, stream, "route_place");
}

int nvfp4_plan_experts(const nvfp4_routing* r, void* stream_v) {
    PlanSizes s;
    if (int rc = check_routing(r, &s)) return rc;
    if (!r->offset || (r->tokens > 0 && (!r->expert || !r->row))) return fail(NVFP4_ERR_INVALID_ARGUMENT, "expert, row and offset must not be NULL");
    cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
    DeviceCtx* c = nullptr;
    if (int rc = check_device(&c)) return rc;
    PlanParams q = plan_params(r, s);
    if (r->tokens == 0) return empty_plan(q, stream);
    // Without the choice, how many tokens there are does not count: one chunk / more (us) 200 x 6 of 32 3.9 / 4.2, of 256
    // 6.3 / 5.4, 350 x 4 of 32 4.2 / 4.4, 384 x 4 of 64 4.5 / 4.5.
    if (static_cast<long long>(r->tokens) * r->top_k <= (r->experts <= 128 ? 1408 : 1024)) set_chunks(&q, r->tokens, 1);
    const size_t smem = q.chunks > 1 && plan_smem(q) < kPlaceSmem ? kPlaceSmem : plan_smem(q);
    if (int rc = allow_smem(c, 75, reinterpret_cast<const void*>(plan_kernel), smem)) return rc;
    if (int rc = launch(plan_kernel, q.chunks, kPlaceThreads, smem, 1, stream, "plan_experts", q)) return rc;
    return place(c, q, stream, "plan_experts_place");
}

int nvfp4_quantize_routed(const void* x, int32_t x_is_bf16, int64_t x_row_stride, int32_t k, const nvfp4_routing* r, void* packed,
                          int64_t packed_row_stride, void* sf, void* stream_v) {
    PlanSizes s;
    if (int rc = check_routing(r, &s)) return rc;
    if (k < 64 || k % 64) return fail(NVFP4_ERR_INVALID_ARGUMENT, "k must be a positive multiple of 64 (got %d)", k);
    if (r->tokens > 0 && (!x || !packed || !sf || !r->row)) return fail(NVFP4_ERR_INVALID_ARGUMENT, "x, packed, sf and row must not be NULL");
    if (!aligned(x, 16) || x_row_stride % 8 || x_row_stride < 0 || (x_row_stride < k && x_row_stride != 0 && r->tokens > 1))
        return fail(NVFP4_ERR_INVALID_ARGUMENT, "x must be 16-byte aligned with a row stride (elements) that is a multiple of 8 and >= k, or 0");
    if (!aligned(packed, 8) || packed_row_stride % 8 || packed_row_stride < k / 2 || !aligned(sf, 16))
        return fail(NVFP4_ERR_INVALID_ARGUMENT, "packed must be 8-byte aligned with a row stride that is a multiple of 8 and >= k/2, sf 16-byte aligned");
    DeviceCtx* c = nullptr;
    if (int rc = check_device(&c)) return rc;
    if (r->tokens == 0) return NVFP4_OK;
    const PlanParams q = plan_params(r, s);
    QuantizeRoutedParams p;
    p.x = static_cast<const uint8_t*>(x);
    p.packed = static_cast<uint8_t*>(packed);
    p.sf = static_cast<uint8_t*>(sf);
    p.row = q.row; p.sf_row = q.sf_row;
    p.tokens = r->tokens; p.top_k = r->top_k; p.k = k;
    p.rows = r->tokens * r->top_k; p.sf_rows = static_cast<int>(s.sf_rows);
    p.x_row_stride = 2 * x_row_stride; p.packed_row_stride = packed_row_stride;
    const long long units = static_cast<long long>(r->tokens) * ((k + kRoutedCols - 1) / kRoutedCols);
    const long long grid = (units + 7) / 8;
    if (grid > 0x7fffffffll) return fail(NVFP4_ERR_INVALID_ARGUMENT, "problem too large: %lld work units", units);
    const bool wide = aligned(x, 32) && x_row_stride % 16 == 0;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
    auto go = [&](auto kernel) { return launch(kernel, static_cast<unsigned>(grid), 256, 0, 1, stream, "quantize_routed", p); };
    if (x_is_bf16) return wide ? go(quantize_routed_kernel<true, true>) : go(quantize_routed_kernel<true, false>);
    return wide ? go(quantize_routed_kernel<false, true>) : go(quantize_routed_kernel<false, false>);
}

int nvfp4_expert_gemm(const nvfp4_expert_problem* p, const nvfp4_routing* r, void* stream_v) {
    if (!p) return fail(NVFP4_ERR_INVALID_ARGUMENT, "problem is NULL");
    PlanSizes s;
    if (int rc = check_routing(r, &s)) return rc;
    if (p->n < 128 || p->n % 128) return fail(NVFP4_ERR_INVALID_ARGUMENT, "n must be a positive multiple of 128 (got %d)", p->n);
    if (p->k < kKPerStage || p->k % kKPerStage) return fail(NVFP4_ERR_INVALID_ARGUMENT, "k must be a positive multiple of 256 (got %d)", p->k);
    if (p->activation < NVFP4_ACT_NONE || p->activation > NVFP4_ACT_SWIGLU)
        return fail(NVFP4_ERR_INVALID_ARGUMENT, "activation must be NVFP4_ACT_NONE, NVFP4_ACT_RELU, NVFP4_ACT_SILU or NVFP4_ACT_SWIGLU");
    if (p->output != NVFP4_OUT_FP16 && p->output != NVFP4_OUT_NVFP4)
        return fail(NVFP4_ERR_INVALID_ARGUMENT, "output must be NVFP4_OUT_FP16 or NVFP4_OUT_NVFP4");
    const bool to_nvfp4 = p->output == NVFP4_OUT_NVFP4;
    if (!p->w || !p->sfw_perm || (r->tokens > 0 && (!p->a || !p->sfa || !p->out || (to_nvfp4 && !p->out_sf))))
        return fail(NVFP4_ERR_INVALID_ARGUMENT, "a, sfa, w, sfw_perm, out (and out_sf for NVFP4 output) must not be NULL");
    if (!aligned(p->a, 16) || !aligned(p->sfa, 16) || !aligned(p->w, 16) || !aligned(p->sfw_perm, 16) || !aligned(p->out, 16) || !aligned(p->out_sf, 16) ||
        !aligned(p->alpha, 4) || !aligned(p->bias, 2))
        return fail(NVFP4_ERR_INVALID_ARGUMENT, "operands, scales and outputs must be 16-byte aligned, alpha and bias to their elements");
    const int n_out = p->activation == NVFP4_ACT_SWIGLU ? p->n / 2 : p->n;
    if (p->a_row_stride % 16 || p->w_row_stride % 16 || p->a_row_stride < p->k / 2 || p->w_row_stride < p->k / 2)
        return fail(NVFP4_ERR_INVALID_ARGUMENT, "row strides of a and w must be multiples of 16 bytes and >= k/2");
    // (the bias may be one for all; weights that several experts share cannot be described to tensor loads)
    if (r->experts > 1 && (p->w_expert_stride % 16 || p->sfw_perm_expert_stride % 16 || p->w_expert_stride < p->k / 2 || p->sfw_perm_expert_stride < 512 ||
                           (p->bias && p->bias_expert_stride < 0)))
        return fail(NVFP4_ERR_INVALID_ARGUMENT, "expert strides must keep 16-byte alignment and the experts' weights and scales apart, the bias's must not be negative");
    if (to_nvfp4 ? (p->out_row_stride % 16 || p->out_row_stride < n_out / 2) : (p->out_row_stride % 8 || p->out_row_stride < n_out))
        return fail(NVFP4_ERR_INVALID_ARGUMENT, "out_row_stride must keep 16-byte alignment and hold a row");
    DeviceCtx* c = nullptr;
    if (int rc = check_device(&c)) return rc;
    if (r->tokens == 0) return NVFP4_OK;
    const PlanParams q = plan_params(r, s);
    ExpertGemmParams g;
    std::memset(&g, 0, sizeof(g));
    const uint64_t kbytes = static_cast<uint64_t>(p->k) / 2;
    const uint64_t rows = static_cast<uint64_t>(r->tokens) * r->top_k;
    const uint64_t w_es = r->experts > 1 ? static_cast<uint64_t>(p->w_expert_stride) : static_cast<uint64_t>(p->w_row_stride) * p->n;
    if (int rc = encode_map(make_key(p->w, kbytes, p->n, r->experts, p->w_row_stride, w_es, kBKBytes, kBM, CU_TENSOR_MAP_DATA_TYPE_UINT8), &g.tma_w)) return rc;
    if (int rc = encode_map(make_sf_key(p->sfw_perm, p->n, p->k, r->experts, p->sfw_perm_expert_stride, 1), &g.tma_sfw)) return rc;
    for (int i = 0; i < 4; ++i)
        if (int rc = encode_map(make_key(p->a, kbytes, rows, 1, p->a_row_stride, static_cast<uint64_t>(p->a_row_stride) * rows, kBKBytes, 16u << i,
                                         CU_TENSOR_MAP_DATA_TYPE_UINT8), &g.tma_x[i])) return rc;
    for (int i = 0; i < 2; ++i)
        if (int rc = encode_map(make_sf_key(p->sfa, static_cast<int>(s.sf_rows), p->k, 1, 0, i + 1), &g.tma_sfx[i])) return rc;
    g.tiles = q.tiles;
    g.tile_count = q.tile_count;
    g.alpha = p->alpha;
    g.bias = static_cast<const __half*>(p->bias);
    g.bias_stride = p->bias_expert_stride;
    g.activation = p->activation;
    g.out_scale = p->out_scale;
    g.out_nvfp4 = to_nvfp4 ? 1 : 0;
    if (to_nvfp4) {
        g.out_packed = static_cast<uint8_t*>(p->out);
        g.out_packed_row_stride = p->out_row_stride;
        g.out_sf = static_cast<uint8_t*>(p->out_sf);
    } else {
        g.c = static_cast<__half*>(p->out);
        g.c_row_stride = p->out_row_stride;
    }
    g.n = p->n; g.n_out = n_out;
    g.experts = r->experts;
    g.rows = static_cast<int>(rows);
    g.most_tiles = static_cast<int>(s.max_tiles);
    g.k_tiles = p->k / kKPerStage;
    g.status = c->status_dev;
    g.timeout_cycles = g_timeout_ns.load() * 2;   // SM clock <= 2 GHz: at least the requested time
    cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
    if (s.tile_tokens == kTileFew) {
        g.tiles_n = p->n / kBM;
        return launch_expert_gemm<1, kTileFew, 4, 4, 2>(c, 72, g, s.max_tiles, stream, "expert_gemm_t32");
    }
    g.tiles_n = (p->n + 2 * kBM - 1) / (2 * kBM);
    return launch_expert_gemm<2, kTileMany, 5, 8, 1>(c, 73, g, s.max_tiles, stream, "expert_gemm_2cta_t256");
}

int nvfp4_combine_experts(const void* y, int64_t y_row_stride, int32_t y_rows, const int32_t* row, const float* weights, int32_t tokens, int32_t top_k,
                          int32_t n, const void* residual, int64_t residual_row_stride, void* out, int64_t out_row_stride, int32_t out_is_bf16,
                          void* stream_v) {
    if (tokens < 0 || top_k < 1 || top_k > kMaxTopK || n < 8 || n % 8 || y_rows < 0)
        return fail(NVFP4_ERR_INVALID_ARGUMENT, "n must be a positive multiple of 8, top_k 1 to %d, tokens and y_rows not negative (got %d, %d, %d, %d)", kMaxTopK, n,
                    top_k, tokens, y_rows);
    if (tokens == 0) return NVFP4_OK;
    if (!row || !weights || !out || (!y && y_rows > 0)) return fail(NVFP4_ERR_INVALID_ARGUMENT, "y, row, weights and out must not be NULL");
    if (!aligned(y, 16) || !aligned(residual, 16) || !aligned(out, 16) || !aligned(row, 4) || !aligned(weights, 4) || y_row_stride % 8 ||
        residual_row_stride % 8 || out_row_stride % 8 || y_row_stride < 0 || residual_row_stride < 0 || (tokens > 1 && out_row_stride < n))
        return fail(NVFP4_ERR_INVALID_ARGUMENT, "y, residual and out must be 16-byte aligned with row strides that keep that, out's at least n");
    DeviceCtx* c = nullptr;
    if (int rc = check_device(&c)) return rc;
    CombineParams p;
    p.y = static_cast<const __half*>(y);
    p.rows = row;
    p.weights = weights;
    p.residual = static_cast<const uint8_t*>(residual);
    p.out = static_cast<uint8_t*>(out);
    p.y_row_stride = y_row_stride; p.residual_row_stride = residual_row_stride; p.out_row_stride = out_row_stride;
    p.y_rows = y_rows; p.tokens = tokens; p.top_k = top_k; p.n = n;
    const long long grid = (static_cast<long long>(tokens) * (n / 8) + 255) / 256;
    if (grid > 0x7fffffffll) return fail(NVFP4_ERR_INVALID_ARGUMENT, "problem too large: %lld CTAs", grid);
    cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
    auto go = [&](auto kernel) { return launch(kernel, static_cast<unsigned>(grid), 256, 0, 1, stream, "combine_experts", p); };
    if (out_is_bf16) return top_k <= 2 ? go(combine_kernel<true, 2>) : top_k <= 4 ? go(combine_kernel<true, 4>) : go(combine_kernel<true, 8>);
    return top_k <= 2 ? go(combine_kernel<false, 2>) : top_k <= 4 ? go(combine_kernel<false, 4>) : go(combine_kernel<false, 8>);
}

}  // extern "C"
