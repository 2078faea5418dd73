// Routing to experts, and the two data movements around the experts' products:
//   * route: router logits -> the experts of every token, their weights, and the plan;
//   * plan: the stable order of all (token, choice) pairs by expert: each pair's row in that order, the
//     experts' first rows, and the table of token tiles that the grouped product walks;
//   * quantize_routed: token rows -> NVFP4 rows in expert order, with the scales in the atoms of each tile;
//   * combine: rows in expert order -> weighted sum per token plus residual.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "ptx.cuh"
#include "quantize.cuh"

namespace nvfp4 {

constexpr int kMaxExperts = 1024, kMaxTopK = 32, kMaxGroups = 32;
constexpr int kPlanPairs = 256;      // pairs ranked at a time: a word of bits per 32 of them and expert
constexpr int kPlanWords = kPlanPairs / 32;

enum Scoring : int { kScoreSoftmax = 0, kScoreSigmoid = 1 };
enum LogitType : int { kLogitFp16 = 0, kLogitBf16 = 1, kLogitFp32 = 2 };

struct RouteParams {
    const void* logits;
    int logit_type;
    long long logits_row_stride;   // elements
    const float* bias;             // [experts] or null
    int scoring, groups, top_groups, group_top;   // group_top: how many of a group's best choices make its score, 1 or 2
    int renormalize;
    float scale;
    float* weights;                // [tokens][top_k]
};
// The plan's memory.  `plan` words: tile count, 3 unused, tiles {expert, first row, rows, 0}, scale rows [tokens][top_k],
// counts [chunks][experts].
struct PlanParams {
    int tokens, top_k, experts, tile_tokens, tile_sf_rows;
    int chunk_tokens, chunks;
    int* expert;      // [tokens][top_k]
    int* row;         // [tokens][top_k]
    int* offset;      // [experts + 1]
    int* tile_count;
    int4* tiles;
    int* sf_row;      // [tokens][top_k]
    int* counts;
};

// ------------------------------------------------------------------------------------------------ choice
// Order-preserving unsigned keys; 0 is below every number.
__device__ __forceinline__ uint32_t key_of(float v) {
    const uint32_t b = __float_as_uint(v + 0.f);   // (-0 becomes +0)
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t key_of(double v) {
    const uint64_t b = static_cast<uint64_t>(__double_as_longlong(v + 0.0));
    return b >> 63 ? ~b : b | 0x8000000000000000ull;
}
__device__ __forceinline__ double value_of(uint64_t key) {
    return __longlong_as_double(static_cast<long long>(key >> 63 ? key & 0x7fffffffffffffffull : ~key));
}
// Largest key of the warp; lanes that do not hold it get the same value.
__device__ __forceinline__ uint32_t warp_max(uint32_t k) { return __reduce_max_sync(0xffffffffu, k); }
__device__ __forceinline__ uint64_t warp_max(uint64_t k) {
    const uint32_t hi = static_cast<uint32_t>(k >> 32);
    const uint32_t top = __reduce_max_sync(0xffffffffu, hi);
    const uint32_t lo = __reduce_max_sync(0xffffffffu, hi == top ? static_cast<uint32_t>(k) : 0u);
    return static_cast<uint64_t>(top) << 32 | lo;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int s = 16; s; s >>= 1) v += __shfl_xor_sync(0xffffffffu, v, s);
    return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int s = 16; s; s >>= 1) v += __shfl_xor_sync(0xffffffffu, v, s);
    return v;
}

// A logit as the router sees it: NaN and -inf mark an expert that cannot be chosen, +inf counts as the largest number.
__device__ __forceinline__ float load_logit(const RouteParams& p, long long at) {
    float x;
    if (p.logit_type == kLogitFp32) x = static_cast<const float*>(p.logits)[at];
    else if (p.logit_type == kLogitBf16) x = __bfloat162float(static_cast<const __nv_bfloat16*>(p.logits)[at]);
    else x = __half2float(static_cast<const __half*>(p.logits)[at]);
    return x != x ? -INFINITY : fminf(x, 3.402823466e38f);
}

// The choice of one token by one warp: lane holds experts lane, lane + 32, ...  Slot j's expert and weight end
// in lane j.  Key: uint32_t where the order of the logits is the order of the choice (no bias, and groups judged by
// their best), else uint64_t, the choice score in 64 bits: two scores may be nearer to each other than 32 bits
// show, and the experts that are taken must not depend on it.
template <typename Key, int VPL>
__device__ __forceinline__ void choose(const RouteParams& p, const PlanParams& q, long long token, int lane, Key* group_keys, int& expert,
                                       float& weight) {
    constexpr bool kByLogit = sizeof(Key) == 4;
    float x[VPL];
    Key key[VPL];
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
        const int e = i * 32 + lane;
        x[i] = e < q.experts ? load_logit(p, token * p.logits_row_stride + e) : -INFINITY;
        top = fmaxf(top, x[i]);
    }
    double total = 0.0;    // softmax: sum of exp(x - top)
    if (p.scoring == kScoreSoftmax) {
        const uint32_t t = warp_max(key_of(top));
        top = __uint_as_float(t & 0x80000000u ? t & 0x7fffffffu : ~t);
        if constexpr (kByLogit) {
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < VPL; ++i) sum += x[i] == -INFINITY ? 0.f : expf(x[i] - top);
            total = warp_sum(sum);
        } else {
#pragma unroll
            for (int i = 0; i < VPL; ++i) total += x[i] == -INFINITY ? 0.0 : exp(static_cast<double>(x[i]) - top);
            total = warp_sum(total);
        }
    }
    auto score = [&](float v) {
        return p.scoring == kScoreSoftmax ? exp(static_cast<double>(v) - top) / total : 1.0 / (1.0 + exp(-static_cast<double>(v)));
    };
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
        const int e = i * 32 + lane;
        if constexpr (kByLogit) {
            key[i] = x[i] == -INFINITY ? 0u : key_of(x[i]);
        } else {
            double c = -INFINITY;
            if (x[i] != -INFINITY) c = score(x[i]) + (p.bias ? static_cast<double>(p.bias[e]) : 0.0);
            key[i] = c == c && c != -INFINITY ? key_of(c) : 0ull;     // (a bias of -inf or NaN masks its expert too)
        }
    }
    if (p.groups > 1) {
        // keys to shared memory; lane g judges group g and the warp takes the best top_groups of them
        __syncwarp();
#pragma unroll
        for (int i = 0; i < VPL; ++i)
            if (i * 32 + lane < q.experts) group_keys[i * 32 + lane] = key[i];
        __syncwarp();
        const int per = q.experts / p.groups;
        Key mine = 0;
        if (lane < p.groups) {
            Key first = 0, second = 0;
            for (int i = 0; i < per; ++i) {
                const Key k = group_keys[lane * per + i];
                if (k > first) { second = first; first = k; }
                else if (k > second) second = k;
            }
            mine = first;
            if constexpr (!kByLogit)
                if (p.group_top == 2 && second) mine = key_of(value_of(first) + value_of(second));
        }
        uint32_t kept = 0;
        for (int g = 0; g < p.top_groups; ++g) {
            const Key best = warp_max(mine);
            if (best == 0) break;
            const int at = __ffs(__ballot_sync(0xffffffffu, mine == best)) - 1;
            kept |= 1u << at;
            if (lane == at) mine = 0;
        }
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            const int e = i * 32 + lane;
            if (e < q.experts && !(kept >> (e / per) & 1u)) key[i] = 0;
        }
    }
    expert = -1;
    float logit = 0.f;
    for (int j = 0; j < q.top_k; ++j) {
        Key best = key[0];
        int at = 0;
#pragma unroll
        for (int i = 1; i < VPL; ++i)
            if (key[i] > best) { best = key[i]; at = i; }
        const Key top_key = warp_max(best);
        if (top_key == 0) break;
        // ties: the lowest index, over all lanes
        const uint32_t e = __reduce_min_sync(0xffffffffu, best == top_key ? static_cast<uint32_t>(at * 32 + lane) : 0xffffffffu);
        const int owner = e & 31, slot = e >> 5;
        float l = 0.f;
#pragma unroll
        for (int i = 0; i < VPL; ++i)
            if (i == slot) {
                l = x[i];
                if (lane == owner) key[i] = 0;
            }
        l = __shfl_sync(0xffffffffu, l, owner);
        if (lane == j) { expert = static_cast<int>(e); logit = l; }
    }
    double s = expert >= 0 ? score(logit) : 0.0;
    if (p.renormalize) {
        const double sum = warp_sum(s);
        s = sum > 0.0 ? s / sum : 0.0;
    }
    weight = static_cast<float>(s * p.scale);
}

// -------------------------------------------------------------------------------------------------- plan
// Exclusive sums over the experts of a CTA: first row and first tile of each.  count[e] in, row0[e] / tile0[e] out
// (both of experts + 1 entries); all threads of the CTA take part.  scratch: 2 x 32 words.
__device__ __forceinline__ void scan_experts(const int* count, int* row0, int* tile0, int experts, int tile_tokens, int* scratch) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    int carry_r = 0, carry_t = 0;
    for (int base = 0; base < experts; base += blockDim.x) {
        const int e = base + threadIdx.x;
        const int c = e < experts ? count[e] : 0;
        int r = c, t = (c + tile_tokens - 1) / tile_tokens;
        const int t_own = t;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
            const int a = __shfl_up_sync(0xffffffffu, r, s), b = __shfl_up_sync(0xffffffffu, t, s);
            if (lane >= s) { r += a; t += b; }
        }
        if (lane == 31) { scratch[warp] = r; scratch[32 + warp] = t; }
        __syncthreads();
        int before_r = carry_r, before_t = carry_t;
        for (int w = 0; w < warps; ++w) {
            if (w < warp) { before_r += scratch[w]; before_t += scratch[32 + w]; }
            carry_r += scratch[w];
            carry_t += scratch[32 + w];
        }
        if (e < experts) { row0[e] = before_r + r - c; tile0[e] = before_t + t - t_own; }
        __syncthreads();
    }
    if (threadIdx.x == 0) { row0[experts] = carry_r; tile0[experts] = carry_t; }
    __syncthreads();
}

// Rows of a chunk's pairs.  next[e]: how many pairs of expert e stand before the chunk (changed here); bits: experts x kPlanWords words.
// Pairs are ranked kPlanPairs at a time by a bit per pair and expert, so that the order is that of the pairs whichever
// thread comes first, and the same expert twice in a token gets two rows.
__device__ __forceinline__ void place_pairs(const PlanParams& q, long long first_pair, int pairs, const int* row0, const int* tile0, int* next,
                                            uint32_t* bits) {
    for (int base = 0; base < pairs; base += kPlanPairs) {
        for (int i = threadIdx.x; i < q.experts * kPlanWords; i += blockDim.x) bits[i] = 0u;
        __syncthreads();
        const int here = min(kPlanPairs, pairs - base);
        for (int i = threadIdx.x; i < here; i += blockDim.x) {
            const int e = q.expert[first_pair + base + i];
            if (e >= 0 && e < q.experts) atomicOr(&bits[e * kPlanWords + (i >> 5)], 1u << (i & 31));
        }
        __syncthreads();
        for (int i = threadIdx.x; i < here; i += blockDim.x) {
            const int e = q.expert[first_pair + base + i];
            int row = -1, sf_row = -1;
            if (e >= 0 && e < q.experts) {
                int rank = next[e];
#pragma unroll
                for (int w = 0; w < kPlanWords; ++w) {
                    const uint32_t b = bits[e * kPlanWords + w];
                    rank += w < (i >> 5) ? __popc(b) : w == (i >> 5) ? __popc(b & ((1u << (i & 31)) - 1u)) : 0;
                }
                row = row0[e] + rank;
                sf_row = (tile0[e] + rank / q.tile_tokens) * q.tile_sf_rows + rank % q.tile_tokens;
            }
            q.row[first_pair + base + i] = row;
            q.sf_row[first_pair + base + i] = sf_row;
        }
        __syncthreads();
        for (int e = threadIdx.x; e < q.experts; e += blockDim.x) {
            int n = 0;
#pragma unroll
            for (int w = 0; w < kPlanWords; ++w) n += __popc(bits[e * kPlanWords + w]);
            next[e] += n;
        }
        __syncthreads();
    }
}

// offsets and the tile table, by the threads of one CTA (all of them look at row0 / tile0 of shared memory)
__device__ __forceinline__ void write_tables(const PlanParams& q, const int* row0, const int* tile0) {
    for (int e = threadIdx.x; e <= q.experts; e += blockDim.x) q.offset[e] = row0[e];
    if (threadIdx.x == 0) *q.tile_count = tile0[q.experts];
    for (int e = threadIdx.x; e < q.experts; e += blockDim.x)
        for (int r = row0[e], t = tile0[e]; r < row0[e + 1]; r += q.tile_tokens, ++t)
            q.tiles[t] = make_int4(e, r, min(q.tile_tokens, row0[e + 1] - r), 0);
}

// Shared memory of the plan: counts / next [experts], row0 and tile0 [experts + 1], scan scratch, bits.
__host__ __device__ constexpr int plan_smem_words(int experts) { return 3 * (experts + 1) + 64 + experts * kPlanWords; }

// One chunk's share of the order, where the counts of all chunks are known.  Every CTA adds up the counts of all
// chunks for itself (at most 160 x experts words from L2) instead of a launch between.
__global__ void __launch_bounds__(512) place_kernel(const PlanParams q) {
    extern __shared__ __align__(16) int plan_smem[];
    int* next = plan_smem;
    int* row0 = next + q.experts + 1;
    int* tile0 = row0 + q.experts + 1;
    int* scratch = tile0 + q.experts + 1;
    uint32_t* bits = reinterpret_cast<uint32_t*>(scratch + 64);
    ptx::grid_dependency_launch_dependents();
    ptx::grid_dependency_wait();
    const int chunk = blockIdx.x;
    // (row0 holds the totals until the scan has read them: count and result of an expert belong to one thread)
    for (int e = threadIdx.x; e < q.experts; e += blockDim.x) {
        int before = 0, all = 0;
#pragma unroll 8
        for (int c = 0; c < q.chunks; ++c) {
            const int n = q.counts[static_cast<long long>(c) * q.experts + e];
            before += c < chunk ? n : 0;
            all += n;
        }
        next[e] = before;
        row0[e] = all;
    }
    __syncthreads();
    scan_experts(row0, row0, tile0, q.experts, q.tile_tokens, scratch);
    if (chunk == 0) write_tables(q, row0, tile0);
    const long long first = static_cast<long long>(chunk) * q.chunk_tokens;
    const int tokens = static_cast<int>(min(static_cast<long long>(q.chunk_tokens), q.tokens - first));
    place_pairs(q, first * q.top_k, tokens * q.top_k, row0, tile0, next, bits);
}

// The rest of a CTA that knows its chunk's experts (in global memory, written by this CTA or given): the counts of
// the chunk, or everything where the chunk is the only one.
__device__ __forceinline__ void count_and_place(const PlanParams& q, int chunk, int* smem) {
    int* next = smem;
    int* row0 = next + q.experts + 1;
    int* tile0 = row0 + q.experts + 1;
    int* scratch = tile0 + q.experts + 1;
    uint32_t* bits = reinterpret_cast<uint32_t*>(scratch + 64);
    for (int e = threadIdx.x; e < q.experts; e += blockDim.x) row0[e] = 0;
    __syncthreads();
    const long long first = static_cast<long long>(chunk) * q.chunk_tokens;
    const int pairs = static_cast<int>(min(static_cast<long long>(q.chunk_tokens), q.tokens - first)) * q.top_k;
    for (int i = threadIdx.x; i < pairs; i += blockDim.x) {
        const int e = q.expert[first * q.top_k + i];
        if (e >= 0 && e < q.experts) atomicAdd(&row0[e], 1);
    }
    __syncthreads();
    if (q.chunks > 1) {
        for (int e = threadIdx.x; e < q.experts; e += blockDim.x) q.counts[static_cast<long long>(chunk) * q.experts + e] = row0[e];
        return;
    }
    for (int e = threadIdx.x; e < q.experts; e += blockDim.x) next[e] = 0;
    scan_experts(row0, row0, tile0, q.experts, q.tile_tokens, scratch);
    write_tables(q, row0, tile0);
    place_pairs(q, 0, pairs, row0, tile0, next, bits);
}

__global__ void __launch_bounds__(512) plan_kernel(const PlanParams q) {
    extern __shared__ __align__(16) int plan_smem[];
    ptx::grid_dependency_launch_dependents();
    ptx::grid_dependency_wait();
    count_and_place(q, blockIdx.x, plan_smem);
}

// A warp per token, a chunk of tokens per CTA.  Shared memory: the plan's, or before that a row of keys per warp for the groups.
template <typename Key, int VPL>
__global__ void __launch_bounds__(512) route_kernel(const RouteParams p, const PlanParams q) {
    extern __shared__ __align__(16) int plan_smem[];
    ptx::grid_dependency_launch_dependents();
    ptx::grid_dependency_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    Key* group_keys = reinterpret_cast<Key*>(plan_smem) + warp * q.experts;
    const long long first = static_cast<long long>(blockIdx.x) * q.chunk_tokens;
    const int tokens = static_cast<int>(min(static_cast<long long>(q.chunk_tokens), q.tokens - first));
    for (int t = warp; t < tokens; t += warps) {
        int expert;
        float weight;
        choose<Key, VPL>(p, q, first + t, lane, group_keys, expert, weight);
        if (lane < q.top_k) {
            q.expert[(first + t) * q.top_k + lane] = expert;
            p.weights[(first + t) * q.top_k + lane] = weight;
        }
    }
    __syncthreads();     // (the experts that the other threads wrote are read back from global memory by this CTA)
    count_and_place(q, blockIdx.x, plan_smem);
}

// ------------------------------------------------------------------------------------------ routed quantiser
struct QuantizeRoutedParams {
    const uint8_t* x;
    uint8_t* packed;
    uint8_t* sf;             // atoms [scale rows / 128][k / 64][512]
    const int* row;          // [tokens][top_k]
    const int* sf_row;
    int tokens, top_k, k;
    long long x_row_stride, packed_row_stride;   // bytes
};

constexpr int kRoutedCols = 512;     // columns per warp
// A lane takes one scale block (16 elements, 32 bytes) of a token, a warp 512 columns; the codes and scales, made once, are
// stored in each of the token's rows.
template <bool BF16, bool kWide>
__global__ void __launch_bounds__(256) quantize_routed_kernel(const QuantizeRoutedParams p) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int blocks = p.k / 16;
    const unsigned col_units = (p.k + kRoutedCols - 1) / kRoutedCols;
    const long long unit = static_cast<long long>(blockIdx.x) * 8 + warp;
    const long long token = unit / col_units;
    const int blk = static_cast<int>(unit - token * col_units) * (kRoutedCols / 16) + lane;
    ptx::grid_dependency_launch_dependents();
    ptx::grid_dependency_wait();
    if (token >= p.tokens) return;
    const bool in_row = blk < blocks;
    int row = -1, sf_row = -1;
    if (lane < p.top_k) { row = p.row[token * p.top_k + lane]; sf_row = p.sf_row[token * p.top_k + lane]; }
    uint32_t codes[2] = {0u, 0u}, scales = 0u;
    if (in_row) {
        uint32_t w[8];
        load_block16<kWide>(p.x + token * p.x_row_stride + blk * 32ll, w);
        scales = quantize_words<BF16>(w, codes) << (8 * (lane & 3));
    }
    scales |= __shfl_xor_sync(0xffffffffu, scales, 1);
    scales |= __shfl_xor_sync(0xffffffffu, scales, 2);
    for (int j = 0; j < p.top_k; ++j) {
        const int r = __shfl_sync(0xffffffffu, row, j), s = __shfl_sync(0xffffffffu, sf_row, j);
        if (r < 0 || !in_row) continue;
        *reinterpret_cast<uint2*>(p.packed + r * p.packed_row_stride + blk * 8) = make_uint2(codes[0], codes[1]);
        if ((lane & 3) == 0)
            *reinterpret_cast<uint32_t*>(p.sf + (static_cast<long long>(s / 128) * (blocks / 4) + blk / 4) * 512 + (s % 32) * 16 + (s % 128) / 32 * 4) = scales;
    }
}

// ------------------------------------------------------------------------------------------------- combine
struct CombineParams {
    const __half* y;
    const int* rows;          // [tokens][top_k]
    const float* weights;     // [tokens][top_k]
    const uint8_t* residual;  // or null
    uint8_t* out;
    long long y_row_stride, residual_row_stride, out_row_stride;   // elements
    int y_rows, tokens, top_k, n;
};
template <bool BF16>
__device__ __forceinline__ float2 to_float2(uint32_t w) {
    if (BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <bool BF16>
__device__ __forceinline__ uint32_t from_float2(float a, float b) {
    if (BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// A thread takes eight columns (16 bytes) of a token; the rows are added in the order of the choices, in fp32.
template <bool BF16>
__global__ void __launch_bounds__(256) combine_kernel(const CombineParams p) {
    const unsigned vecs = p.n / 8;
    ptx::grid_dependency_launch_dependents();
    ptx::grid_dependency_wait();
    const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
    const long long token = i / vecs;
    if (token >= p.tokens) return;
    const long long col = (i - token * vecs) * 8;
    float s[8] = {};
    const int* rows = p.rows + token * p.top_k;
    const float* weights = p.weights + token * p.top_k;
    for (int j0 = 0; j0 < p.top_k; j0 += 8) {
        uint4 v[8];
        float w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            w[j] = 0.f;
            v[j] = make_uint4(0u, 0u, 0u, 0u);
            if (j0 + j < p.top_k) {
                const int r = rows[j0 + j];
                if (r >= 0 && r < p.y_rows) {
                    w[j] = weights[j0 + j];
                    v[j] = __ldcs(reinterpret_cast<const uint4*>(p.y + r * p.y_row_stride + col));
                }
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t q[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 f = to_float2<false>(q[e]);
                s[2 * e] = fmaf(w[j], f.x, s[2 * e]);
                s[2 * e + 1] = fmaf(w[j], f.y, s[2 * e + 1]);
            }
        }
    }
    if (p.residual) {
        const uint4 v = __ldcs(reinterpret_cast<const uint4*>(p.residual + (token * p.residual_row_stride + col) * 2));
        const uint32_t q[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 f = to_float2<BF16>(q[e]);
            s[2 * e] += f.x;
            s[2 * e + 1] += f.y;
        }
    }
    uint32_t o[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = from_float2<BF16>(s[2 * e], s[2 * e + 1]);
    *reinterpret_cast<uint4*>(p.out + (token * p.out_row_stride + col) * 2) = make_uint4(o[0], o[1], o[2], o[3]);
}

}  // namespace nvfp4
