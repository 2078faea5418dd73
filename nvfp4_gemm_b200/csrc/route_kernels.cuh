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
    int chunk_ctas;                // CTAs (a cluster) that share a chunk
    int key_words;                 // shared memory of a warp, a multiple of 4
    int per_magic;                 // e * per_magic >> 20 is the group of expert e < 1024
    int group_lanes;               // lanes that judge a group: 32 / groups, rounded down to a power of two
    int direct_lanes;              // lanes whose experts are just a group's (a power of two), or 0
    int vector;                    // a lane's logits can be read in pieces of 16 bytes, or as much as it has
};
// Counts of a chunk: 16 bits an expert, whole 32-byte sectors.
__host__ __device__ constexpr int counts_row(int experts) { return (experts + 15) & ~15; }
constexpr int kMaxChunkPairs = 65535;
constexpr int kPlaceThreads = 512;

// The plan's memory: the word of the tile count, 3 unused, tiles {expert, first row, rows, 0}, the chunks' counts, scale rows [tokens][top_k].
struct PlanParams {
    int tokens, top_k, experts;
    int tile_tokens, tile_shift, tile_sf_rows;     // rows of a tile (a power of two, and which), of its scales
    int chunk_tokens, chunks;
    int bit_words;    // words of bits per expert: pairs are ranked 32 times as many at a time
    int* expert;      // [tokens][top_k]
    int* row;         // [tokens][top_k]
    int* offset;      // [experts + 1]
    int* tile_count;
    int4* tiles;
    int* sf_row;      // [tokens][top_k]
    uint16_t* counts; // [chunks][counts_row(experts)]
};

// ------------------------------------------------------------------------------------------------ choice
// Order-preserving unsigned keys.  0 is what cannot be chosen: the 32-bit keys are counted from that of -inf.
constexpr uint32_t kLowestKey = 0x007fffffu;
__device__ __forceinline__ uint32_t key_of(float v) {
    const uint32_t b = __float_as_uint(v + 0.f);   // (-0 becomes +0)
    return (b & 0x80000000u ? ~b : b | 0x80000000u) - kLowestKey;
}
__device__ __forceinline__ uint64_t key_of(double v) {
    const uint64_t b = static_cast<uint64_t>(__double_as_longlong(v + 0.0));
    return b >> 63 ? ~b : b | 0x8000000000000000ull;
}
__device__ __forceinline__ double value_of(uint64_t key) {
    return __longlong_as_double(static_cast<long long>(key >> 63 ? key & 0x7fffffffffffffffull : ~key));
}
__device__ __forceinline__ float value_of(uint32_t key) {
    key += kLowestKey;
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
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
__device__ __forceinline__ float as_logit(float x) { return fminf(fmaxf(x, -INFINITY), 3.402823466e38f); }      // (the larger of NaN and a number is the number)
__device__ __forceinline__ float load_logit(const RouteParams& p, long long at) {
    if (p.logit_type == kLogitFp32) return as_logit(static_cast<const float*>(p.logits)[at]);
    if (p.logit_type == kLogitBf16) return as_logit(__bfloat162float(static_cast<const __nv_bfloat16*>(p.logits)[at]));
    return as_logit(__half2float(static_cast<const __half*>(p.logits)[at]));
}
// A lane's logits of a token, experts lane * VPL and on, as they stand in memory (all loads on their way together: with a look at
// the type at each, one load waited for the other), and as numbers.
template <int VPL>
__device__ __forceinline__ void load_raw(const RouteParams& p, long long at, int lane, int experts, uint32_t (&raw)[VPL]) {
    const int e0 = lane * VPL;
    const bool vector = p.vector && e0 + VPL <= experts;       // (whole 16-byte pieces, or all that the lane has)
    if (p.logit_type == kLogitFp32) {
        const uint32_t* src = static_cast<const uint32_t*>(p.logits) + at + e0;
        if (VPL >= 4 && vector) {
#pragma unroll
            for (int j = 0; j < VPL / 4; ++j) {
                const uint4 v = reinterpret_cast<const uint4*>(src)[j];
                raw[4 * j] = v.x; raw[4 * j + 1] = v.y; raw[4 * j + 2] = v.z; raw[4 * j + 3] = v.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < VPL; ++i) raw[i] = e0 + i < experts ? src[i] : 0u;
        }
    } else {
        const uint16_t* src = static_cast<const uint16_t*>(p.logits) + at + e0;
        if (VPL >= 2 && vector) {
            uint32_t w[VPL / 2 ? VPL / 2 : 1];
            if constexpr (VPL >= 8) {
#pragma unroll
                for (int j = 0; j < VPL / 8; ++j) {
                    const uint4 v = reinterpret_cast<const uint4*>(src)[j];
                    w[4 * j] = v.x; w[4 * j + 1] = v.y; w[4 * j + 2] = v.z; w[4 * j + 3] = v.w;
                }
            } else if constexpr (VPL == 4) {
                const uint2 v = *reinterpret_cast<const uint2*>(src);
                w[0] = v.x; w[1] = v.y;
            } else {
                w[0] = *reinterpret_cast<const uint32_t*>(src);
            }
#pragma unroll
            for (int j = 0; j < VPL / 2; ++j) { raw[2 * j] = w[j] & 0xffffu; raw[2 * j + 1] = w[j] >> 16; }
        } else {
#pragma unroll
            for (int i = 0; i < VPL; ++i) raw[i] = e0 + i < experts ? src[i] : 0u;
        }
    }
}
template <int VPL>
__device__ __forceinline__ void as_logits(const RouteParams& p, int lane, int experts, const uint32_t (&raw)[VPL], float (&x)[VPL]) {
    if (p.logit_type == kLogitFp32) {
#pragma unroll
        for (int i = 0; i < VPL; ++i) x[i] = as_logit(__uint_as_float(raw[i]));
    } else if (p.logit_type == kLogitBf16) {
#pragma unroll
        for (int i = 0; i < VPL; ++i) x[i] = as_logit(__uint_as_float(raw[i] << 16));
    } else {
#pragma unroll
        for (int i = 0; i < VPL; ++i) x[i] = as_logit(__half2float(__ushort_as_half(static_cast<unsigned short>(raw[i]))));
    }
    if (experts != 32 * VPL) {
#pragma unroll
        for (int i = 0; i < VPL; ++i)
            if (lane * VPL + i >= experts) x[i] = -INFINITY;
    }
}

// Takes the key out of the warp's keys that is top_key, the one of the lowest expert where several are: that expert.  (Each key is compared
// with the place that is to go: picked by an index the keys would live in local memory.)
template <typename Key, int VPL>
__device__ __forceinline__ uint32_t take(Key (&key)[VPL], Key top_key, int lane) {
    uint32_t mine = 0xffffffffu;
#pragma unroll
    for (int i = VPL - 1; i >= 0; --i)
        if (key[i] == top_key) mine = lane * VPL + i;
    const uint32_t e = __reduce_min_sync(0xffffffffu, mine);
#pragma unroll
    for (int i = 0; i < VPL; ++i)
        if (e == static_cast<uint32_t>(lane * VPL + i)) key[i] = 0;
    return e;
}

// The choice of one token by one warp: lane holds experts lane * VPL, lane * VPL + 1, ...
//
// Keys.  Where the order of the logits is the order of the choice (no bias, and groups judged by their best) the keys
// are those of the logits, and exact.  Otherwise two scores may be nearer to each other than 32 bits show, and which
// experts are taken must not depend on how an exponential rounds.  The scores are computed in 32 bits all the same, with a
// bound on their error, and every decision is checked against it: where two neighbours of the ranking are not further
// apart than the bound allows, the candidates' scores are computed and ranked in 64 bits; where groups are not, theirs
// are, or (groups whose experts are not those of whole lanes) the token is chosen again in 64 bits (choose_exactly).  A launch waits
// for its slowest token, so these paths count although few tokens take them.
//
// Bound by instructions (1200 a token of 256 experts, 2.2 a cycle and SM): 8192 tokens of 256 experts take 20.0 us by sigmoid, bias and eight groups, 15.0 by
// softmax (5 of either for the order of the pairs behind it); one token of 64 or 256 experts 3.3 and 3.7.
//
// Ranking.  The top_k largest keys are not below the top_k-th largest of the lanes' maxima.  What is not below it, seldom much
// more than top_k keys, is put side by side, one to a lane, and each counts those ahead of it.  (Taking the largest top_k
// times from all lanes' keys took 919 instructions a token of 256 experts, and waited for most of them.)

// The same in 64 bits and by taking the largest again and again, for the few tokens that need it: apart from the other, so that its
// registers are not the kernel's.  Slot j's expert and its logit end in lane j.  keys: experts words of 64 bits of shared memory (with
// groups).
template <bool BY_LOGIT, int VPL>
__device__ __noinline__ int choose_exactly(const RouteParams& p, const PlanParams& q, long long token, int lane, uint64_t* keys, int& expert,
                                            float& logit) {
    float x[VPL];
    uint64_t key[VPL];
    float top = -INFINITY;
    {
        uint32_t raw[VPL];
        load_raw<VPL>(p, token * p.logits_row_stride, lane, q.experts, raw);
        as_logits<VPL>(p, lane, q.experts, raw, x);
    }
#pragma unroll
    for (int i = 0; i < VPL; ++i) top = fmaxf(top, x[i]);
    double total = 0.0;    // softmax: sum of exp(x - top)
    if (!BY_LOGIT && p.scoring == kScoreSoftmax) {
        top = value_of(warp_max(key_of(top)));
#pragma unroll 1
        for (int i = 0; i < VPL; ++i) total += x[i] == -INFINITY ? 0.0 : exp(static_cast<double>(x[i]) - top);
        total = warp_sum(total);
    }
#pragma unroll 1
    for (int i = 0; i < VPL; ++i) {
        const int e = lane * VPL + i;
        double c = x[i];
        if (!BY_LOGIT && x[i] != -INFINITY)
            c = (p.scoring == kScoreSoftmax ? exp(static_cast<double>(x[i]) - top) / total : 1.0 / (1.0 + exp(-static_cast<double>(x[i])))) +
                (p.bias ? static_cast<double>(p.bias[e]) : 0.0);
        key[i] = c == c && c != -INFINITY ? key_of(c) : 0ull;     // (a bias of -inf or NaN masks its expert too)
    }
    if (p.groups > 1) {
        __syncwarp();
#pragma unroll
        for (int i = 0; i < VPL; ++i)
            if (lane * VPL + i < q.experts) keys[lane * VPL + i] = key[i];
        __syncwarp();
        const int per = q.experts / p.groups;
        uint64_t mine = 0;
        if (lane < p.groups) {
            uint64_t first = 0, second = 0;
            for (int i = 0; i < per; ++i) {
                const uint64_t k = keys[lane * per + i];
                if (k > first) { second = first; first = k; }
                else if (k > second) second = k;
            }
            mine = !BY_LOGIT && p.group_top == 2 && second ? key_of(value_of(first) + value_of(second)) : first;
        }
        uint32_t kept = 0;
        for (int g = 0; g < p.top_groups; ++g) {
            const uint64_t best = warp_max(mine);
            if (best == 0) break;
            const int at = __ffs(__ballot_sync(0xffffffffu, mine == best)) - 1;
            kept |= 1u << at;
            if (lane == at) mine = 0;
        }
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            const int e = lane * VPL + i;
            if (e < q.experts && !(kept >> (e / per) & 1u)) key[i] = 0;
        }
        __syncwarp();
    }
    expert = -1;
    int n = 0;
    for (; n < q.top_k; ++n) {
        uint64_t best = key[0];
#pragma unroll
        for (int i = 1; i < VPL; ++i) best = key[i] > best ? key[i] : best;
        const uint64_t top_key = warp_max(best);
        if (top_key == 0) break;
        const uint32_t e = take(key, top_key, lane);
        if (lane == n) expert = static_cast<int>(e);
    }
    logit = expert >= 0 ? load_logit(p, token * p.logits_row_stride + expert) : 0.f;
    return n;
}

// A choice in 64 bits.  all: sum of exp(x - top) over the experts (softmax).
__device__ __forceinline__ double exact_choice(int scoring, float x, float top, double all, float bias) {
    const double l = x;
    return (scoring == kScoreSoftmax ? exp(l - top) / all : 1.0 / (1.0 + exp(-l))) + static_cast<double>(bias);
}
// (for loops that stand unrolled)
__device__ __noinline__ double exact_choice_call(int scoring, float x, float top, double all, float bias) { return exact_choice(scoring, x, top, all, bias); }
template <int VPL>
__device__ __forceinline__ double exact_total(const float (&x)[VPL], float top) {
    double all = 0.0;
#pragma unroll
    for (int i = 0; i < VPL; ++i) all += x[i] == -INFINITY ? 0.0 : exp(static_cast<double>(x[i]) - top);
    return warp_sum(all);
}

// Rank of this lane's key among `of` keys of shared memory (16-byte aligned, the last four filled up with zeros): larger ones, and
// as large ones of a lower place.
__device__ __forceinline__ int rank_of(uint32_t mine, int place, const uint32_t* of, int count) {
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < count; j += 4) {
        const uint4 o = *reinterpret_cast<const uint4*>(of + j);
        rank += (o.x > mine || (o.x == mine && j < place)) + (o.y > mine || (o.y == mine && j + 1 < place)) +
                (o.z > mine || (o.z == mine && j + 2 < place)) + (o.w > mine || (o.w == mine && j + 3 < place));
    }
    return rank;
}

// x: the token's logits.  most: above every |choice|.  keys: shared memory of this warp (p.key_words, 16-byte aligned).  A lane whose slot is not negative has the
// expert of that slot; slots that no lane has are nobody's.  Returns how many there are.
template <bool BY_LOGIT, int VPL>
__device__ __forceinline__ int choose(const RouteParams& p, const PlanParams& q, long long token, int lane, const float (&x)[VPL], const float (&bias)[VPL],
                                      float most, uint32_t* keys, int& slot, int& expert, float& weight) {
    uint32_t key[VPL];
    float top = 0.f, total = 1.f;    // softmax: the largest logit, sum of exp(x - top)
    [[maybe_unused]] float t[VPL];   // scores
    if (p.scoring == kScoreSoftmax) {
        top = x[0];
#pragma unroll
        for (int i = 1; i < VPL; ++i) top = fmaxf(top, x[i]);
        top = value_of(warp_max(key_of(top)));
    }
    // (a branch around each loop, not a choice in it: both sides of a choice are computed)
    if (p.scoring == kScoreSoftmax) {
        if (!BY_LOGIT || !p.renormalize) {
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < VPL; ++i) {
                t[i] = x[i] == -INFINITY ? 0.f : __expf(x[i] - top);
                sum += t[i];
            }
            total = warp_sum(sum);
            if constexpr (!BY_LOGIT) {
                const float inv = __fdividef(1.f, total);
#pragma unroll
                for (int i = 0; i < VPL; ++i) t[i] *= inv;
            }
        }
    } else if constexpr (!BY_LOGIT) {
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            const float u = __expf(-fabsf(x[i]));
            t[i] = __fdividef(x[i] >= 0.f ? 1.f : u, 1.f + u);
        }
    }
    float apart = 0.f;    // decisions are sure where the values are further apart than this
    if constexpr (BY_LOGIT) {
#pragma unroll
        for (int i = 0; i < VPL; ++i) key[i] = key_of(x[i]);
    } else {
        // Errors in units of u = 2^-24.
        // Softmax.  exp(-d) by __expf is off by (4 + 3.35 d) u of itself (2 + 1.173 d ulp of two u, and d's own rounding): 4 u of the
        // largest at most.  Its product with 1 / total adds one: 5 / total is what a choice has of its own.  All scores share the error of
        // 1 / total: VPL + 5 for the additions, 4 for the quotient, and G for the exponentials that were summed, the mean of 4 + 3.35 d over the
        // total.  G is largest where most of the total lies a few units below the largest logit: 10.1, 11.7, 13.4, 15.2, 17.0,
        // 18.9 for 32, 64, ... 1024 experts.  What is shared counts by how far two scores differ, 1 / total at most.  With a rounding of
        // `most` for either choice, two choices are off by (VPL + 19 + G) / total + 2 most; 2 (VPL + 16) / total + 2 most is taken,
        // which is more as long as G < VPL + 13.  Sums of two choices each: twice that, and 4 most for the sums' own roundings.
        // Sigmoid: 5.4 of a score of at most 1 (exponential, sum, quotient); 10 are taken.
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            // (an expert whose logit or bias is -inf or NaN: -inf)
            const float c = fmaxf(x[i] == -INFINITY ? -INFINITY : t[i] + bias[i], -INFINITY);
            key[i] = key_of(c);
        }
        const float units = p.scoring == kScoreSoftmax ? __fdividef(VPL + 16.f, fmaxf(total, 1.f)) : 10.f;      // (the largest softmax score is 1 / total, and total 0 where nothing can be chosen)
        apart = 2.f * 5.9604645e-8f * (units + most);
    }
    if (p.groups > 1) {
        // A group's experts are those of direct_lanes neighbouring lanes; or, where lanes hold experts of several groups, the keys go through
        // shared memory, 32 / (groups rounded up to a power of two) lanes judge a group, rows of keys one word apart, against
        // bank conflicts.
        const bool direct = p.direct_lanes != 0;
        const int lanes = direct ? p.direct_lanes : p.group_lanes, g = lane / lanes;
        uint32_t first = 0, second = 0;
        if (direct) {
#pragma unroll
            for (int i = 0; i < VPL; ++i) {
                second = max(second, min(first, key[i]));
                first = max(first, key[i]);
            }
        } else {
            __syncwarp();
            const int per = q.experts / p.groups;
#pragma unroll
            for (int i = 0; i < VPL; ++i) {
                const int e = lane * VPL + i;
                if (e < q.experts) keys[e + (e * p.per_magic >> 20)] = key[i];
            }
            __syncwarp();
            if (g < p.groups)
                for (int i = lane & (lanes - 1); i < per; i += lanes) {
                    const uint32_t k = keys[g * (per + 1) + i];
                    second = max(second, min(first, k));
                    first = max(first, k);
                }
        }
        for (int s = 1; s < lanes; s <<= 1) {
            const uint32_t f = __shfl_xor_sync(0xffffffffu, first, s), u = __shfl_xor_sync(0xffffffffu, second, s);
            second = max(min(first, f), max(second, u));
            first = max(first, f);
        }
        uint32_t mine = first;
        if (!BY_LOGIT && p.group_top == 2 && second) mine = key_of(value_of(first) + value_of(second));
        // rank of the group among all: better ones, and as good ones of a lower index
        int rank = 0;
#pragma unroll 8
        for (int h = 0; h < p.groups; ++h) {
            const uint32_t other = __shfl_sync(0xffffffffu, mine, h * lanes);
            rank += other > mine || (other == mine && h < g);
        }
        bool keep = g < p.groups && rank < p.top_groups;
        if constexpr (!BY_LOGIT) {
            const uint32_t worst = __reduce_min_sync(0xffffffffu, keep ? mine : 0xffffffffu);
            const uint32_t best = __reduce_max_sync(0xffffffffu, keep || g >= p.groups ? 0u : mine);
            const float margin = 2.f * apart + 4.f * 5.9604645e-8f * most;
            if (best != 0 && worst != 0 && !(value_of(worst) - value_of(best) > margin)) {
                if (!direct) {
                    apart = INFINITY;
                } else {
                    // Groups that are that near to the border compete for the places there with scores of 64 bits, made of the choices that may
                    // be their largest (one such token in 8192 cost 2.5 us of the launch when it was chosen again as a whole).
                    const bool open = g < p.groups && (keep ? !(value_of(mine) - value_of(best) > margin) : !(value_of(worst) - value_of(mine) > margin));
                    const uint32_t last = p.group_top == 2 ? second : first;
                    const uint32_t from = last ? max(key_of(value_of(last) - apart), 1u) : 1u;
                    double all = 1.0, e1 = -INFINITY, e2 = -INFINITY;
                    if (p.scoring == kScoreSoftmax) all = exact_total<VPL>(x, top);
#pragma unroll
                    for (int i = 0; i < VPL; ++i)
                        if (open && key[i] >= from) {
                            const double c = exact_choice_call(p.scoring, x[i], top, all, bias[i]);
                            e2 = fmax(e2, fmin(e1, c));
                            e1 = fmax(e1, c);
                        }
                    for (int s = 1; s < lanes; s <<= 1) {
                        const double f = __shfl_xor_sync(0xffffffffu, e1, s), u = __shfl_xor_sync(0xffffffffu, e2, s);
                        e2 = fmax(fmin(e1, f), fmax(e2, u));
                        e1 = fmax(e1, f);
                    }
                    const double score = p.group_top == 2 && e2 != -INFINITY ? e1 + e2 : e1;
                    const uint32_t opened = __ballot_sync(0xffffffffu, open);
                    const int places = __popc(__ballot_sync(0xffffffffu, open && keep && (lane & (lanes - 1)) == 0));
                    int ahead = 0;
                    for (int h = 0; h < p.groups; ++h) {
                        const double other = __shfl_sync(0xffffffffu, score, h * lanes);
                        ahead += (opened >> (h * lanes) & 1u) && (other > score || (other == score && h < g));
                    }
                    if (open) keep = ahead < places;
                }
            }
        }
        if (direct) {
#pragma unroll
            for (int i = 0; i < VPL; ++i) key[i] = keep ? key[i] : 0u;
        } else {
            const uint32_t heads = __ballot_sync(0xffffffffu, keep && (lane & (lanes - 1)) == 0);      // bit h * lanes: group h is kept
#pragma unroll
            for (int i = 0; i < VPL; ++i) {
                const int e = lane * VPL + i;
                if (e < q.experts && !(heads >> ((e * p.per_magic >> 20) * lanes) & 1u)) key[i] = 0;
            }
            __syncwarp();
        }
    }
    // candidates, one to a lane: cand holds their keys, ids their experts
    uint32_t* const cand = keys;
    uint32_t* const ids = keys + 32;
    [[maybe_unused]] float* const logits = reinterpret_cast<float*>(keys + 96);       // (those of the scores' candidates)
    const bool unsure_group = !BY_LOGIT && apart == INFINITY;
    int n = 0, rank = 0;
    uint32_t mine = 0u;
    expert = -1;
    bool tight = false;         // the candidates may not be all that are too near to the last one to be told apart
    float logit = 0.f;
    if constexpr (VPL == 1) {
        mine = key[0];
        expert = lane;
        logit = x[0];
        cand[lane] = mine;
        n = __popc(__ballot_sync(0xffffffffu, mine != 0));
        __syncwarp();
        rank = rank_of(mine, lane, cand, 32);
    } else {
        const int least = q.top_k + (BY_LOGIT ? 0 : 1);       // (by scores the next one is needed too, to be told apart)
        uint32_t best = key[0];
#pragma unroll
        for (int i = 1; i < VPL; ++i) best = max(best, key[i]);
        cand[lane] = best;
        __syncwarp();
        int ahead = 0;      // lanes whose best is larger: the least-th largest is the smallest that fewer than that are ahead of
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
            const uint4 o = *reinterpret_cast<const uint4*>(cand + j);
            ahead += (o.x > best) + (o.y > best) + (o.z > best) + (o.w > best);
        }
        uint32_t floor_key = least > 32 ? 0u : __reduce_min_sync(0xffffffffu, ahead < least ? best : 0xffffffffu);
        if (!BY_LOGIT && floor_key) floor_key = key_of(value_of(floor_key) - apart);
        floor_key = max(floor_key, 1u);
        __syncwarp();
        cand[lane] = 0u;
        __syncwarp();
        int pos = 0;        // candidates of the lanes ahead: side by side in the order of the experts
        auto count_candidates = [&]() {
            n = pos = 0;
#pragma unroll
            for (int i = 0; i < VPL; ++i) {
                const uint32_t b = __ballot_sync(0xffffffffu, key[i] >= floor_key);
                pos += __popc(b & ((1u << lane) - 1u));
                n += __popc(b);
            }
        };
        count_candidates();
        if (n > 32 && least <= 32 && !unsure_group) {
            // More than lanes: fewer lanes have anything than are to be chosen (few groups or experts are left, a lane's experts are neighbours), or
            // nearly as many are to be chosen as there are lanes.  A threshold that `least` to 32 keys are not below, by halves.
            // (8192 tokens of 256 experts, by logits: 2 of 8 groups 17.4 us, chosen in 64 bits 56; 24 and 32 of all 21.4 and 24.5, in 64 bits 53 and 64.
            // By scores 24 and 31 of all take 26.8 and 33.6; for 32 the 33rd would be needed too, one more than lanes, so where more than 32 can
            // be chosen these are chosen in 64 bits: 72.5.)
            uint32_t low = floor_key, high = warp_max(best);      // more than 32 are not below low; fewer than least above high
#pragma unroll 1
            while (low < high) {
                const uint32_t mid = low + (high - low + 1) / 2;
                int c = 0;
#pragma unroll
                for (int i = 0; i < VPL; ++i) c += key[i] >= mid;
                c = __reduce_add_sync(0xffffffffu, c);
                if (c > 32) low = mid;
                else if (c < least) high = mid - 1;
                else {
                    floor_key = mid;
                    tight = true;
                    break;
                }
            }
            if (tight) count_candidates();
        }
#pragma unroll
        for (int i = 0; i < VPL; ++i)
            if (key[i] >= floor_key) {
                if (pos < 32) {
                    cand[pos] = key[i];
                    ids[pos] = lane * VPL + i;
                    if (!BY_LOGIT) logits[pos] = x[i];
                }
                ++pos;
            }
        __syncwarp();
        if (lane < n) {
            mine = cand[lane];
            expert = ids[lane];
            if (!BY_LOGIT) logit = logits[lane];
        }
        rank = rank_of(mine, lane, cand, min(n, 32));
    }
    bool by_hand = n > 32 || unsure_group;
    if (!by_hand) {
        if constexpr (!BY_LOGIT) {
            uint32_t* const sorted = keys + 64;
            if (mine) sorted[rank] = mine;
            __syncwarp();
            bool sure = true;
            if (lane < q.top_k && lane + 1 < n) sure = value_of(sorted[lane]) - value_of(sorted[lane + 1]) > apart;
            const bool all_sure = __all_sync(0xffffffffu, sure);
            // (candidates by halves hold at least one more than are chosen: those that may be chosen, if the last is sure to be none of them)
            by_hand = !all_sure && tight && !(value_of(sorted[q.top_k - 1]) - value_of(sorted[n - 1]) > apart);
            if (!all_sure && !by_hand) {
                const double all = p.scoring == kScoreSoftmax ? exact_total<VPL>(x, top) : 1.0;
                uint64_t exact = 0;
                if (mine) exact = key_of(exact_choice(p.scoring, logit, top, all, p.bias ? p.bias[expert] : 0.f));
                rank = 0;
#pragma unroll 4
                for (int j = 0; j < (VPL == 1 ? 32 : n); ++j) {
                    const uint64_t other = __shfl_sync(0xffffffffu, exact, j);
                    rank += other > exact || (other == exact && j < lane);
                }
            }
        }
        slot = mine && rank < q.top_k ? rank : -1;
        if (BY_LOGIT && slot >= 0) logit = value_of(mine);
    }
    if (by_hand) {
        // more alike than lanes, or groups that 32 bits cannot tell apart
        __syncwarp();
        n = choose_exactly<BY_LOGIT, VPL>(p, q, token, lane, reinterpret_cast<uint64_t*>(keys), expert, logit);
        slot = expert >= 0 ? lane : -1;
    }
    float s = 0.f;
    if (slot >= 0) {
        const float a = expf(p.scoring == kScoreSoftmax ? logit - top : -fabsf(logit));
        s = p.scoring == kScoreSoftmax ? a / total : (logit >= 0.f ? 1.f : a) / (1.f + a);
    }
    if (p.renormalize) {
        const float sum = warp_sum(s);
        if (sum > 1e-30f) {
            s /= sum;
        } else {       // scores that 32 bits hardly hold: their ratios in 64
            const double far = slot < 0 ? 0.0 : p.scoring == kScoreSoftmax ? exp(static_cast<double>(logit) - top) : 1.0 / (1.0 + exp(-static_cast<double>(logit)));
            const double all = warp_sum(far);
            s = all > 0.0 ? static_cast<float>(far / all) : 0.f;
        }
    }
    weight = s * p.scale;
    return min(n, q.top_k);
}

// -------------------------------------------------------------------------------------------------- plan
// Exclusive sums over the experts of a CTA: first row and first tile of each.  count[e] in, row0[e] / tile0[e] out
// (both of experts + 1 entries); all threads of the CTA take part.  scratch: 2 x 32 words.
__device__ __forceinline__ void scan_experts(const int* count, int* row0, int* tile0, int experts, int tile_shift, int* scratch) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    int carry_r = 0, carry_t = 0;
    for (int base = 0; base < experts; base += blockDim.x) {
        const int e = base + threadIdx.x;
        const int c = e < experts ? count[e] : 0;
        int r = c, t = (c + (1 << tile_shift) - 1) >> tile_shift;
        const int t_own = t;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
            const int a = __shfl_up_sync(0xffffffffu, r, s), b = __shfl_up_sync(0xffffffffu, t, s);
            if (lane >= s) { r += a; t += b; }
        }
        if (lane == 31) { scratch[warp] = r; scratch[32 + warp] = t; }
        __syncthreads();
        // (every warp adds up the warps' sums itself)
        int wr = lane < warps ? scratch[lane] : 0, wt = lane < warps ? scratch[32 + lane] : 0;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
            const int a = __shfl_up_sync(0xffffffffu, wr, s), b = __shfl_up_sync(0xffffffffu, wt, s);
            if (lane >= s) { wr += a; wt += b; }
        }
        const int up_r = __shfl_sync(0xffffffffu, wr, max(warp - 1, 0)), up_t = __shfl_sync(0xffffffffu, wt, max(warp - 1, 0));
        const int before_r = carry_r + (warp ? up_r : 0), before_t = carry_t + (warp ? up_t : 0);
        carry_r += __shfl_sync(0xffffffffu, wr, 31);
        carry_t += __shfl_sync(0xffffffffu, wt, 31);
        if (e < experts) { row0[e] = before_r + r - c; tile0[e] = before_t + t - t_own; }
        __syncthreads();
    }
    if (threadIdx.x == 0) { row0[experts] = carry_r; tile0[experts] = carry_t; }
    __syncthreads();
}

// A pair's row and the row of its scales, where its rank among the expert's pairs is known.
__device__ __forceinline__ void put_rows(const PlanParams& q, long long pair, int e, int rank, const int* row0, const int* tile0) {
    const bool some = e >= 0 && e < q.experts;
    q.row[pair] = some ? row0[e] + rank : -1;
    q.sf_row[pair] = some ? (tile0[e] + (rank >> q.tile_shift)) * q.tile_sf_rows + (rank & (q.tile_tokens - 1)) : -1;
}

// offsets and the tile table, by the threads of one CTA (all of them look at row0 / tile0 of shared memory)
__device__ __forceinline__ void write_tables(const PlanParams& q, const int* row0, const int* tile0) {
    for (int e = threadIdx.x; e <= q.experts; e += blockDim.x) q.offset[e] = row0[e];
    if (threadIdx.x == 0) *q.tile_count = tile0[q.experts];
    for (int e = threadIdx.x; e < q.experts; e += blockDim.x)
        for (int r = row0[e], t = tile0[e]; r < row0[e + 1]; r += q.tile_tokens, ++t)
            q.tiles[t] = make_int4(e, r, min(q.tile_tokens, row0[e + 1] - r), 0);
}

// Shared memory of the plan, in words: next, row0 and tile0 [experts + 1], scan scratch, bits.
__host__ __device__ constexpr int plan_head_words(int experts) { return (3 * (experts + 1) + 64 + 3) & ~3; }
struct PlanSmem {
    int *next, *row0, *tile0, *scratch;
    uint32_t* bits;
    __device__ PlanSmem(int* smem, int experts)
        : next(smem), row0(next + experts + 1), tile0(row0 + experts + 1), scratch(tile0 + experts + 1),
          bits(reinterpret_cast<uint32_t*>(smem + plan_head_words(experts))) {}
};

// One or two chunks' share of the order, where the counts of all chunks (16 bits each) and every pair's rank in its chunk are known.  The eight CTAs of a
// cluster share the work of adding the counts up: each sums every eighth chunk, over all chunks and over those ahead of the cluster's, and takes the
// others' sums from their shared memory.  (Each CTA for itself: 148 CTAs read the same 75 KB of 256 experts' counts in 8000 cycles.)
// Two chunks where one each would be more CTAs than clusters of eight find room for at one CTA an SM (choice and order of 8192 x 8 of 256, softmax: 14.9 us, 17.3
// with one).
constexpr int kPlaceCluster = 8;
template <int CHUNKS>
__global__ void __launch_bounds__(kPlaceThreads, 1) place_kernel(const PlanParams q) {
    constexpr int kAtOnce = 2 * CHUNKS;
    extern __shared__ __align__(16) int plan_smem[];
    const PlanSmem s(plan_smem, q.experts);
    int* const sums = reinterpret_cast<int*>(s.bits);       // [2][experts]: ahead of the cluster's chunks, of all (this CTA's share)
    int* const next1 = sums + 2 * q.experts;                // s.next of the second chunk
    ptx::grid_dependency_wait();
    const int lane = threadIdx.x & 31;
    const int rank = static_cast<int>(ptx::cluster_ctarank());
    const int cluster_first = (static_cast<int>(blockIdx.x) - rank) * CHUNKS, chunk = static_cast<int>(blockIdx.x) * CHUNKS;
    const int count_row = counts_row(q.experts);
    const int chunk_pairs = q.chunk_tokens * q.top_k;
    const long long first = static_cast<long long>(chunk) * chunk_pairs;
    const int pairs = static_cast<int>(max(min(static_cast<long long>(CHUNKS) * chunk_pairs, static_cast<long long>(q.tokens) * q.top_k - first), 0ll));
    // this thread's first pairs: asked for ahead of everything that it waits for
    int e[kAtOnce], r[kAtOnce];
    auto ask = [&](int base) {
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) {
            const int i = base + j * kPlaceThreads + threadIdx.x;
            if (i < pairs) { e[j] = q.expert[first + i]; r[j] = q.row[first + i]; }
        }
    };
    ask(0);
    // a warp takes sixteen experts (a sector of a chunk's row), a lane a chunk
    for (int e0 = (threadIdx.x >> 5) * 16; e0 < q.experts; e0 += kPlaceThreads / 32 * 16) {
        int before[16] = {}, all[16] = {};
        for (int c = rank + kPlaceCluster * lane; c < q.chunks; c += kPlaceCluster * 32) {
            const uint4* src = reinterpret_cast<const uint4*>(q.counts + static_cast<long long>(c) * count_row + e0);
            const uint4 v0 = src[0], v1 = src[1];
            const uint32_t w[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const int n = (w[j >> 1] >> (16 * (j & 1))) & 0xffffu;
                all[j] += n;
                before[j] += c < cluster_first ? n : 0;
            }
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const int b = __reduce_add_sync(0xffffffffu, before[j]), t = __reduce_add_sync(0xffffffffu, all[j]);
            if (lane == j && e0 + j < q.experts) { sums[e0 + j] = b; sums[q.experts + e0 + j] = t; }
        }
    }
    ptx::cluster_arrive();
    // the chunks of this cluster ahead of this CTA's (last)
    for (int x = threadIdx.x; x < q.experts; x += kPlaceThreads) {
        int n = 0, own = 0;
#pragma unroll
        for (int i = 0; i < kPlaceCluster * CHUNKS - 1; ++i) {
            const int c = cluster_first + i;
            const int here = c <= (CHUNKS > 1 ? chunk : chunk - 1) && c < q.chunks ? q.counts[static_cast<long long>(c) * count_row + x] : 0;
            if (c == chunk) own = here;
            else n += here;
        }
        s.next[x] = n;
        if (CHUNKS > 1) next1[x] = n + own;
    }
    ptx::cluster_wait();
    ptx::grid_dependency_launch_dependents();
    for (int x = threadIdx.x; x < q.experts; x += kPlaceThreads) {
        const uint32_t at = ptx::smem_u32(sums + x);
        int before = 0, all = 0;
#pragma unroll
        for (int c = 0; c < kPlaceCluster; ++c) {
            const uint32_t from = ptx::mapa_u32(at, c);
            before += static_cast<int>(ptx::ld_shared_cluster_u32(from));
            all += static_cast<int>(ptx::ld_shared_cluster_u32(from + q.experts * 4));
        }
        s.next[x] += before;
        if (CHUNKS > 1) next1[x] += before;
        s.row0[x] = all;
    }
    if (pairs <= 0) {
        __syncthreads();
        ptx::cluster_arrive_relaxed();
    } else {
        scan_experts(s.row0, s.row0, s.tile0, q.experts, q.tile_shift, s.scratch);
        ptx::cluster_arrive_relaxed();      // (behind a barrier of the CTA: the others' sums have been read)
        if (chunk == 0) write_tables(q, s.row0, s.tile0);
        for (int base = 0; base < pairs; base += kAtOnce * kPlaceThreads) {
            if (base) ask(base);
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j) {
                const int i = base + j * kPlaceThreads + threadIdx.x;
                if (i < pairs) {
                    const bool some = e[j] >= 0 && e[j] < q.experts;
                    put_rows(q, first + i, e[j], some ? (CHUNKS == 1 || i < chunk_pairs ? s.next : next1)[e[j]] + r[j] : 0, s.row0, s.tile0);
                }
            }
        }
    }
    ptx::cluster_wait();        // none leaves while its sums are being read
}

// The rest of a CTA whose chunk's choices are in global memory: the pairs are counted in s.row0 (zero so far) and ranked.  Where the chunk is the
// only one this is all; else counts and ranks (in the place of the rows) go to place_kernel.
//
// Pairs are ranked 32 * bit_words at a time by a bit per pair and expert, so that the order is that of the pairs whichever
// thread comes first, and the same expert twice in a token gets two rows.
__device__ __forceinline__ void finish_chunk(const PlanParams& q, int chunk, const PlanSmem& s) {
    const long long first = static_cast<long long>(chunk) * q.chunk_tokens * q.top_k;
    const int pairs = static_cast<int>(min(static_cast<long long>(q.chunk_tokens) * q.top_k, static_cast<long long>(q.tokens) * q.top_k - first));
    const int words = q.bit_words, batch = 32 * words, stride = words | 1;     // (odd: an expert's words and the next one's in other banks)
    const bool only = q.chunks == 1;
    for (int e = threadIdx.x; e < q.experts; e += blockDim.x) s.next[e] = 0;     // pairs ahead of the batch
    if (pairs > batch && only) {       // the rows need all counts first
        for (int i = threadIdx.x; i < pairs; i += blockDim.x) {
            const int e = q.expert[first + i];
            if (e >= 0 && e < q.experts) atomicAdd(&s.row0[e], 1);
        }
        __syncthreads();
        scan_experts(s.row0, s.row0, s.tile0, q.experts, q.tile_shift, s.scratch);
    }
    for (int base = 0; base < pairs; base += batch) {
        const int here = min(batch, pairs - base);
        for (int i = threadIdx.x; i < q.experts * stride; i += blockDim.x) s.bits[i] = 0u;
        __syncthreads();
        for (int i = threadIdx.x; i < here; i += blockDim.x) {
            const int e = q.expert[first + base + i];
            if (e >= 0 && e < q.experts) {
                atomicOr(&s.bits[e * stride + (i >> 5)], 1u << (i & 31));
                if (!only || pairs <= batch) atomicAdd(&s.row0[e], 1);
            }
        }
        __syncthreads();
        if (only && pairs <= batch) scan_experts(s.row0, s.row0, s.tile0, q.experts, q.tile_shift, s.scratch);
        for (int i = threadIdx.x; i < here; i += blockDim.x) {
            const int e = q.expert[first + base + i];
            int rank = 0;
            if (e >= 0 && e < q.experts) {
                rank = s.next[e] + __popc(s.bits[e * stride + (i >> 5)] & ((1u << (i & 31)) - 1u));
#pragma unroll 4
                for (int w = 0; w < (i >> 5); ++w) rank += __popc(s.bits[e * stride + w]);
            }
            if (only) put_rows(q, first + base + i, e, rank, s.row0, s.tile0);
            else q.row[first + base + i] = rank;
        }
        if (base + batch >= pairs) break;
        __syncthreads();
        for (int e = threadIdx.x; e < q.experts; e += blockDim.x) {
            int n = 0;
            for (int w = 0; w < words; ++w) n += __popc(s.bits[e * stride + w]);
            s.next[e] += n;
        }
        __syncthreads();
    }
    if (only) write_tables(q, s.row0, s.tile0);
    else
        for (int e = threadIdx.x; e < q.experts; e += blockDim.x) q.counts[static_cast<long long>(chunk) * counts_row(q.experts) + e] = static_cast<uint16_t>(s.row0[e]);
}

__global__ void __launch_bounds__(kPlaceThreads) plan_kernel(const PlanParams q) {
    extern __shared__ __align__(16) int plan_smem[];
    const PlanSmem s(plan_smem, q.experts);
    for (int e = threadIdx.x; e < q.experts; e += blockDim.x) s.row0[e] = 0;
    __syncthreads();
    ptx::grid_dependency_launch_dependents();
    ptx::grid_dependency_wait();
    finish_chunk(q, blockIdx.x, s);
}

// A warp per token; the CTAs of a cluster share a chunk of tokens, and the first of them counts its pairs (and, where it is the only chunk,
// brings them into order).  The warps' keys stand where the plan's bits come later.
// (1024 threads leave 64 registers each; 256 experts by scores spill then: one token 6.5 us, 5.2 with 640 threads.)
constexpr int route_threads(int vpl) { return vpl <= 4 ? 1024 : vpl <= 8 ? 640 : vpl <= 16 ? 512 : 256; }
template <bool BY_LOGIT, int VPL>
__global__ void __launch_bounds__(route_threads(VPL)) route_kernel(const RouteParams p, const PlanParams q) {
    extern __shared__ __align__(16) int plan_smem[];
    const PlanSmem s(plan_smem, q.experts);
    for (int e = threadIdx.x; e < q.experts; e += blockDim.x) s.row0[e] = 0;
    __syncthreads();
    ptx::grid_dependency_launch_dependents();
    ptx::grid_dependency_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    uint32_t* const keys = s.bits + warp * p.key_words;
    const int ctas = p.chunk_ctas, chunk = blockIdx.x / ctas, rank = blockIdx.x - chunk * ctas;
    const long long chunk_first = static_cast<long long>(chunk) * q.chunk_tokens;
    const int in_chunk = static_cast<int>(min(static_cast<long long>(q.chunk_tokens), q.tokens - chunk_first));
    const int share = (in_chunk + ctas - 1) / ctas;
    const long long first = chunk_first + rank * share;
    const int tokens = min(share, in_chunk - rank * share);
    float bias[VPL];
    uint32_t ahead[VPL];     // the logits of a token are asked for while the one before is worked on
    if (warp < tokens) load_raw<VPL>(p, (first + warp) * p.logits_row_stride, lane, q.experts, ahead);
#pragma unroll
    for (int i = 0; i < VPL; ++i) bias[i] = !BY_LOGIT && p.bias && lane * VPL + i < q.experts ? p.bias[lane * VPL + i] : 0.f;
    float most = 0.f;        // above every choice: scores are at most 1
    if constexpr (!BY_LOGIT) {
#pragma unroll
        for (int i = 0; i < VPL; ++i)
            if (bias[i] == bias[i] && bias[i] != -INFINITY) most = fmaxf(most, fabsf(bias[i]));
        most = 1.f + __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most)));
    }
    for (int t = warp; t < tokens; t += warps) {
        float x[VPL];
        as_logits<VPL>(p, lane, q.experts, ahead, x);
        if (t + warps < tokens) load_raw<VPL>(p, (first + t + warps) * p.logits_row_stride, lane, q.experts, ahead);
        int slot, expert;
        float weight;
        const int n = choose<BY_LOGIT, VPL>(p, q, first + t, lane, x, bias, most, keys, slot, expert, weight);
        const long long at = (first + t) * q.top_k;
        if (slot >= 0) {
            q.expert[at + slot] = expert;
            p.weights[at + slot] = weight;
        }
        if (lane >= n && lane < q.top_k) {
            q.expert[at + lane] = -1;
            p.weights[at + lane] = 0.f;
        }
        __syncwarp();
    }
    __syncthreads();     // (the experts that the other threads wrote are read back from global memory by this CTA)
    if (ctas > 1) {
        ptx::cluster_arrive();     // releases what the CTAs have written
        ptx::cluster_wait();
        if (rank != 0) return;
    }
    finish_chunk(q, chunk, s);
}

// ------------------------------------------------------------------------------------------ routed quantiser
struct QuantizeRoutedParams {
    const uint8_t* x;
    uint8_t* packed;
    uint8_t* sf;             // atoms [scale rows / 128][k / 64][512]
    const int* row;          // [tokens][top_k]
    const int* sf_row;
    int tokens, top_k, k;
    int rows, sf_rows;       // bounds of what row and sf_row may say
    long long x_row_stride, packed_row_stride;   // bytes
};

constexpr int kRoutedCols = 512;     // columns per warp
// A lane takes one scale block (16 elements, 32 bytes) of a token, a warp 512 columns; the codes and scales, made once, are
// stored in each of the token's rows.  Bound by what it writes: 8192 x 8 rows of 7168 take 88 us (4.3 TB/s), 55 without the scales, four bytes of
// each row and four blocks in a sector of their own, which cost L2 as many writes as the codes; 8192 x 2 x 4096 20 (5.2 TB/s); one token 2.1.
template <bool BF16, bool kWide>
__global__ void __launch_bounds__(256) quantize_routed_kernel(const QuantizeRoutedParams p) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int blocks = p.k / 16;
    const unsigned col_units = (p.k + kRoutedCols - 1) / kRoutedCols;
    const long long unit = static_cast<long long>(blockIdx.x) * 8 + warp;
    const long long token = unit / col_units;
    const int blk = static_cast<int>(unit - token * col_units) * (kRoutedCols / 16) + lane;
    ptx::grid_dependency_wait();
    ptx::grid_dependency_launch_dependents();     // (behind the wait: the product that follows looks at the routing's tables ahead of its own)
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
        if (r < 0 || r >= p.rows || s < 0 || s >= p.sf_rows || !in_row) continue;
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

// A thread takes eight columns (16 bytes) of a token; the rows are added in the order of the choices, in fp32.  AT_ONCE: rows on their way at
// a time, no more than there are choices, so that the threads of few choices are many on an SM.  Bound by HBM: 4096 x 8 x 7168 93.5 us, 0.97 of the
// measured copy rate (32 bytes a thread: 99.0, 0.92).
template <bool BF16, int AT_ONCE>
__global__ void __launch_bounds__(256) combine_kernel(const CombineParams p) {
    const unsigned vecs = p.n / 8;
    ptx::grid_dependency_launch_dependents();
    ptx::grid_dependency_wait();
    const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
    const long long token = i / vecs;
    if (token >= p.tokens) return;
    const long long col = (i - token * vecs) * 8;
    const int* rows = p.rows + token * p.top_k;
    const float* weights = p.weights + token * p.top_k;
    // (eight rows' loads go ahead of the residual's: 4096 x 8 x 7168 97.9 us the other way round; with two it is better asked for
    // first: 4096 x 2 x 7168 40 us, after them 59)
    uint4 add = make_uint4(0u, 0u, 0u, 0u);
    if (AT_ONCE < 8 && p.residual) add = __ldcs(reinterpret_cast<const uint4*>(p.residual + (token * p.residual_row_stride + col) * 2));
    float s[8] = {};
    for (int j0 = 0; j0 < p.top_k; j0 += AT_ONCE) {
        uint4 v[AT_ONCE];
        float w[AT_ONCE];
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {
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
        for (int j = 0; j < AT_ONCE; ++j) {
            const uint32_t q[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 f = to_float2<false>(q[e]);
                s[2 * e] = fmaf(w[j], f.x, s[2 * e]);
                s[2 * e + 1] = fmaf(w[j], f.y, s[2 * e + 1]);
            }
        }
    }
    if (AT_ONCE == 8 && p.residual) add = __ldcs(reinterpret_cast<const uint4*>(p.residual + (token * p.residual_row_stride + col) * 2));
    if (p.residual) {
        const uint32_t q[4] = {add.x, add.y, add.z, add.w};
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
