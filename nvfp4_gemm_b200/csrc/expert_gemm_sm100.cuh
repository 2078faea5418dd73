// Grouped NVFP4 product of a mixture of experts for sm_100a: rows of activations in expert order, each expert's rows
// times that expert's weights, with scale, bias, (gated) activation and re-quantising in the epilogue.
//
// The weights are the M operand of the tensor core (128 of their rows = output columns per CTA), the rows of one expert the
// N operand: how many rows an expert has is known to the device alone, and N is a field of the instruction
// descriptor that a tile sets for itself, in steps of 16 or 32, while M would be padded to 128.
//
// Work is (token tile, block of weight rows); the table of token tiles {expert, first row, rows} comes from the
// plan.  A token tile's weight blocks are neighbours in the order, so that its rows and, tile after tile of one expert, its weights
// come from L2.
//
// Two forms: pairs of CTAs (tcgen05 with cta_group::2, 256 weight rows x up to 256 rows) where experts have many rows,
// and single CTAs with 128 weight rows x up to 32 rows, two on an SM, where what counts is how many bytes of
// weights are on their way.
//
// Warp roles: warp 0 TMA producer, warp 1 MMA issuer, one thread each; the others epilogue.  The accumulator holds one
// output column per TMEM lane and one row per TMEM column.  It is read in the fragment order of 16 lanes x 8 columns,
// where a thread has columns t and t + 8 of the output for the same row: gate and up, alternating in groups of eight,
// meet in a thread.  The finished fp16 pairs are turned round by stmatrix on their way to shared memory and leave as 16-byte pieces.
//
// Bounds and figures (us; weights E x n x k, rows in all).  Few rows: HBM, each touched expert's weights once: 8 x 4096 x 7168 for one token
// 20.7 (6.4 TB/s), 32 x 4096 x 4096 for 64 tokens x 4 45.4, 32 x 7168 x 2048 for 64 x 8 39.8 (6.6 TB/s).  Many rows: what the dense pair kernel
// is bound by, and its rates: 65536 rows evenly over 32 experts, 4096 x 7168 693-703 (5.5 PFLOP/s; dense, 8 batches 677), 7168 x 2048 426-437 (dense 434); in
// a loop the 1000 W limit holds the SM clock at 1.15 to 1.25 GHz.  Short K: the epilogue of a 256 x 256 tile takes 2.8 of its own, 3.3 with its
// stores, beside 3.0 of MMAs at k = 2048, and the next tile's MMAs wait for the half of it that reads what the accumulators share: 32768 rows,
// 7168 x 2048, 229-232 at full clock, the tensor pipe 59 % busy.
//
// Every wait is bounded.  No load uses cluster multicast.
#pragma once
#include "gemm_sm100.cuh"

namespace nvfp4 {

enum ExpertActivation : int { kExpertNone = 0, kExpertRelu = 1, kExpertSilu = 2, kExpertSwiglu = 3 };

struct ExpertGemmParams {
    CUtensorMap tma_w;        // weights {K/2 bytes, n rows, experts}, box {128, 128, 1}, 128B swizzle
    CUtensorMap tma_sfw;      // their scale atoms {128 words, K/64 atoms, row blocks, experts}, box {128, 4, 1, 1}
    CUtensorMap tma_x[4];     // rows in expert order {K/2 bytes, rows, 1}, boxes of 16, 32, 64 and 128 rows
    CUtensorMap tma_sfx[2];   // their scale atoms {128 words, K/64 atoms, blocks of all tiles, 1}, boxes of one and two blocks
    const int4* tiles;        // {expert, first row, rows, 0}
    const int* tile_count;
    const float* alpha;       // [experts] or null
    const __half* bias;       // [experts][n] or null
    long long bias_stride;    // elements
    int activation;
    float out_scale;
    int out_nvfp4;
    __half* c;
    long long c_row_stride;            // elements
    uint8_t* out_packed;
    long long out_packed_row_stride;   // bytes
    uint8_t* out_sf;                   // atoms, tile after tile like the input's
    int n, n_out, k_tiles, tiles_n;
    int experts, rows, most_tiles;     // bounds of what the tables hold
    int* status;
    unsigned long long timeout_cycles;
};

constexpr int kExpertPrefetch = 4;   // k-tiles of a CTA's first tile prefetched ahead of the dependency wait

template <int CG, int BT, int STAGES, int EPI_WARPS>
struct ExpertSmem {
    static constexpr uint32_t kWBytes = kBM * kBKBytes;
    static constexpr uint32_t kXRows = BT / CG;
    static constexpr uint32_t kXBytes = kXRows * kBKBytes;
    static constexpr uint32_t kSfwBytes = kMmaPerStage * kSfAtomBytes;
    static constexpr uint32_t kSfxBlocks = (BT + 127) / 128;
    static constexpr uint32_t kSfxBytes = kSfxBlocks * kMmaPerStage * kSfAtomBytes;
    static constexpr uint32_t kStageBytes = kWBytes + kXBytes + kSfwBytes + kSfxBytes;
    static constexpr int kThreads = 64 + 32 * EPI_WARPS;
    static constexpr uint32_t kStagingPerWarp = 2048;          // 32 rows x 32 columns of fp16
    static constexpr uint32_t kEpiOff = STAGES * kStageBytes;
    static constexpr uint32_t kBarOff = kEpiOff + EPI_WARPS * kStagingPerWarp;
    static constexpr uint32_t kNumBars = 2 * STAGES + 4;       // full, empty, accumulator full[2], empty[2]
    static constexpr uint32_t kBytes = kBarOff + kNumBars * 8 + 16;
    static constexpr uint32_t kDynamicBytes = kBytes + 1024;   // slack for manual 1024-byte alignment
    // TMEM: two accumulators and two buffers of either operand's scales.  256 columns: the accumulators overlap
    // by half, as in gemm_sm100.cuh.
    static constexpr bool kOverlap = BT == 256;
    static constexpr uint32_t kAccStride = kOverlap ? 128 : BT;
    static constexpr uint32_t kSfwCol = kOverlap ? 384 : 2 * BT;
    static constexpr uint32_t kSfxCol = kSfwCol + 32;
    static constexpr uint32_t kSfxColsPerMma = 4 * kSfxBlocks;
    static constexpr uint32_t kTmemUsed = kSfxCol + 2 * kMmaPerStage * kSfxColsPerMma;
    static constexpr uint32_t kTmemCols = kTmemUsed <= 128 ? 128 : kTmemUsed <= 256 ? 256 : 512;
    static_assert(kTmemUsed <= 512 && kStageBytes % 1024 == 0 && kDynamicBytes <= 232448, "does not fit an SM");
    static_assert(BT % (32 * CG) == 0 && kXRows <= 128 && (BT <= 128 || BT == 256), "token tile");
};

// A worker's tiles: every workers-th of (token tile, block of weight rows).  The table entry of the next one is asked for
// while the present one is worked on: read when it is needed it kept the MMA issuer waiting 500 cycles a tile.
// What the table says is brought within the bounds of the operands (it is the plan's, but the plan's memory is the caller's).
template <int BT>
struct ExpertTiles {
    const int4* tiles;
    int tiles_n, idx, total, step, experts, rows;
    int4 ahead;
    __device__ ExpertTiles(const ExpertGemmParams& p, int worker, int workers)
        : tiles(p.tiles), tiles_n(p.tiles_n), idx(worker - workers), total(min(__ldcg(p.tile_count), p.most_tiles) * p.tiles_n), step(workers),
          experts(p.experts), rows(p.rows) {
        look_ahead(worker);
    }
    __device__ __forceinline__ void look_ahead(int i) {
        if (i < total) ahead = __ldcg(&tiles[i / tiles_n]);
    }
    // the next tile: its entry, which token tile and which block it is
    __device__ __forceinline__ bool next(int4* t, int* tt, int* nt) {
        idx += step;
        if (idx >= total) return false;
        t->x = min(max(ahead.x, 0), experts - 1);
        t->z = min(max(ahead.z, 1), min(BT, rows));
        t->y = min(max(ahead.y, 0), rows - t->z);
        *tt = idx / tiles_n;
        *nt = idx - *tt * tiles_n;
        look_ahead(idx + step);
        return true;
    }
};

template <int CG, int BT, int STAGES, int EPI_WARPS, int CTAS_PER_SM>
__global__ void __launch_bounds__(ExpertSmem<CG, BT, STAGES, EPI_WARPS>::kThreads, CTAS_PER_SM) expert_gemm_kernel(const __grid_constant__ ExpertGemmParams p) {
    using S = ExpertSmem<CG, BT, STAGES, EPI_WARPS>;
    constexpr int kGroups = EPI_WARPS / 4;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* smem_gen = smem_raw + (smem_base - ptx::smem_u32(smem_raw));
    const uint32_t bar_full = smem_base + S::kBarOff;
    const uint32_t bar_empty = bar_full + STAGES * 8;
    const uint32_t bar_acc_full = bar_empty + STAGES * 8;
    const uint32_t bar_acc_empty = bar_acc_full + 2 * 8;
    const uint32_t tmem_slot = bar_acc_empty + 2 * 8;
    volatile uint32_t* tmem_slot_gen = reinterpret_cast<volatile uint32_t*>(smem_gen + S::kBarOff + S::kNumBars * 8);
    volatile uint32_t* abort_flag = tmem_slot_gen + 1;

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int cta_rank = CG == 2 ? static_cast<int>(ptx::cluster_ctarank()) : 0;
    const bool leader = cta_rank == 0;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            ptx::mbar_init(bar_full + s * 8, 1);
            ptx::mbar_init(bar_empty + s * 8, 1);
        }
        for (int a = 0; a < 2; ++a) {
            ptx::mbar_init(bar_acc_full + a * 8, 1);
            ptx::mbar_init(bar_acc_empty + a * 8, EPI_WARPS * CG);
        }
        *abort_flag = 0u;
        ptx::fence_mbar_init();
        ptx::prefetch_tensormap(&p.tma_w);
        ptx::prefetch_tensormap(&p.tma_sfw);
    }
    __syncthreads();
    if constexpr (CG == 2) {
        ptx::cluster_arrive();
        ptx::cluster_wait();
    }
    if (warp == 1) {
        ptx::tmem_alloc<CG>(tmem_slot, S::kTmemCols);
        ptx::tmem_relinquish<CG>();
        ptx::tc_fence_before();
    }
    const int KT = p.k_tiles;
    const int worker = static_cast<int>(blockIdx.x) / CG, workers = static_cast<int>(gridDim.x) / CG;
    // The weights of this CTA's first tile are asked into L2 ahead of the dependency wait: the router is usually done by now, only the kernel
    // that quantises the rows is not.  What stands in the table may still change (it may even be another call's left-overs): nothing
    // but a prefetch is made of it, and it is read past L1, so that what is read after the wait is read anew.
    if (warp == 0) {
        if (ptx::elect_one()) {
            const int count = min(__ldcg(p.tile_count), p.most_tiles);
            if (worker < count * p.tiles_n) {
                const int expert = __ldcg(&p.tiles[worker / p.tiles_n].x);
                const int wb = (worker % p.tiles_n) * CG + cta_rank;
                if (expert >= 0 && expert < p.experts)
                    for (int kt = 0; kt < min(kExpertPrefetch, KT); ++kt) {
                        ptx::tma_prefetch_3d(&p.tma_w, kt * kBKBytes, wb * kBM, expert);
                        ptx::tma_prefetch_4d(&p.tma_sfw, 0, kt * kMmaPerStage, wb, expert);
                    }
            }
        }
        __syncwarp();
    }
    ptx::grid_dependency_wait();
    ptx::grid_dependency_launch_dependents();     // (behind the wait: see the prefetch above, of the kernel that follows)
    uint32_t tmem_base = 0;
    if (warp != 0) {
        ptx::named_bar_sync(3, S::kThreads - 32);
        ptx::tc_fence_after();
        tmem_base = *tmem_slot_gen;
    }
    const uint64_t timeout = p.timeout_cycles;
    // rows of a tile -> columns of its MMAs
    auto mma_n = [](int rows) { return CG == 2 ? (rows + 31) & ~31 : (rows + 15) & ~15; };

    if (warp == 0) {
        // ------------------------------------------------------------ producer
        if (ptx::elect_one()) {
            // (also where an expert has several tiles of 32 rows: their blocks of the weights run side by side and meet in L2.  Weights that are
            // kept gain nothing there, 512 x 8 of 256 experts of up to 292 rows, 2048 x 2048: 103.7 us, 103.8 so, and cost
            // where there is one tile: 64 x 8 of 32, 4096 x 4096: 51.2, 44.8 so)
            const uint64_t pol_w = ptx::policy_evict_first();
            const uint64_t pol_x = ptx::policy_evict_last();
            uint32_t stage = 0, phase = 0;
            bool ok = true;
            ExpertTiles<BT> work(p, worker, workers);
            int4 t;
            int tt, nt;
            while (ok && work.next(&t, &tt, &nt)) {
                const int n = mma_n(t.z), xrows = n / CG;
                const int box = xrows <= 16 ? 0 : xrows <= 32 ? 1 : xrows <= 64 ? 2 : 3;
                const CUtensorMap* map_x = &p.tma_x[box];
                const CUtensorMap* map_sfx = &p.tma_sfx[n > 128 ? 1 : 0];
                const uint32_t bytes = CG * (S::kWBytes + S::kSfwBytes + (16u << box) * kBKBytes + (n > 128 ? 2u : 1u) * kMmaPerStage * kSfAtomBytes);
                const int wb = nt * CG + cta_rank;             // 128-row block of the weights
                const int xrow = t.y + cta_rank * xrows;
                const int sfx = tt * static_cast<int>(S::kSfxBlocks);
                for (int kt = 0; kt < KT; ++kt) {
                    ok = ptx::mbar_wait_bounded(bar_empty + stage * 8, phase ^ 1u, abort_flag, timeout);
                    if (!ok) break;
                    const uint32_t sw = smem_base + stage * S::kStageBytes;
                    const uint32_t sx = sw + S::kWBytes, ssfw = sx + S::kXBytes, ssfx = ssfw + S::kSfwBytes;
                    if constexpr (CG == 1) {
                        const uint32_t full = bar_full + stage * 8;
                        ptx::mbar_expect_tx(full, bytes);
                        ptx::tma_load_3d(sw, &p.tma_w, kt * kBKBytes, wb * kBM, t.x, full, pol_w);
                        ptx::tma_load_4d(ssfw, &p.tma_sfw, 0, kt * kMmaPerStage, wb, t.x, full);
                        ptx::tma_load_3d(sx, map_x, kt * kBKBytes, xrow, 0, full, pol_x);
                        ptx::tma_load_4d(ssfx, map_sfx, 0, kt * kMmaPerStage, sfx, 0, full);
                    } else {
                        const uint32_t full = ptx::mapa_u32(bar_full + stage * 8, 0);
                        if (leader) ptx::mbar_expect_tx(bar_full + stage * 8, bytes);
                        ptx::tma_load_3d_pair(sw, &p.tma_w, kt * kBKBytes, wb * kBM, t.x, full, pol_x);
                        ptx::tma_load_4d_pair(ssfw, &p.tma_sfw, 0, kt * kMmaPerStage, wb, t.x, full);
                        ptx::tma_load_3d_pair(sx, map_x, kt * kBKBytes, xrow, 0, full, pol_x);
                        ptx::tma_load_4d_pair(ssfx, map_sfx, 0, kt * kMmaPerStage, sfx, 0, full);
                    }
                    if (++stage == STAGES) { stage = 0; phase ^= 1u; }
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ------------------------------------------------------ MMA issuer (one thread, see gemm_sm100.cuh)
        if (leader) {
            const uint64_t desc_ab0 = ptx::smem_desc_sw128(smem_base);
            const uint64_t desc_sf0 = ptx::smem_desc_sf(smem_base + S::kWBytes + S::kXBytes);
            const uint32_t ab_lo0 = static_cast<uint32_t>(desc_ab0), ab_hi = static_cast<uint32_t>(desc_ab0 >> 32);
            const uint32_t sf_lo0 = static_cast<uint32_t>(desc_sf0), sf_hi = static_cast<uint32_t>(desc_sf0 >> 32);
            if (ptx::elect_one()) {
                uint32_t stage = 0, phase = 0, acc_it = 0, sf_buf = 0;
                bool ok = true;
                ExpertTiles<BT> work(p, worker, workers);
                int4 t;
                int tt, nt;
                while (ok && work.next(&t, &tt, &nt)) {
                    const int n = mma_n(t.z);
                    const uint32_t idesc = ptx::idesc_nvf4(kBM * CG, 0) | (static_cast<uint32_t>(n >> 3) << 17);
                    const bool two_blocks = n > 128;
                    const uint32_t acc = acc_it & 1u;
                    const uint32_t empty_bar = bar_acc_empty + (S::kOverlap ? 0u : acc * 8);
                    const uint32_t empty_phase = S::kOverlap ? (acc_it & 1u) : ((acc_it >> 1) & 1u);
                    ok = ptx::mbar_wait_bounded(empty_bar, empty_phase ^ 1u, abort_flag, timeout);
                    if (!ok) break;
                    ptx::tc_fence_after();
                    const uint32_t d_tmem = tmem_base + acc * S::kAccStride;
                    for (int kt = 0; kt < KT; ++kt) {
                        ok = ptx::mbar_wait_bounded(bar_full + stage * 8, phase, abort_flag, timeout);
                        if (!ok) break;
                        ptx::tc_fence_after();
                        const uint32_t slot_off = stage * (S::kStageBytes >> 4);
                        const uint32_t w_lo = ab_lo0 + slot_off, x_lo = w_lo + (S::kWBytes >> 4);
                        const uint32_t sfw_lo = sf_lo0 + slot_off, sfx_lo = sfw_lo + (S::kSfwBytes >> 4);
                        const uint32_t t_sfw = tmem_base + S::kSfwCol + sf_buf * 16;
                        const uint32_t t_sfx = tmem_base + S::kSfxCol + sf_buf * (kMmaPerStage * S::kSfxColsPerMma);
#pragma unroll
                        for (int kb = 0; kb < kMmaPerStage; ++kb) {
                            ptx::tc_cp_sf<CG>(t_sfw + kb * 4, sfw_lo + kb * (kSfAtomBytes >> 4), sf_hi);
                            ptx::tc_cp_sf<CG>(t_sfx + kb * S::kSfxColsPerMma, sfx_lo + kb * (kSfAtomBytes >> 4), sf_hi);
                            if (S::kSfxBlocks > 1 && two_blocks)
                                ptx::tc_cp_sf<CG>(t_sfx + kb * S::kSfxColsPerMma + 4, sfx_lo + ((kMmaPerStage + kb) * kSfAtomBytes >> 4), sf_hi);
                        }
#pragma unroll
                        for (int kb = 0; kb < kMmaPerStage; ++kb)
                            ptx::tc_mma_nvf4<CG>(d_tmem, w_lo + 2 * kb, x_lo + 2 * kb, ab_hi, idesc, t_sfw + kb * 4, t_sfx + kb * S::kSfxColsPerMma,
                                                 (kt > 0 || kb > 0) ? 1u : 0u);
                        if constexpr (CG == 2) ptx::tc_commit_pair(bar_empty + stage * 8, 0x3);
                        else ptx::tc_commit(bar_empty + stage * 8);
                        if (kt + 1 == KT) {
                            if constexpr (CG == 2) ptx::tc_commit_pair(bar_acc_full + acc * 8, 0x3);
                            else ptx::tc_commit(bar_acc_full + acc * 8);
                        }
                        sf_buf ^= 1u;
                        if (++stage == STAGES) { stage = 0; phase ^= 1u; }
                    }
                    ++acc_it;
                }
            }
            __syncwarp();
        }
    } else {
        // ------------------------------------------------------------ epilogue
        const int quad = warp & 3;             // TMEM lane quadrant this warp may read
        const int group = (warp - 2) / 4;      // which share of a tile's rows
        const uint32_t staging = smem_base + S::kEpiOff + (warp - 2) * S::kStagingPerWarp;
        uint8_t* const staging_gen = smem_gen + S::kEpiOff + (warp - 2) * S::kStagingPerWarp;
        const bool gated = p.activation == kExpertSwiglu;
        uint32_t acc_it = 0;
        ExpertTiles<BT> work(p, worker, workers);
        int4 t;
        int tt, nt;
        while (work.next(&t, &tt, &nt)) {
            const int wb = nt * CG + cta_rank;
            const bool exists = CG == 1 || wb * kBM < p.n;     // (n is a multiple of 128: a pair's second half may lie beyond it)
            const float alpha = (p.alpha ? p.alpha[t.x] : 1.f);
            // this thread's output columns: quad * 32 + half * 16 + {0, 8} + lane / 4 of the block
            float bias[2][2] = {};
            if (p.bias && exists) {
                const __half* b = p.bias + t.x * p.bias_stride + wb * kBM + quad * 32 + (lane >> 2);
#pragma unroll
                for (int h = 0; h < 4; ++h) bias[h >> 1][h & 1] = __half2float(b[h * 8]);
            }
            const uint32_t acc = acc_it & 1u;
            const uint32_t acc_phase = (acc_it >> 1) & 1u;
            bool got = true;
            if (warp == 2) got = ptx::mbar_wait_bounded(bar_acc_full + acc * 8, acc_phase, abort_flag, timeout);
            if (!ptx::named_bar_and(2, 32 * EPI_WARPS, got)) break;
            ptx::tc_fence_after();
            const uint32_t t_acc = tmem_base + acc * S::kAccStride + (static_cast<uint32_t>(quad * 32) << 16);
            auto release_acc = [&]() {
                ptx::tc_fence_before();
                __syncwarp();
                const uint32_t bar = bar_acc_empty + (S::kOverlap ? 0u : acc * 8);
                if (lane == 0) {
                    if (CG == 2 && !leader) ptx::mbar_arrive_cluster_signal(bar, 0);
                    else ptx::mbar_arrive(bar);
                }
            };
            // 32 rows at a time, those in columns that the other accumulator has too first
            const int chunks = (t.z + 31) >> 5;
            const int shared = !S::kOverlap ? chunks : acc == 0 ? max(chunks - 4, 0) : min(chunks, 4);
            const int first = (S::kOverlap && acc == 0 && chunks > 4) ? 4 : 0;
            auto chunk_at = [&](int pos) { return pos < shared ? first + pos : (S::kOverlap && acc == 0) ? pos - shared : pos; };
            // Two chunks of a group go to registers together: with two groups these are all that the accumulators share, and
            // the hand-back does not wait for anything to be converted or stored.
            bool released = false;
            uint32_t held[2][32];
            for (int i = 0, pos = group; pos < chunks; ++i, pos += kGroups) {
                uint32_t (&v)[32] = held[0];
                if ((i & 1) == 0) {
                    const int pos2 = pos + kGroups;
                    if (!released && pos >= shared) { release_acc(); released = true; }
                    const uint32_t at = t_acc + chunk_at(pos) * 32;
                    ptx::tc_ld_16lanes_32cols(at, held[0]);
                    ptx::tc_ld_16lanes_32cols(at + (16u << 16), held[0] + 16);
                    if (pos2 < chunks) {
                        const uint32_t at2 = t_acc + chunk_at(pos2) * 32;
                        ptx::tc_ld_16lanes_32cols(at2, held[1]);
                        ptx::tc_ld_16lanes_32cols(at2 + (16u << 16), held[1] + 16);
                    }
                    ptx::tc_wait_ld();
                    if (!released && pos2 + kGroups >= shared) { release_acc(); released = true; }
                } else {
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] = held[1][j];
                }
                const int chunk = chunk_at(pos);
                if (!exists) continue;
                float z[32];     // [half][8 rows of tokens][column t: even, odd token | column t + 8: even, odd token]
#pragma unroll
                for (int i = 0; i < 32; ++i) z[i] = fmaf(alpha, __uint_as_float(v[i]), bias[i >> 4][(i >> 1) & 1]);
                const int rows_left = t.z - chunk * 32;
                const long long row0 = t.y + chunk * 32;
                auto half2_of = [&](float a, float b) {
                    const __half2 h = __floats2half2_rn(a, b);
                    return *reinterpret_cast<const uint32_t*>(&h);
                };
                __syncwarp();    // the previous chunk's pieces have been read
                if (gated) {
                    // 16 output columns per warp: staging rows of 32 bytes, the two 16-byte units of rows 4 .. 7 (mod 8) exchanged
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t o[4];
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            float r[2];
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const float g = z[h * 16 + c * 4 + e];
                                r[e] = __fdividef(g, 1.f + __expf(-g)) * z[h * 16 + c * 4 + 2 + e] * p.out_scale;
                            }
                            o[c] = half2_of(r[0], r[1]);
                        }
                        ptx::st_matrix_x4_trans(staging + lane * 32 + ((h ^ (lane >> 2 & 1)) << 4), o[0], o[1], o[2], o[3]);
                    }
                } else {
                    if (p.activation == kExpertRelu) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) z[i] = ptx::relu(z[i]);
                    } else if (p.activation == kExpertSilu) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) z[i] = __fdividef(z[i], 1.f + __expf(-z[i]));
                    }
                    // staging rows of 64 bytes, their 16-byte units permuted so that eight rows' same unit spreads over all banks
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        uint32_t o[4];
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const int i = (u >> 1) * 16 + c * 4 + (u & 1) * 2;
                            o[c] = half2_of(z[i] * p.out_scale, z[i + 1] * p.out_scale);
                        }
                        ptx::st_matrix_x4_trans(staging + lane * 64 + ((u ^ (lane >> 1 & 3)) << 4), o[0], o[1], o[2], o[3]);
                    }
                }
                __syncwarp();
                const int col0 = gated ? (wb * kBM + quad * 32) / 2 : wb * kBM + quad * 32;
                if (!p.out_nvfp4) {
                    if (gated) {
#pragma unroll
                        for (int it = 0; it < 2; ++it) {
                            const int r = it * 16 + (lane >> 1), u = lane & 1;
                            const uint4 q = *reinterpret_cast<const uint4*>(staging_gen + r * 32 + ((u ^ (r >> 2 & 1)) << 4));
                            if (r < rows_left) *reinterpret_cast<uint4*>(p.c + (row0 + r) * p.c_row_stride + col0 + u * 8) = q;
                        }
                    } else {
#pragma unroll
                        for (int it = 0; it < 4; ++it) {
                            const int r = it * 8 + (lane >> 2), u = lane & 3;
                            const uint4 q = *reinterpret_cast<const uint4*>(staging_gen + r * 64 + ((u ^ (r >> 1 & 3)) << 4));
                            if (r < rows_left) *reinterpret_cast<uint4*>(p.c + (row0 + r) * p.c_row_stride + col0 + u * 8) = q;
                        }
                    }
                } else if (lane < rows_left) {
                    // a lane takes a row: one scale block (gated) or two
                    const int row = chunk * 32 + lane;
                    uint8_t* const sf = p.out_sf + (static_cast<long long>(tt) * S::kSfxBlocks + (row >> 7)) * (p.n_out / 64) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4;
                    uint8_t* const dst = p.out_packed + (row0 + lane) * p.out_packed_row_stride + col0 / 2;
#pragma unroll 1
                    for (int b = 0; b < (gated ? 1 : 2); ++b) {
                        uint32_t w[8];
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            const uint4 q = gated ? *reinterpret_cast<const uint4*>(staging_gen + lane * 32 + ((u ^ (lane >> 2 & 1)) << 4))
                                                  : *reinterpret_cast<const uint4*>(staging_gen + lane * 64 + (((2 * b + u) ^ (lane >> 1 & 3)) << 4));
                            w[4 * u] = q.x; w[4 * u + 1] = q.y; w[4 * u + 2] = q.z; w[4 * u + 3] = q.w;
                        }
                        uint32_t codes[2];
                        const uint32_t s = quantize_words<false>(w, codes);
                        const int blk = col0 / 16 + b;
                        *reinterpret_cast<uint2*>(dst + b * 8) = make_uint2(codes[0], codes[1]);
                        sf[(blk >> 2) * 512 + (blk & 3)] = static_cast<uint8_t>(s);
                    }
                }
            }
            if (!released) release_acc();
            ++acc_it;
        }
    }

    // ---------------------------------------------------------------- teardown
    ptx::tc_fence_before();
    __syncthreads();
    meet_cluster<CG>(abort_flag, tmem_slot + 4, p.status);
    const bool gave_up = CG > 1 && *abort_flag;
    if (warp == 1) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc<CG>(tmem_base, S::kTmemCols);
    }
    if constexpr (CG > 1) {
        // (also where nothing went wrong: no CTA may leave while the pair's other one frees its share of TMEM)
        if (gave_up) let_copies_land();
        ptx::cluster_arrive();
        ptx::cluster_wait();
    }
}

}  // namespace nvfp4
