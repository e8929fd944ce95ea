// Matrix products of several experts on tcgen05, 16-bit operands with float32 sums.  Expert e has rows ends[e - 1] .. ends[e] - 1:
//
//     rows:      C[r, n] = sum_k A[r, k] W_e[n, k]         for its rows r; the weight K-major or, for the input's gradient, MN-major
//     weights:   C_e[m, n] = sum_r A[r, m] B[r, n]         over its rows: K is as long as the expert has rows
//
// The ends are read by every CTA, which lays the tiles out for itself: a table of the experts' first rows and of their tiles before them in
// shared memory, in which a tile's number is looked up.  CTAs (or pairs) go round the tiles of all experts, an expert's one after the other.
//
// A tile's operand rows may be the next expert's: rows of results are its own, and those beyond its end are not written.  Where rows are
// summed over, the last stage of an expert is one that others' rows must not reach: its rows beyond the end are set to zero in shared memory, by two warps,
// between its arrival and its MMAs (zeros on one side alone would leave NaN from the other).
//
// Few rows an expert: they lie along the accumulator's columns, with 128 weight rows on its lanes, and what counts are the weights' bytes.
//
// Full tiles are bound by the tensor cores (92 % active; the rows of an expert's last tile that are not its own are computed with the others), and in a loop by the
// board's power: 16384 rows of 32 experts, 2048 -> 4096, 215 us (1.28 PFLOP/s of results), the weights' gradient 266 us (1.03, 60 % active), both at 1.2 GHz.  Few rows by
// memory: 64 rows over 64 experts, 2048 -> 1024, 26 us, 6.5 TB/s of weights.
//
// The ring of stages and the accumulators are those of wide_gemm.cuh; results leave from the registers of the warps that empty an
// accumulator, through its staging only where rows do not start on 16 bytes.
#pragma once

#include "wide_gemm.cuh"

namespace th {
namespace {

constexpr int kMostExperts = 1024;

struct ExpertArgs {
    GemmArgs g;  // m: of the output's rows (weights: of an expert's), n: of its columns; k_tiles, splits are not used
    const int32_t *ends;
    int experts, rows, k;
    int tile_rows;  // of an expert's rows in a tile
};

template <bool A_MN, bool B_MN, int BN, int CG, bool SWAP, bool OVER_ROWS, int CTAS>
struct ExpertShape {
    static constexpr int kK = 64;
    static constexpr int kBRows = BN / CG;
    static constexpr int kABytes = kGemmRows * 128, kBBytes = kBRows * 128, kStage = kABytes + kBBytes;
    static constexpr int kGroups = SWAP ? 1 : 2;  // of four warps that empty an accumulator, each its part of the columns
    static constexpr int kThreads = 128 + 128 * kGroups, kColumns = BN / kGroups;
    static constexpr int kFixed = SWAP ? 0 : 4 * kGroups * kPieceBytes;
    static constexpr int kTables = OVER_ROWS ? 4 * (kMostExperts + 1) : 8 * (kMostExperts + 1);
    static constexpr int kSmem = (CTAS == 1 ? 226 : 112) * 1024 - kTables;  // barriers are beside it
    static constexpr int kFit = (kSmem - kFixed - 1024) / kStage;
    static constexpr int kStages = kFit > 8 ? 8 : kFit;
    static constexpr int kBytes = kStages * kStage + kFixed + 1024;
    static constexpr int kTmemCols = 2 * BN < 32 ? 32 : 2 * BN;
    static_assert(kStages >= 3 && CTAS * kTmemCols <= 512, "tile does not fit");
};

// A stage's four MMAs and the commit to its barrier, by the lane whose `issue` is not zero: predicated instructions, the warp stays together
template <int CG, bool A_MN, bool B_MN>
__device__ __forceinline__ void expert_stage(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate, uint32_t issue, uint32_t stage_bar, uint32_t leader) {
    constexpr uint32_t kLeading = (kBoxBytes >> 4) << 16;  // MN-major operands lie in boxes of 64 columns
    constexpr int kStepA = A_MN ? 2048 >> 4 : 2, kStepB = B_MN ? 2048 >> 4 : 2;
    const uint32_t la = desc_low(a) | (A_MN ? kLeading : 0u), lb = desc_low(b) | (B_MN ? kLeading : 0u);
    if constexpr (CG == 1)
        asm volatile(
            "{\n\t.reg .pred p, t, f;\n\t.reg .b64 a0, a1, a2, a3, b0, b1, b2, b3;\n\t"
            "setp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 t, 0, 0;\n\tsetp.ne.b32 f, %6, 0;\n\t"
            "mov.b64 a0, {%1, %9};\n\tadd.s64 a1, a0, %7;\n\tadd.s64 a2, a1, %7;\n\tadd.s64 a3, a2, %7;\n\t"
            "mov.b64 b0, {%2, %9};\n\tadd.s64 b1, b0, %8;\n\tadd.s64 b2, b1, %8;\n\tadd.s64 b3, b2, %8;\n\t"
            "@p tcgen05.mma.cta_group::1.kind::f16 [%0], a0, b0, %3, f;\n\t"
            "@p tcgen05.mma.cta_group::1.kind::f16 [%0], a1, b1, %3, t;\n\t"
            "@p tcgen05.mma.cta_group::1.kind::f16 [%0], a2, b2, %3, t;\n\t"
            "@p tcgen05.mma.cta_group::1.kind::f16 [%0], a3, b3, %3, t;\n\t"
            "@p tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%5];\n\t}\n" ::"r"(d),
            "r"(la), "r"(lb), "r"(idesc), "r"(issue), "r"(stage_bar), "r"(accumulate), "n"(kStepA), "n"(kStepB), "r"(kDescHigh) : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p, t, f;\n\t.reg .b64 a0, a1, a2, a3, b0, b1, b2, b3;\n\t"
            "setp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 t, 0, 0;\n\tsetp.ne.b32 f, %6, 0;\n\t"
            "mov.b64 a0, {%1, %9};\n\tadd.s64 a1, a0, %7;\n\tadd.s64 a2, a1, %7;\n\tadd.s64 a3, a2, %7;\n\t"
            "mov.b64 b0, {%2, %9};\n\tadd.s64 b1, b0, %8;\n\tadd.s64 b2, b1, %8;\n\tadd.s64 b3, b2, %8;\n\t"
            "@p tcgen05.mma.cta_group::2.kind::f16 [%0], a0, b0, %3, f;\n\t"
            "@p tcgen05.mma.cta_group::2.kind::f16 [%0], a1, b1, %3, t;\n\t"
            "@p tcgen05.mma.cta_group::2.kind::f16 [%0], a2, b2, %3, t;\n\t"
            "@p tcgen05.mma.cta_group::2.kind::f16 [%0], a3, b3, %3, t;\n\t"
            "@p tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%5], %10;\n\t}\n" ::"r"(d),
            "r"(la), "r"(lb), "r"(idesc), "r"(issue), "r"(stage_bar), "r"(accumulate), "n"(kStepA), "n"(kStepB), "r"(kDescHigh),
            "h"(static_cast<unsigned short>(3u << leader)) : "memory");
}

template <int CG>
__device__ __forceinline__ void expert_load(uint32_t dst, const CUtensorMap *map, int x, int y, int z, uint32_t mbar) {
    if constexpr (CG == 1)
        asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
                     "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(mbar) : "memory");
    else
        asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
                     "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(mbar) : "memory");
}

// A tile: its expert, the expert's rows, and its place among the expert's tiles
struct ExpertTile {
    int expert, first, end;  // rows of the expert
    int tm, tn;              // along the rows of the output (weights: of the expert's matrix), and along its columns
};

// By one warp: the first row of every expert and the tiles ahead of it, both with one more entry behind the last.  A running maximum and a
// running sum, 32 experts at a time.
__device__ __forceinline__ void expert_tables(const ExpertArgs &a, int *firsts, int *tiles) {
    const int lane = threadIdx.x & 31;
    int row = 0, before = 0;
    if (lane == 0) firsts[0] = 0;
    if (tiles && lane == 0) tiles[0] = 0;
    for (int e0 = 0; e0 < a.experts; e0 += 32) {
        const int e = e0 + lane;
        int end = e < a.experts ? min(a.ends[e], a.rows) : 0;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int other = __shfl_up_sync(~0u, end, off);
            if (lane >= off) end = max(end, other);
        }
        end = max(end, row);
        const int start = __shfl_up_sync(~0u, end, 1);
        int count = end - (lane ? start : row);
        if (e >= a.experts) count = 0;
        int sum = (count + a.tile_rows - 1) / a.tile_rows;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int other = __shfl_up_sync(~0u, sum, off);
            if (lane >= off) sum += other;
        }
        if (e < a.experts) {
            firsts[e + 1] = end;
            if (tiles) tiles[e + 1] = before + sum;
        }
        row = __shfl_sync(~0u, end, 31);
        before += __shfl_sync(~0u, sum, 31);
    }
}

template <bool SWAP, bool OVER_ROWS>
__device__ __forceinline__ ExpertTile expert_tile(const ExpertArgs &a, const int *firsts, const int *tiles, int unit) {
    ExpertTile t;
    int r, rows_of_tiles;
    if constexpr (OVER_ROWS) {
        const int per = a.g.tiles_m * a.g.tiles_n;
        t.expert = unit / per;
        r = unit - t.expert * per;
        rows_of_tiles = a.g.tiles_m;
    } else {
        // the last expert whose tiles begin at or before this one's
        const int at = unit / a.g.tiles_n;
        int low = 0, high = a.experts;
        while (high - low > 1) {
            const int mid = (low + high) >> 1;
            if (tiles[mid] <= at) low = mid;
            else high = mid;
        }
        t.expert = low;
        r = unit - tiles[low] * a.g.tiles_n;
        rows_of_tiles = tiles[low + 1] - tiles[low];
    }
    t.first = firsts[t.expert];
    t.end = firsts[t.expert + 1];
    // groups of tile rows, down a group's columns: the rows' operand stays in L2 while the columns' passes by
    const int per_group = a.g.group * a.g.tiles_n, group = r / per_group, begin = group * a.g.group, height = min(a.g.group, rows_of_tiles - begin);
    r -= group * per_group;
    t.tm = begin + r % height;
    t.tn = r / height;
    return t;
}

// SWAP: weights along the accumulator's lanes, rows along its columns; the output is C transposed
template <bool A_MN, bool B_MN, int BN, int CG, bool SWAP, bool OVER_ROWS, int CTAS>
__global__ void __launch_bounds__(ExpertShape<A_MN, B_MN, BN, CG, SWAP, OVER_ROWS, CTAS>::kThreads, CTAS)
expert_gemm_kernel(const ExpertArgs x, const __grid_constant__ CUtensorMap a_map, const __grid_constant__ CUtensorMap b_map,
                   const __grid_constant__ CUtensorMap few_map) {
    using S = ExpertShape<A_MN, B_MN, BN, CG, SWAP, OVER_ROWS, CTAS>;
    const GemmArgs &g = x.g;
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) unsigned long long full[S::kStages], empty[S::kStages], acc_full[2], acc_empty[2];
    __shared__ __align__(8) unsigned long long last_full[OVER_ROWS ? S::kStages : 1], last_ready[OVER_ROWS ? S::kStages : 1];  // of an expert's last stage
    __shared__ int firsts[kMostExperts + 1], tiles[OVER_ROWS ? 1 : kMostExperts + 1];
    __shared__ uint32_t tmem_holder;
    __shared__ int abort_flag;
    const uint32_t smem = (smem_addr(smem_raw) + 1023u) & ~1023u;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = CG == 2 ? cluster_rank() : 0;  // the pair's first CTA leads
    const int start = blockIdx.x / CG, step = gridDim.x / CG;

    if (threadIdx.x == 32) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&a_map)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&b_map)) : "memory");
    }
    if (threadIdx.x == 0) {
        abort_flag = 0;
        const auto init = [](unsigned long long *bar, uint32_t count) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(bar)), "r"(count) : "memory");
        };
        for (int s = 0; s < S::kStages; ++s) {
            init(&full[s], 1);
            init(&empty[s], 1);
            if constexpr (OVER_ROWS) {
                init(&last_full[s], 1);
                init(&last_ready[s], 2 * CG);
            }
        }
        for (int b = 0; b < 2; ++b) {
            init(&acc_full[b], 1);
            init(&acc_empty[b], 4 * S::kGroups * CG);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if constexpr (CG == 2) {  // an allocation for a pair takes columns on both SMs: the other CTA must have started
        __syncwarp();
        cluster_sync_all();
    }
    if (warp == 2) {
        if constexpr (CG == 1) {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_holder)), "r"(S::kTmemCols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_holder)), "r"(S::kTmemCols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        }
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (CG == 2) cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem = tmem_holder;
    after_previous();
    if (warp == 3) expert_tables(x, firsts, OVER_ROWS ? nullptr : tiles);
    __syncthreads();
    const int units = OVER_ROWS ? x.experts * g.tiles_m * g.tiles_n : tiles[x.experts] * g.tiles_n;
    // stages of a tile, and the rows that its last one has (64 where it is whole)
    const auto stages_of = [&](const ExpertTile &t) { return ((OVER_ROWS ? t.end - t.first : x.k) + S::kK - 1) / S::kK; };
    const auto rest_of = [&](const ExpertTile &t) { return OVER_ROWS ? (t.end - t.first) % S::kK : 0; };

    if (warp == 0) {
        // ---- operands ----
        int it = 0;
        bool ok = true;
        for (int unit = start; unit < units && ok; unit += step) {
            const ExpertTile t = expert_tile<SWAP, OVER_ROWS>(x, firsts, tiles, unit);
            // where this CTA's operand rows begin: lanes (A) and columns (B); rows of an expert count from its first
            const int lane0 = (t.tm * CG + static_cast<int>(rank)) * kGemmRows, column0 = t.tn * BN + static_cast<int>(rank) * S::kBRows;
            const int a0 = SWAP ? t.tn * kGemmRows : OVER_ROWS ? lane0 : t.first + lane0, b0 = SWAP ? t.first + t.tm * BN : column0;
            const int az = SWAP ? t.expert : 0, bz = SWAP || OVER_ROWS ? 0 : t.expert;
            const int stages = stages_of(t), rest = rest_of(t);
            // An expert's last rows come 32 at a time, and those behind its end from outside of all rows: zeros, which cost no traffic and little power
            const bool few = !SWAP && !OVER_ROWS && a0 + kGemmRows > t.end;
            for (int kt = 0; kt < stages; ++kt, ++it) {
                const int s = it % S::kStages;
                const bool got = lane_wait(smem_addr(&empty[s]), ((it / S::kStages) & 1) ^ 1, &abort_flag);
                if (elect_one() && got) {
                    const uint32_t mine = smem_addr(&full[s]);
                    const bool partial = OVER_ROWS && rest && kt == stages - 1;
                    uint32_t bar = CG == 2 ? in_cta(mine, 0) : mine;
                    if (rank == 0) {
                        if (partial) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(mine) : "memory");  // nothing of it is waited for there
                        else asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(mine), "r"(static_cast<uint32_t>(CG * S::kStage)) : "memory");
                    }
                    if constexpr (OVER_ROWS) {
                        if (partial) {  // each CTA clears its own rows: it has to see its own boxes arrive
                            bar = smem_addr(&last_full[s]);
                            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(static_cast<uint32_t>(S::kStage)) : "memory");
                        }
                    }
                    const uint32_t a = smem + s * S::kStage, b = a + S::kABytes;
                    const int k = OVER_ROWS ? t.first + kt * S::kK : kt * S::kK;
                    if constexpr (A_MN) {
                        expert_load<CG>(a, &a_map, a0, k, az, bar);
                        expert_load<CG>(a + kBoxBytes, &a_map, a0 + 64, k, az, bar);
                    } else if (few) {
#pragma unroll
                        for (int r = 0; r < kGemmRows; r += 32) expert_load<CG>(a + r * 128, &few_map, k, a0 + r < t.end ? a0 + r : x.rows, az, bar);
                    } else {
                        expert_load<CG>(a, &a_map, k, a0, az, bar);
                    }
                    if constexpr (B_MN) {
#pragma unroll
                        for (int j = 0; j < S::kBRows / 64; ++j) expert_load<CG>(b + j * kBoxBytes, &b_map, b0 + 64 * j, k, bz, bar);
                    } else {
                        expert_load<CG>(b, &b_map, k, b0, bz, bar);
                    }
                }
                ok = __all_sync(~0u, got);
                if (!ok) break;
            }
        }
    } else if (warp == 1) {
        // ---- MMAs ----
        if (rank == 0) {
            int it = 0, done = 0;
            uint32_t last_phase = 0;
            bool ok = true;
            const uint32_t issue = elect_one() ? 1u : 0u;
            __syncwarp();
            for (int unit = start; unit < units && ok; unit += step) {
                const ExpertTile t = expert_tile<SWAP, OVER_ROWS>(x, firsts, tiles, unit);
                const int stages = stages_of(t), rest = rest_of(t);
                if (stages == 0) continue;  // an expert without rows: zeros, which need no accumulator
                const int buf = done & 1;
                ok = gemm_wait(smem_addr(&acc_empty[buf]), ((done >> 1) & 1) ^ 1, &abort_flag);
                if (!ok) break;
                tc_fence_after();
                const uint32_t d = tmem + buf * BN;
                for (int kt = 0; kt < stages; ++kt, ++it) {
                    const int s = it % S::kStages;
                    ok = gemm_wait(smem_addr(&full[s]), (it / S::kStages) & 1, &abort_flag);
                    if constexpr (OVER_ROWS) {
                        if (ok && rest && kt == stages - 1) {
                            ok = gemm_wait<CG == 2>(smem_addr(&last_ready[s]), (last_phase >> s) & 1, &abort_flag);
                            last_phase ^= 1u << s;
                        }
                    }
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t a = smem + s * S::kStage;
                    expert_stage<CG, A_MN, B_MN>(d, a, a + S::kABytes, g.idesc, kt > 0 ? 1u : 0u, issue, smem_addr(&empty[s]), 0);
                    if (kt == stages - 1 && issue) gemm_commit<CG>(smem_addr(&acc_full[buf]), 0);
                    __syncwarp();
                }
                ++done;
            }
        }
    } else if (warp < 4) {
        // ---- rows of an expert's last stage that are not its own ----
        if constexpr (OVER_ROWS) {
            int it = 0;
            uint32_t last_phase = 0;
            bool ok = true;
            for (int unit = start; unit < units && ok; unit += step) {
                const ExpertTile t = expert_tile<SWAP, OVER_ROWS>(x, firsts, tiles, unit);
                const int stages = stages_of(t), rest = rest_of(t);
                it += stages;
                if (!rest) continue;
                const int s = (it - 1) % S::kStages;
                ok = gemm_wait(smem_addr(&last_full[s]), (last_phase >> s) & 1, &abort_flag);
                if (!ok) break;
                last_phase ^= 1u << s;
                // boxes of 64 rows of 128 bytes; the swizzle stays within a row
                const uint32_t at = smem + s * S::kStage + (threadIdx.x - 64) * 16;
#pragma unroll
                for (int box = 0; box < S::kStage / kBoxBytes; ++box)
                    for (int r = rest - rest % 8; r < S::kK; r += 8)
                        if (r + static_cast<int>(threadIdx.x - 64) / 8 >= rest) st_shared_16(at + box * kBoxBytes + r * 128, make_uint4(0, 0, 0, 0));
                fence_async_smem();
                __syncwarp();
                if (lane == 0) {
                    const uint32_t bar = smem_addr(&last_ready[s]);
                    // the leader's MMAs read this CTA's boxes and the zeros in them: a release to the cluster, once an expert's tile
                    if constexpr (CG == 2) asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(in_cta(bar, 0)) : "memory");
                    else asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
                }
            }
        }
    } else {
        // ---- sums -> output ----
        const int quarter = warp & 3, group = (warp - 4) >> 2;
        const uint32_t staging = smem + S::kStages * S::kStage + (warp - 4) * kPieceBytes;
        constexpr int kStep = S::kColumns < 32 ? S::kColumns : 32;
        int done = 0;
        bool ok = true;
        for (int unit = start; unit < units && ok; unit += step) {
            const ExpertTile t = expert_tile<SWAP, OVER_ROWS>(x, firsts, tiles, unit);
            const bool none = OVER_ROWS && t.end == t.first;
            const int buf = done & 1;
            if (!none) {
                ok = gemm_wait(smem_addr(&acc_full[buf]), (done >> 1) & 1, &abort_flag);
                if (!ok) break;
                tc_fence_after();
                ++done;
            }
            // lanes and columns of this warp's part in the output, and where the output's rows end
            const int lane0 = SWAP ? t.tn * kGemmRows + 32 * quarter : (t.tm * CG + static_cast<int>(rank)) * kGemmRows + 32 * quarter;
            const int row0 = OVER_ROWS ? t.expert * g.m + lane0 : t.first + lane0, rows_end = OVER_ROWS ? (t.expert + 1) * g.m : t.end;
            const int column0 = SWAP ? t.first + t.tm * BN : t.tn * BN + group * S::kColumns;
            unsigned short *row = static_cast<unsigned short *>(g.out) + static_cast<long long>(row0 + lane) * g.out_stride;
            const uint32_t d = tmem + buf * BN + group * S::kColumns + (static_cast<uint32_t>(32 * quarter) << 16);
#pragma unroll 1
            for (int c0 = 0; c0 < S::kColumns; c0 += kStep) {
                uint32_t raw[32];
                if (none) {
#pragma unroll
                    for (int k = 0; k < 32; ++k) raw[k] = 0;
                } else {
                    if constexpr (kStep == 32) tmem_ld32(d + c0, raw);
                    else tmem_ld16(d + c0, raw);
                    tmem_ld_wait();
                    if (c0 + kStep >= S::kColumns) {
                        // the accumulator is read: the next tile but one may fill it
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) {
                            // What is handed over lies in tensor memory, ordered by the fence above: a release to the cluster would also wait for the
                            // results that are on their way to global memory
                            if constexpr (CG == 2)
                                asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(in_cta(smem_addr(&acc_empty[buf]), 0)) : "memory");
                            else
                                asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(&acc_empty[buf])) : "memory");
                        }
                    }
                }
                if constexpr (SWAP) {
                    const int m = lane0 + lane;
                    if (m < g.n) {
#pragma unroll
                        for (int k = 0; k < kStep; ++k)
                            if (column0 + c0 + k < t.end)
                                store_one(g.out, static_cast<long long>(column0 + c0 + k) * g.out_stride + m, __uint_as_float(raw[k]), g.out_dtype);
                    }
                } else {
                    const int at = column0 + c0;
                    if (at >= g.n || row0 >= rows_end) continue;
                    uint32_t v[16];
#pragma unroll
                    for (int k = 0; k < 16; ++k) v[k] = pack_out(__uint_as_float(raw[2 * k]), __uint_as_float(raw[2 * k + 1]), g.out_dtype);
                    if (g.out_tma && at + 32 <= g.n) {
                        if (row0 + lane < rows_end) {
                            store_32(reinterpret_cast<unsigned char *>(row + at), v, g.out_tma);
                            store_32(reinterpret_cast<unsigned char *>(row + at + 16), v + 8, g.out_tma);
                        }
                    } else {
                        copy_piece(g, staging, v, row0, rows_end, at, 2);
                        if (at + 16 < g.n) copy_piece(g, staging, v + 8, row0, rows_end, at + 16, 2);
                    }
                }
            }
        }
        if constexpr (!OVER_ROWS) {
            // ---- rows behind the last expert: zeros, by all CTAs ----
            const int behind = firsts[x.experts], width = g.n;
            const long long stride = g.out_stride;
            unsigned short *out = static_cast<unsigned short *>(g.out);
            const bool wide = g.out_tma && width % 8 == 0;
            const int per_row = wide ? width / 8 : width;
            const long long total = static_cast<long long>(x.rows - behind) * per_row;
            for (long long i = static_cast<long long>(blockIdx.x) * (S::kThreads - 128) + threadIdx.x - 128; i < total; i += static_cast<long long>(gridDim.x) * (S::kThreads - 128)) {
                const long long r = i / per_row;
                const int c = static_cast<int>(i - r * per_row);
                if (wide) *reinterpret_cast<uint4 *>(out + (behind + r) * stride + 8 * c) = make_uint4(0, 0, 0, 0);
                else out[(behind + r) * stride + c] = 0;
            }
        }
    }
    __syncthreads();
    if (abort_flag && threadIdx.x == 0) {
        drain_copies(full, S::kStages);
        if constexpr (OVER_ROWS) drain_copies(last_full, S::kStages);
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (CG == 2) cluster_sync_all();
    if (warp == 2) {
        if constexpr (CG == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::kTmemCols) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::kTmemCols) : "memory");
    }
    if constexpr (CG == 2) {  // and neither CTA ends before both have given theirs back
        __syncwarp();
        cluster_sync_all();
    }
}

// ---- host ---------------------------------------------------------------------------------------------------

// Matrices of `outer` rows of `inner` 16-bit elements, `count` of them; boxes of 64 elements x box_outer rows in the 128-byte swizzle
bool expert_map(CUtensorMap *map, const void *base, long long inner, long long outer, long long stride, long long count, long long apart, int box_outer) {
    EncodeTiledFn encode = encode_tiled_fn();
    if (!encode || !aligned_to(base, 16) || stride % 8 || apart % 8) return false;
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(outer), static_cast<cuuint64_t>(count)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(stride) * 2, static_cast<cuuint64_t>(count > 1 ? apart : outer * stride) * 2};
    const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_outer), 1};
    const cuuint32_t elem[3] = {1, 1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<void *>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The operands of a product as they lie in memory: rows of `inner` elements, `count` matrices of them
struct ExpertOperand {
    const void *base;
    long long inner, outer, stride, count, apart;
};

template <bool A_MN, bool B_MN, int BN, int CG, bool SWAP, bool OVER_ROWS, int CTAS>
int launch_experts(ExpertArgs x, const ExpertOperand &a, const ExpertOperand &b, bool bf16, cudaStream_t stream) {
    using S = ExpertShape<A_MN, B_MN, BN, CG, SWAP, OVER_ROWS, CTAS>;
    auto kernel = expert_gemm_kernel<A_MN, B_MN, BN, CG, SWAP, OVER_ROWS, CTAS>;
    // Once per thread and device, and ahead of the maps: it also makes the device's context current in this thread, which encoding
    // a map needs and an autograd thread may not have yet.
    static thread_local unsigned long long ready = 0;
    int device = 0;
    if (int rc = cuda_status(cudaGetDevice(&device), "cudaGetDevice")) return rc;
    if (device >= 64 || !(ready >> device & 1)) {
        if (int rc = cuda_status(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes), "cudaFuncSetAttribute(expert_gemm_kernel)"))
            return rc;
        if (device < 64) ready |= 1ull << device;
    }
    CUtensorMap a_map, b_map, few_map;
    const auto operand = [](CUtensorMap *map, const ExpertOperand &o, bool mn, int box_rows) {
        return expert_map(map, o.base, o.inner, o.outer, o.stride, o.count, o.apart, mn ? 64 : box_rows);
    };
    if (!operand(&a_map, a, A_MN, kGemmRows) || !operand(&b_map, b, B_MN, S::kBRows))
        return fail(TH_ERR_ALIGNMENT, "product of experts: operand rows must start on 16 bytes");
    if (SWAP || OVER_ROWS) few_map = a_map;  // not looked at
    else if (!operand(&few_map, a, false, 32)) return fail(TH_ERR_ALIGNMENT, "product of experts: operand rows must start on 16 bytes");
    GemmArgs &g = x.g;
    x.tile_rows = SWAP ? BN : CG * kGemmRows;
    g.tiles_m = OVER_ROWS ? divide_up(g.m, CG * kGemmRows) : 0;
    g.tiles_n = SWAP ? divide_up(g.n, kGemmRows) : divide_up(g.n, BN);
    g.group = 16;  // 16 tile rows of 256 x 2048: 16 MB
    g.idesc = instr_desc(CG * kGemmRows, BN, bf16, A_MN, B_MN);
    g.out_tma = rows_start_on(g.out, g.out_stride, 2);
    // at most so many tiles: an expert's last one may be part of one
    const long long rows_of_tiles = OVER_ROWS ? static_cast<long long>(x.experts) * g.tiles_m : x.rows / x.tile_rows + std::min(x.experts, x.rows);
    const long long units = rows_of_tiles * g.tiles_n;
    if (units > 0x7fffffffll) return fail(TH_ERR_UNSUPPORTED, "product of experts: too many tiles");
    const long long clusters = std::min<long long>(units, std::max(1, CTAS * sm_count() / CG));
    return launch_chained("expert_gemm_kernel launch", kernel, static_cast<unsigned>(clusters * CG), S::kThreads, S::kBytes, stream, CG, x, a_map, b_map, few_map);
}

}  // namespace
}  // namespace th
