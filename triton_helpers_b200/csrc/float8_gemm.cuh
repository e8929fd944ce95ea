// Products of 8-bit floating-point blocks on tcgen05 (kind::f8f6f4), with a scale for every 128 of K on both sides:
//
//     C[m, n] = sum_b a_scale[m, b] b_scale[n, b] P_b[m, n]        P_b[m, n] = sum_{k in block b} A[m, k] B[n, k]
//
// A stage of K is one block, 128 bytes.  The tensor cores leave P_b in one of a few accumulators in tensor memory; eight warps take it out while
// they fill the next, and add it, times its scales, to sums that stay in their registers until the tile's K ends.  So what is summed in
// the tensor cores is one block, and the sums over blocks are ordinary float32 ones.
//
// One persistent CTA per SM, or one pair of CTAs on one 256-row tile (cta_group::2): warp 0 brings operands by TMA through a ring of stages,
// warp 1 issues the MMAs, warps 2 and 3 bring the scales, some blocks ahead, as products through a ring of their own, and warps 4 to 11 keep the
// sums, with the registers that the others leave them.  Operand tiles have rows of 128 bytes in the 128-byte swizzle; a weight whose rows are
// summed over (the input's gradient) is read MN-major as it lies, 128 rows x 128 columns a stage.
//
// Bound by a block's chain: the commit wakes the warps that keep sums, they read the accumulator in two parts and hand it back; 969 cycles for 256 x 256 x 128,
// of which 506 are MMAs.  8192 x 4096 -> 4096 142 us (1.9 PFLOP/s), -> 16384 533 us (2.06; in a loop, at the board's power limit, 620).
//
// Few tokens lie along the accumulator's columns, with 128 weight rows, one row of weight blocks, on its lanes; K is then split over the CTAs
// of a cluster, as it is for few tiles (wide_gemm.cuh).
#pragma once

#include "wide_gemm.cuh"

namespace th {
namespace {

constexpr int kF8Block = 128;
constexpr int kF8Step = 64;        // columns of an accumulator that a warp reads at a time
constexpr int kF8Batch = 4;        // blocks whose scales a warp asks for at a time

struct F8Scale {
    const float *at;
    long long row, block;  // strides: rows (or blocks of 128 rows) and blocks of K
};

struct F8Gemm {
    GemmArgs g;
    F8Scale tokens, weight;
};

// CTAS: CTAs that share an SM
template <int BN, int CG, bool SWAP, int CTAS>
struct F8Shape {
    static constexpr int kBRows = BN / CG;
    static constexpr int kABytes = kGemmRows * 128, kBBytes = kBRows * 128, kStage = kABytes + kBBytes;
    static constexpr int kGroups = 2;  // of four warps that keep sums
    static constexpr int kWarps = 4 * kGroups, kThreads = 128 + 32 * kWarps;
    static constexpr int kStaging = SWAP ? 0 : kWarps * kPieceBytes;
    static constexpr int kFactors = SWAP ? BN : kGemmRows * (BN == 256 ? 2 : 1);  // of a block: a token's for every row of weight blocks
    static constexpr int kFitAccs = 512 / CTAS / BN, kAccs = kFitAccs > 4 ? 4 : kFitAccs;  // accumulators in tensor memory's 512 columns
    static constexpr int kSlots = 4 * kAccs;  // blocks whose factors are held
    static constexpr int kSmem = (CTAS == 1 ? 226 : 112) * 1024 - 2 * BN * 4 - kSlots * 2 * kFactors * 4;  // biases, factors and barriers are beside it
    static constexpr int kFit = (kSmem - kStaging - 1024) / kStage;
    static constexpr int kStages = kFit > 8 ? 8 : kFit;
    static constexpr int kBytes = kStages * kStage + kStaging + 1024;
    static constexpr int kTmemCols = kAccs * BN < 32 ? 32 : kAccs * BN;
    static constexpr int kColumns = BN / kGroups;  // of each group
    static constexpr bool kSplits = kGemmRows * BN * 4 <= kStages * kStage;
    // Registers a thread: at launch what the SM's 65536 allow; then the first four warps give theirs to those that keep sums
    static constexpr int kLaunchRegs = CTAS == 1 ? 168 : 80, kFewRegs = CTAS == 1 ? 56 : 40, kSumRegs = CTAS == 1 ? 224 : 96;
    static_assert(kFewRegs + kGroups * kSumRegs <= (1 + kGroups) * kLaunchRegs, "more registers than the launch has");
    static_assert(kStages >= 3 && kAccs >= 2 && CTAS * kTmemCols <= 512, "tile does not fit");
};

// kind::f8f6f4 instruction descriptor: e4m3 operands, float32 sums
__host__ __device__ constexpr uint32_t instr_desc_e4m3(int m, int n, bool b_mn) {
    return (1u << 4) | (static_cast<uint32_t>(b_mn) << 16) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

// A block's four MMAs, then the commits to its accumulator's and its stage's barriers, by the lane whose `issue` is not zero.  The instructions are
// predicated and the warp stays together: behind a branch for one lane the four and their commits took longer (see the kernel).
template <int CG, bool B_MN>
__device__ __forceinline__ void f8_block(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t issue, uint32_t done_bar, uint32_t stage_bar, uint32_t leader) {
    constexpr uint32_t kLeading = B_MN ? (128u * 128u >> 4) << 16 : 0u;  // an MN-major operand of 256 columns lies in two boxes of 128
    constexpr uint32_t kStepB = B_MN ? 32 * 128 >> 4 : 2;
    const uint32_t la = desc_low(a), lb = desc_low(b) | kLeading;
    if constexpr (CG == 1)
        asm volatile(
            "{\n\t.reg .pred p, t, f;\n\t.reg .b64 a0, a1, a2, a3, b0, b1, b2, b3;\n\t"
            "setp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 t, 0, 0;\n\tsetp.ne.b32 f, 0, 0;\n\t"
            "mov.b64 a0, {%1, %8};\n\tadd.s64 a1, a0, 2;\n\tadd.s64 a2, a0, 4;\n\tadd.s64 a3, a0, 6;\n\t"
            "mov.b64 b0, {%2, %8};\n\tadd.s64 b1, b0, %7;\n\tadd.s64 b2, b1, %7;\n\tadd.s64 b3, b2, %7;\n\t"
            "@p tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a0, b0, %3, f;\n\t"
            "@p tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a1, b1, %3, t;\n\t"
            "@p tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a2, b2, %3, t;\n\t"
            "@p tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a3, b3, %3, t;\n\t"
            "@p tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%5];\n\t"
            "@p tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%6];\n\t}\n" ::"r"(d),
            "r"(la), "r"(lb), "r"(idesc), "r"(issue), "r"(done_bar), "r"(stage_bar), "n"(kStepB), "r"(kDescHigh) : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p, t, f;\n\t.reg .b64 a0, a1, a2, a3, b0, b1, b2, b3;\n\t"
            "setp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 t, 0, 0;\n\tsetp.ne.b32 f, 0, 0;\n\t"
            "mov.b64 a0, {%1, %8};\n\tadd.s64 a1, a0, 2;\n\tadd.s64 a2, a0, 4;\n\tadd.s64 a3, a0, 6;\n\t"
            "mov.b64 b0, {%2, %8};\n\tadd.s64 b1, b0, %7;\n\tadd.s64 b2, b1, %7;\n\tadd.s64 b3, b2, %7;\n\t"
            "@p tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], a0, b0, %3, f;\n\t"
            "@p tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], a1, b1, %3, t;\n\t"
            "@p tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], a2, b2, %3, t;\n\t"
            "@p tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], a3, b3, %3, t;\n\t"
            "@p tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%5], %9;\n\t"
            "@p tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%6], %9;\n\t}\n" ::"r"(d),
            "r"(la), "r"(lb), "r"(idesc), "r"(issue), "r"(done_bar), "r"(stage_bar), "n"(kStepB), "r"(kDescHigh), "h"(static_cast<unsigned short>(3u << leader)) : "memory");
}

// The scales' product is one factor where it is between 2^-100 and 2^100.  Where it is not (it may be no float32 at all) a sum takes two factors
// one after the other, of about its square root each: results are then lost only where they are no float32 themselves.  The second one, of the rests that
// split_scale leaves, is beyond float32 itself where both scales are near its end (2^126 and up).  Every sum but zero is then infinite (sums of products are 2^-18 at
// least, the first factor 2^126): the largest float32 in its place says so too, and leaves a sum of zero at zero.
__device__ __forceinline__ float rests_of(float a, float b) {
    const float product = a * b;
    return isinf(product) && isfinite(a) && isfinite(b) ? copysignf(0x1.fffffep127f, product) : product;
}

// Two neighbouring columns' float32 values as one operand of packed arithmetic.  Volatile: what works on values read from tensor memory stays behind the
// wait for them.
__device__ __forceinline__ unsigned long long pair_of(uint32_t lo, uint32_t hi) {
    unsigned long long v;
    asm volatile("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(lo), "r"(hi));
    return v;
}
__device__ __forceinline__ float2 floats_of(unsigned long long v) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
    return f;
}
__device__ __forceinline__ unsigned long long fma_pair(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long d;
    asm volatile("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ unsigned long long mul_pair(unsigned long long a, unsigned long long b) {
    unsigned long long d;
    asm volatile("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// N neighbouring columns of this warp's lanes; they are there after tmem_ld_wait()
template <int N>
__device__ __forceinline__ void f8_read(uint32_t taddr, uint32_t (&v)[N]) {
    if constexpr (N >= 32) {
#pragma unroll
        for (int c = 0; c < N; c += 32) tmem_ld32(taddr + c, *reinterpret_cast<uint32_t(*)[32]>(v + c));
    } else if constexpr (N == 16) {
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                     : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
                       "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                     : "r"(taddr)
                     : "memory");
    } else {
        tmem_ld8_at(taddr, v);
    }
}

__device__ __forceinline__ unsigned long long add_pair(unsigned long long a, unsigned long long b) {
    unsigned long long d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// Where a tile's scales lie: the rows of tokens, and the block (or blocks) of weight rows beside them
template <bool B_MN, int BN, bool SWAP>
struct F8Tile {
    const float *tokens, *weight;
    long long token_block, weight_block, token_row, weight_row;
    int token0, tokens_end, weights_end;

    __device__ __forceinline__ F8Tile(const F8Gemm &f, const GemmUnit &u, int m0) {
        token0 = SWAP ? u.tn * BN : m0;
        const int weight0 = SWAP ? u.tm : u.tn * BN / kF8Block;
        tokens_end = SWAP ? f.g.n : f.g.m;
        weights_end = (SWAP ? f.g.m : f.g.n) - 1;
        token_row = f.tokens.row;
        token_block = f.tokens.block;
        // where K goes along a weight's rows its blocks are numbered the other way round
        weight_row = B_MN ? f.weight.block : f.weight.row;
        weight_block = B_MN ? f.weight.row : f.weight.block;
        tokens = f.tokens.at + token0 * token_row;
        weight = f.weight.at + weight0 * weight_row;
        weights_end = weights_end / kF8Block - weight0;
    }
    __device__ __forceinline__ float token(int t, int kt) const { return tokens[min(t, tokens_end - 1 - token0) * token_row + kt * token_block]; }
    __device__ __forceinline__ float of_weight(int group, int kt) const { return weight[min(group, weights_end) * weight_row + kt * weight_block]; }
};

// SWAP: A is the weight, and the output is C transposed (A's rows are its columns).
template <bool B_MN, int BN, int CG, bool SWAP, int CTAS>
__global__ void __launch_bounds__(F8Shape<BN, CG, SWAP, CTAS>::kThreads, CTAS)
float8_gemm_kernel(const F8Gemm f, const __grid_constant__ CUtensorMap a_map, const __grid_constant__ CUtensorMap b_map) {
    using S = F8Shape<BN, CG, SWAP, CTAS>;
    static_assert(!B_MN || S::kBRows % 128 == 0, "an MN-major box holds 128 columns");
    const GemmArgs &g = f.g;
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) unsigned long long full[S::kStages], empty[S::kStages], acc_full[S::kAccs], acc_empty[S::kAccs];
    __shared__ __align__(16) float factors[S::kSlots][2][S::kFactors];
    __shared__ int far_factors[S::kSlots];
    __shared__ __align__(16) float biases[2][BN];  // read two at a time
    __shared__ uint32_t tmem_holder;
    __shared__ int abort_flag;
    const uint32_t smem = (smem_addr(smem_raw) + 1023u) & ~1023u;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // within the tile: the pair's first CTA leads; the cluster holds one tile's CTAs for every part of K
    const uint32_t place = CG == 2 ? cluster_rank() : 0, rank = place % CG, leader = place - rank;
    const int units = g.tiles_m * g.tiles_n * g.splits, first = blockIdx.x / CG, step = gridDim.x / CG;

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
        }
        for (int b = 0; b < S::kAccs; ++b) {
            init(&acc_full[b], 2);  // the block's MMAs and its scales
            init(&acc_empty[b], S::kWarps * CG);
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
    int ahead = 0;  // stages whose A is on its way already
    if constexpr (SWAP) {
        if (warp == 0 && g.early && first < units) {
            const GemmUnit u = gemm_unit(g, first);
            ahead = min(S::kStages, u.k1 - u.k0);
            if (elect_one()) {
                for (int s = 0; s < ahead; ++s) {
                    const uint32_t bar = smem_addr(&full[s]);
                    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(static_cast<uint32_t>(S::kStage)) : "memory");
                    gemm_load<CG>(smem + s * S::kStage, &a_map, (u.k0 + s) * kF8Block, u.tm * kGemmRows, bar);
                }
            }
            __syncwarp();
        }
    }
    after_previous();

    // Each side of the branch has its registers, so that a split tile is finished within it
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::kFewRegs));
        if (warp == 0) {
            // ---- operands ----
            int it = 0;
            bool ok = true;
            for (int unit = first; unit < units && ok; unit += step) {
                const GemmUnit u = gemm_unit(g, unit);
                const int m0 = (u.tm * CG + static_cast<int>(rank)) * kGemmRows, n0 = u.tn * BN + static_cast<int>(rank) * S::kBRows;
                for (int kt = u.k0; kt < u.k1; ++kt, ++it) {
                    const int s = it % S::kStages;
                    const bool got = lane_wait(smem_addr(&empty[s]), ((it / S::kStages) & 1) ^ 1, &abort_flag);
                    if (elect_one() && got) {
                        const uint32_t mine = smem_addr(&full[s]), bar = CG == 2 ? in_cta(mine, leader) : mine;
                        if (rank == 0 && it >= ahead)
                            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(mine), "r"(static_cast<uint32_t>(CG * S::kStage)) : "memory");
                        const uint32_t a = smem + s * S::kStage, b = a + S::kABytes;
                        const int k = kt * kF8Block;
                        if (it >= ahead) gemm_load<CG>(a, &a_map, k, m0, bar);
                        if constexpr (B_MN) {
#pragma unroll
                            for (int j = 0; j < S::kBRows / 128; ++j) gemm_load<CG>(b + j * 128 * 128, &b_map, n0 + 128 * j, k, bar);
                        } else gemm_load<CG>(b, &b_map, k, n0, bar);
                    }
                    ok = __all_sync(~0u, got);
                    if (!ok) break;
                }
            }
        } else if (warp == 1) {
            // ---- MMAs ----
            if (rank == 0) {
                int it = 0;
                bool ok = true;
                const uint32_t issue = elect_one() ? 1u : 0u;
                __syncwarp();
                for (int unit = first; unit < units && ok; unit += step) {
                    const GemmUnit u = gemm_unit(g, unit);
                    for (int kt = u.k0; kt < u.k1 && ok; ++kt, ++it) {
                        const int s = it % S::kStages, buf = it % S::kAccs;
                        ok = gemm_wait(smem_addr(&full[s]), (it / S::kStages) & 1, &abort_flag);
                        if (!ok) break;
                        ok = gemm_wait(smem_addr(&acc_empty[buf]), ((it / S::kAccs) & 1) ^ 1, &abort_flag);
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t a = smem + s * S::kStage;
                        f8_block<CG, B_MN>(tmem + buf * BN, a, a + S::kABytes, g.idesc, issue, smem_addr(&acc_full[buf]), smem_addr(&empty[s]), leader);
                    }
                }
            }
        } else {
            // ---- scales: the even blocks' by one warp, the odd ones' by the other (one warp for all of them: 545 -> 590 us at 8192 x 4096 -> 16384) ----
            constexpr int kRows = (SWAP ? BN : kGemmRows) / 32 > 0 ? (SWAP ? BN : kGemmRows) / 32 : 1, kGroups = SWAP ? 1 : BN == 256 ? 2 : 1;
            int it0 = 0;
            bool ok = true;
            for (int unit = first; unit < units && ok; unit += step) {
                const GemmUnit u = gemm_unit(g, unit);
                const F8Tile<B_MN, BN, SWAP> tile(f, u, (u.tm * CG + static_cast<int>(rank)) * kGemmRows);
                for (int kt = u.k0 + ((it0 ^ warp) & 1); kt < u.k1 && ok; kt += 2 * kF8Batch) {
                    float token[kF8Batch][kRows], weight[kF8Batch][kGroups];
#pragma unroll
                    for (int b = 0; b < kF8Batch; ++b) {
                        const int at = min(kt + 2 * b, u.k1 - 1);
#pragma unroll
                        for (int r = 0; r < kRows; ++r) token[b][r] = tile.token(32 * r + lane, at);
#pragma unroll
                        for (int q = 0; q < kGroups; ++q) weight[b][q] = tile.of_weight(q, at);
                    }
#pragma unroll
                    for (int b = 0; b < kF8Batch; ++b) {
                        if (kt + 2 * b >= u.k1) break;
                        const int it = it0 + kt + 2 * b - u.k0, s = it % S::kSlots, buf = it % S::kAccs;
                        bool far = false;
                        // The accumulator's block before is complete.  So block it - 2 kAccs has been read out by every warp, and the blocks before it have been
                        // added: a slot that came round since is free.
                        static_assert(S::kSlots > 2 * S::kAccs, "a slot may still be in use");
                        if (it >= S::kAccs) ok = gemm_wait(smem_addr(&acc_full[buf]), ((it / S::kAccs) & 1) ^ 1, &abort_flag);
                        if (!ok) break;
#pragma unroll
                        for (int q = 0; q < kGroups; ++q)
#pragma unroll
                            for (int r = 0; r < kRows; ++r) {
                                const float size = fabsf(token[b][r] * weight[b][q]);
                                far |= size < 0x1p-100f || size > 0x1p100f;  // a NaN is not
                            }
                        far = __any_sync(~0u, far);
#pragma unroll
                        for (int q = 0; q < kGroups; ++q)
#pragma unroll
                            for (int r = 0; r < kRows; ++r) {
                                const int at = q * kGemmRows + 32 * r + lane;
                                if (32 * r + lane >= (SWAP ? BN : kGemmRows)) continue;
                                if (far) {
                                    const float2 x = split_scale(token[b][r]), y = split_scale(weight[b][q]);
                                    factors[s][0][at] = x.x * y.x;
                                    factors[s][1][at] = rests_of(x.y, y.y);
                                } else {
                                    factors[s][0][at] = token[b][r] * weight[b][q];
                                }
                            }
                        __syncwarp();
                        if (lane == 0) {
                            far_factors[s] = far;
                            asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(&acc_full[buf])) : "memory");
                        }
                    }
                }
                it0 += u.k1 - u.k0;
            }
        }
        if constexpr (S::kSplits) {
            if (g.splits > 1) {
                __syncwarp();
                cluster_sync_all();
                cluster_sync_all();
            }
        }
    } else {
        // ---- sums, and the output ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::kSumRegs));
        constexpr int kColumns = S::kColumns, kStep = kColumns < kF8Step ? kColumns : kF8Step, kChunks = kColumns / kStep;
        const int quarter = warp & 3, group = (warp - 4) >> 2, out_bytes = g.out_dtype == TH_F32 ? 4 : 2;
        const uint32_t staging = smem + S::kStages * S::kStage + (warp - 4) * kPieceBytes;
        int it = 0, done = 0;
        bool ok = true;
        const auto column = [&](int c) { return group * kColumns + c; };  // of the tile
        for (int unit = first; unit < units; unit += step, ++done) {
            const GemmUnit u = gemm_unit(g, unit);
            const int tile_m0 = (u.tm * CG + static_cast<int>(rank)) * kGemmRows, m0 = tile_m0 + 32 * quarter, n0 = u.tn * BN, m = m0 + lane;
            // double buffered: a warp that fills the next tile's values has met, at the barrier before, those that read the last but one's
            float *bias = biases[done & 1];
            for (int c = threadIdx.x - 128; c < BN; c += 32 * S::kWarps) bias[c] = !SWAP && g.bias && u.tn * BN + c < g.n ? bias_at(g.bias, g.bias_dtype, u.tn * BN + c) : 0.f;
            asm volatile("bar.sync 1, %0;" ::"n"(32 * S::kWarps) : "memory");
            if (!ok) continue;  // a wait gave up: the barriers are met all the same
            unsigned long long sums[kColumns / 2];
#pragma unroll
            for (int c = 0; c < kColumns / 2; ++c) sums[c] = 0;
#pragma unroll 1
            for (int kt = u.k0; kt < u.k1; ++kt, ++it) {
                const int buf = it % S::kAccs, slot = it % S::kSlots;
                ok = gemm_wait(smem_addr(&acc_full[buf]), (it / S::kAccs) & 1, &abort_flag);
                if (!ok) break;
                tc_fence_after();
                const uint32_t d = tmem + buf * BN + group * kColumns + (static_cast<uint32_t>(32 * quarter) << 16);
                uint32_t raw[kStep];
                f8_read<kStep>(d, raw);
                // a lane's (swapped, it is a column's, and read where it is used)
                constexpr bool kPairs = BN == 256;
                const float *of_lane = &factors[slot][0][SWAP ? group * kColumns : (kPairs ? group * kGemmRows : 0) + 32 * quarter + lane];
                unsigned long long both = 0;
                if constexpr (!SWAP) both = pair_of(__float_as_uint(*of_lane), __float_as_uint(*of_lane));
                const bool far = far_factors[slot] != 0;
#pragma unroll
                for (int chunk = 0; chunk < kChunks; ++chunk) {
                    tmem_ld_wait();
                    if (chunk + 1 == kChunks) {
                        // the accumulator is read: another block may fill it
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) {
                            // What is handed over lies in tensor memory, ordered by the fence above: a release to the cluster would also wait for
                            // everything that is on its way from and to global memory
                            if constexpr (CG == 2)
                                asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(in_cta(smem_addr(&acc_empty[buf]), leader)) : "memory");
                            else
                                asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(&acc_empty[buf])) : "memory");
                        }
                    }
                    unsigned long long *to = sums + chunk * kStep / 2;
                    const float *then = of_lane + S::kFactors;
                    if constexpr (SWAP) {
                        const ulonglong2 *of_columns = reinterpret_cast<const ulonglong2 *>(of_lane + chunk * kStep);
#pragma unroll
                        for (int c = 0; c < kStep / 4; ++c) {
                            const ulonglong2 four = of_columns[c];
                            const unsigned long long x = pair_of(raw[4 * c], raw[4 * c + 1]), y = pair_of(raw[4 * c + 2], raw[4 * c + 3]);
                            if (far) {
                                const ulonglong2 more = reinterpret_cast<const ulonglong2 *>(then + chunk * kStep)[c];
                                to[2 * c] = fma_pair(mul_pair(x, four.x), more.x, to[2 * c]);
                                to[2 * c + 1] = fma_pair(mul_pair(y, four.y), more.y, to[2 * c + 1]);
                            } else {
                                to[2 * c] = fma_pair(x, four.x, to[2 * c]);
                                to[2 * c + 1] = fma_pair(y, four.y, to[2 * c + 1]);
                            }
                        }
                    } else if (far) {
                        const unsigned long long more = pair_of(__float_as_uint(*then), __float_as_uint(*then));
#pragma unroll
                        for (int c = 0; c < kStep / 2; ++c) to[c] = fma_pair(mul_pair(pair_of(raw[2 * c], raw[2 * c + 1]), both), more, to[c]);
                    } else {
#pragma unroll
                        for (int c = 0; c < kStep / 2; ++c) to[c] = fma_pair(pair_of(raw[2 * c], raw[2 * c + 1]), both, to[c]);
                    }
                    if (chunk + 1 < kChunks) f8_read<kStep>(d + (chunk + 1) * kStep, raw);
                }
            }
            if (!ok) continue;
            if constexpr (S::kSplits) {
                if (g.splits > 1) {  // the operands have been read: their shared memory takes the sums
                    if constexpr (SWAP) {
#pragma unroll
                        for (int c = 0; c < kColumns; ++c)
                            if (n0 + column(c) < g.n)
                                asm volatile("st.shared.f32 [%0], %1;" ::"r"(exchange_at<32>(smem, column(c), 8 * quarter + (lane >> 2)) + 4 * (lane & 3)),
                                             "f"(c & 1 ? floats_of(sums[c / 2]).y : floats_of(sums[c / 2]).x) : "memory");
                    } else {
#pragma unroll
                        for (int j = 0; j < kColumns / 4; ++j)
                            st_shared_16(exchange_at<BN / 4>(smem, 32 * quarter + lane, column(4 * j) / 4),
                                         make_uint4(__float_as_uint(floats_of(sums[2 * j]).x), __float_as_uint(floats_of(sums[2 * j]).y),
                                                    __float_as_uint(floats_of(sums[2 * j + 1]).x), __float_as_uint(floats_of(sums[2 * j + 1]).y)));
                    }
                    continue;
                }
            }
            if constexpr (SWAP) {
                const float add = g.bias && m < g.m ? bias_at(g.bias, g.bias_dtype, m) : 0.f;
                if (m < g.m) {
#pragma unroll
                    for (int c = 0; c < kColumns; ++c)
                        if (n0 + column(c) < g.n)
                            store_one(g.out, static_cast<long long>(n0 + column(c)) * g.out_stride + m, (c & 1 ? floats_of(sums[c / 2]).y : floats_of(sums[c / 2]).x) + add,
                                      g.out_dtype);
                }
            } else {
                unsigned char *row = static_cast<unsigned char *>(g.out) + static_cast<long long>(m) * g.out_stride * out_bytes;
#pragma unroll
                for (int c0 = 0; c0 < kColumns; c0 += 16) {
                    const int at = column(c0);
                    if (n0 + at >= g.n) break;
                    if (g.bias) {
#pragma unroll
                        for (int c = 0; c < 8; ++c) sums[c0 / 2 + c] = add_pair(sums[c0 / 2 + c], *reinterpret_cast<const unsigned long long *>(&bias[at + 2 * c]));
                    }
                    uint32_t v[16];
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        const float2 two = floats_of(sums[c0 / 2 + c]);
                        if (out_bytes == 4) {
                            v[2 * c] = __float_as_uint(two.x);
                            v[2 * c + 1] = __float_as_uint(two.y);
                        } else {
                            v[c] = pack_out(two.x, two.y, g.out_dtype);
                        }
                    }
                    if (g.out_tma && n0 + at + 16 <= g.n) {  // a lane writes its row
                        if (m < g.m) {
                            unsigned char *to = row + static_cast<long long>(n0 + at) * out_bytes;
                            store_32(to, v, g.out_tma);
                            if (out_bytes == 4) store_32(to + 32, v + 8, g.out_tma);
                        }
                    } else {
                        copy_piece(g, staging, v, m0, g.m, n0 + at, out_bytes);
                        if (out_bytes == 4 && n0 + at + 8 < g.n) copy_piece(g, staging, v + 8, m0, g.m, n0 + at + 8, 4);
                    }
                }
            }
        }
        if constexpr (S::kSplits) {
            if (g.splits > 1) {
                // ---- a split tile: this CTA's part of it, from everybody's sums ----
                __syncwarp();
                cluster_sync_all();
                if (!abort_flag && threadIdx.x < 128 + kGemmThreads) {
                    const GemmUnit u = gemm_unit(g, first);
                    const float2 *none = nullptr;
                    const int thread = threadIdx.x - 128;
                    if (g.splits <= 2) finish_split<2, BN, CG, SWAP, 8, 2>(g, u, rank, smem, none, biases[0], thread);
                    else if (g.splits <= 4) finish_split<2, BN, CG, SWAP, 4, 4>(g, u, rank, smem, none, biases[0], thread);
                    else if constexpr (CG == 1) finish_split<2, BN, CG, SWAP, 2, 8>(g, u, rank, smem, none, biases[0], thread);
                }
                __syncwarp();
                cluster_sync_all();  // everybody's sums have been read
            }
        }
    }
    __syncthreads();
    if (abort_flag && threadIdx.x == 0) drain_copies(full, S::kStages);
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

struct F8Product {
    Operand tokens, weight;  // 8-bit rows; the weight's extent is the output's columns
    F8Scale token_scale, weight_scale;
    int k;
    const void *bias;
    void *out;
    long long out_stride;
    int out_dtype;
    int weights_settled;  // the weight was complete before the kernel ahead of this one began
};

template <bool B_MN, int BN, int CG, bool SWAP, int CTAS>
int launch_float8(const F8Product &p, int splits, cudaStream_t stream) {
    using S = F8Shape<BN, CG, SWAP, CTAS>;
    auto kernel = float8_gemm_kernel<B_MN, BN, CG, SWAP, CTAS>;
    // Once per thread and device, and ahead of the maps: it also makes the device's context current in this thread, which encoding
    // a map needs and an autograd thread may not have yet.
    static thread_local unsigned long long ready = 0;
    int device = 0;
    if (int rc = cuda_status(cudaGetDevice(&device), "cudaGetDevice")) return rc;
    if (device >= 64 || !(ready >> device & 1)) {
        if (int rc = cuda_status(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes), "cudaFuncSetAttribute(float8_gemm_kernel)"))
            return rc;
        cudaFuncAttributes attributes;
        if (int rc = cuda_status(cudaFuncGetAttributes(&attributes, kernel), "cudaFuncGetAttributes(float8_gemm_kernel)")) return rc;
        if (attributes.numRegs < S::kLaunchRegs) return fail(TH_ERR_UNSUPPORTED, "8-bit product: built with %d registers a thread", attributes.numRegs);
        if (device < 64) ready |= 1ull << device;
    }
    const Operand &a = SWAP ? p.weight : p.tokens, &b = SWAP ? p.tokens : p.weight;
    CUtensorMap a_map, b_map;
    if (!matrix_map(&a_map, a.base, p.k, a.rows, a.stride, 1, 128, kGemmRows) ||
        !(B_MN ? matrix_map(&b_map, b.base, b.rows, p.k, b.stride, 1, 128, 128) : matrix_map(&b_map, b.base, p.k, b.rows, b.stride, 1, 128, S::kBRows)))
        return fail(TH_ERR_ALIGNMENT, "8-bit product: operand rows must start on 16 bytes");
    F8Gemm f{};
    GemmArgs &g = f.g;
    f.tokens = p.token_scale;
    f.weight = p.weight_scale;
    g.m = a.rows;
    g.n = b.rows;
    g.tiles_m = divide_up(g.m, CG * kGemmRows);
    g.tiles_n = divide_up(g.n, BN);
    g.group = static_cast<int>(std::max(4ll, std::min(32ll, (32ll << 20) / (static_cast<long long>(CG) * kGemmRows * p.k))));  // 32 MB of rows (wide_gemm.cuh)
    g.k_tiles = divide_up(p.k, kF8Block);
    g.tiles_per_split = divide_up(g.k_tiles, splits);
    g.splits = divide_up(g.k_tiles, g.tiles_per_split);
    g.idesc = instr_desc_e4m3(CG * kGemmRows, BN, B_MN);
    g.out = p.out;
    g.out_stride = p.out_stride;
    g.out_dtype = g.bias_dtype = p.out_dtype;
    g.bias = p.bias;
    g.early = p.weights_settled;
    const int out_bytes = g.out_dtype == TH_F32 ? 4 : 2;
    if (g.splits > (S::kSplits ? 8 / CG : 1)) return fail(TH_ERR_UNSUPPORTED, "8-bit product: %d parts", g.splits);
    g.out_tma = rows_start_on(g.out, g.out_stride, out_bytes);
    const long long units = static_cast<long long>(g.tiles_m) * g.tiles_n * g.splits;
    if (units > 0x7fffffffll) return fail(TH_ERR_UNSUPPORTED, "8-bit product: too many tiles");
    // a split tile is one unit of every CTA of its cluster; otherwise CTAs go round the tiles
    const long long clusters = g.splits > 1 ? units : std::min<long long>(units, std::max(1, CTAS * sm_count() / CG));
    return launch_chained("float8_gemm_kernel launch", kernel, static_cast<unsigned>(clusters * CG), S::kThreads, S::kBytes, stream, CG * g.splits, f, a_map, b_map);
}

}  // namespace
}  // namespace th
