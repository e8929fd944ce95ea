// Matrix products of the layers for wide networks on tcgen05: 16-bit operands with float32 sums, 8-bit integers with 32-bit sums.
//
//     C[m, n] = sum_k A[m, k] B[n, k]          each operand K-major (k contiguous) or, in 16 bits, MN-major (m or n contiguous)
//
// One persistent CTA per SM, or one pair of CTAs on one 256-row tile (cta_group::2).  Warp 0 brings operand boxes by TMA through a ring
// of stages, warp 1 issues the MMAs, warps 4 to 7 empty one accumulator while the next tile fills the other.  Every operand
// tile has rows of 128 bytes in the 128-byte swizzle: K-major as one box of 128 bytes x rows, MN-major as boxes of 64 columns x 64 K rows.
//
// What bounds a tile is its operands' way into the SM, 64 bytes a cycle: a K step of 128 bytes takes a 128 x 128 tile of one CTA 512
// cycles (its MMAs 256), a 256 x 256 tile of a pair, which share the columns' operand, 512 as well (its MMAs 512).
//
// Few tiles: K is split over the CTAs of a cluster (up to eight), a tile a cluster.  Each leaves its sums in its shared memory and
// finishes a part of the tile from everybody's, added in rank order, so that there is no scratch, no second launch, and results repeat.
#pragma once

#include "chained.cuh"
#include "tc_tiles.cuh"

#include <algorithm>
#include <utility>

namespace th {
namespace {

constexpr int kGemmThreads = 256;
constexpr int kGemmRows = 128;                // accumulator rows of one CTA
constexpr int kBoxBytes = 64 * 128;           // 64 rows of 128 bytes
constexpr int kStagingBytes = 32 * 128;       // one epilogue warp's box: 32 rows of 128 bytes
constexpr int kStagingBoxes = 2;              // per warp: one is filled while the other is stored
constexpr unsigned long long kGemmWaitNs = 1000000000ull;

struct GemmArgs {
    int m, n, tiles_m, tiles_n, group, k_tiles, splits, tiles_per_split;
    uint32_t idesc;
    void *out;             // [m][out_stride], or [n][out_stride] where the product is transposed
    long long out_stride;
    int out_dtype;
    int out_tma;
    int early;             // A was complete before the kernel ahead passed its wait: its first stages are fetched while that one runs
    const float *lane_scale, *column_scale;  // along m and along n (8 bits)
    const void *bias;      // along n (along m where transposed)
    int bias_dtype;
};

// CTAS: CTAs that share an SM
template <int EB, bool A_MN, bool B_MN, int BN, int CG, int CTAS>
struct GemmShape {
    static constexpr int kK = 128 / EB;  // K elements of a stage
    static constexpr int kBRows = BN / CG;
    static constexpr int kABytes = kGemmRows * 128, kBBytes = kBRows * 128, kStage = kABytes + kBBytes;
    static constexpr int kFixed = CTAS == 1 ? 4 * kStagingBoxes * kStagingBytes : 0;  // transposed outputs have no staging
    static constexpr int kSmem = (CTAS == 1 ? 226 : 112) * 1024 - 2 * 3 * BN * 4;     // the scales, biases and barriers are beside it
    static constexpr int kFit = (kSmem - kFixed - 1024) / kStage;
    static constexpr int kStages = kFit > 8 ? 8 : kFit;
    static constexpr int kBytes = kStages * kStage + kFixed + 1024;
    static constexpr int kTmemCols = 2 * BN < 32 ? 32 : 2 * BN;
    static constexpr bool kSplits = kGemmRows * BN * 4 <= kStages * kStage;  // a tile's sums fit where the operands were
    static_assert(!(A_MN || B_MN) || EB == 2, "8-bit operands are K-major");
    static_assert(kStages >= 3 && CTAS * kTmemCols <= 512, "tile does not fit");
};

// kind::i8 instruction descriptor: signed 8-bit operands, 32-bit integer sums
__host__ __device__ constexpr uint32_t instr_desc_i8(int m, int n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

template <int EB, int CG>
__device__ __forceinline__ void gemm_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if constexpr (EB == 2 && CG == 1)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d), "l"(a), "l"(b),
                     "r"(idesc), "r"(accumulate) : "memory");
    else if constexpr (EB == 2)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d), "l"(a), "l"(b),
                     "r"(idesc), "r"(accumulate) : "memory");
    else if constexpr (CG == 1)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d), "l"(a), "l"(b),
                     "r"(idesc), "r"(accumulate) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d), "l"(a), "l"(b),
                     "r"(idesc), "r"(accumulate) : "memory");
}

// An MN-major operand of more than 64 elements lies in several boxes, whose distance is the descriptor's leading offset.
template <bool MN>
__device__ __forceinline__ uint64_t gemm_desc(uint32_t addr) {
    return smem_desc(MN ? desc_low(addr) | ((kBoxBytes >> 4) << 16) : desc_low(addr));
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t in_cta(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}

// A box into this CTA's shared memory, counted on the barrier `mbar` (a shared::cluster address; the pair's first CTA's for CG = 2)
template <int CG>
__device__ __forceinline__ void gemm_load(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t mbar) {
    if constexpr (CG == 1)
        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
                     "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(mbar) : "memory");
    else
        asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
                     "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(mbar) : "memory");
}

// The barrier at this offset in every CTA of the tile completes a phase once the MMAs issued so far have finished
template <int CG>
__device__ __forceinline__ void gemm_commit(uint32_t mbar, uint32_t leader) {
    if constexpr (CG == 1)
        mma_commit(mbar);
    else
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(mbar),
                     "h"(static_cast<unsigned short>(3u << leader)) : "memory");
}

// Bounded: a wait of a second raises the status word and the CTA's abort flag, which ends the other waits.  The answer is a lane's own: lanes may
// see the barrier and the flag in different orders.
__device__ __forceinline__ bool lane_wait(uint32_t bar, uint32_t parity, int *abort_flag) {
    unsigned long long deadline = 0;
    uint32_t done;
    for (unsigned poll = 0;; ++poll) {
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
                     : "=r"(done) : "r"(bar), "r"(parity) : "memory");
        if (done) break;
        if ((poll & 63u) == 63u) {
            if (*reinterpret_cast<volatile int *>(abort_flag)) break;
            unsigned long long now;
            asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
            if (deadline == 0) deadline = now + kGemmWaitNs;
            else if (now > deadline) {
                *reinterpret_cast<volatile int *>(abort_flag) = 1;
                g_tc_status = 1;
                break;
            }
        }
    }
    return done != 0;
}

// A whole warp's: what follows a wait is left by all of its lanes or by none
__device__ __forceinline__ bool gemm_wait(uint32_t bar, uint32_t parity, int *abort_flag) { return __all_sync(~0u, lane_wait(bar, parity, abort_flag)); }

struct GemmUnit {
    int tm, tn, split, k0, k1;
};

// Tiles go in groups of tile rows, down the group's columns: the rows' operand stays in L2 while the columns' passes by.
__device__ __forceinline__ GemmUnit gemm_unit(const GemmArgs &g, int unit) {
    GemmUnit u;
    const int tile = unit / g.splits;
    u.split = unit - tile * g.splits;
    const int per_group = g.group * g.tiles_n, group = tile / per_group, first = group * g.group, height = min(g.group, g.tiles_m - first);
    const int r = tile - group * per_group;
    u.tm = first + r % height;
    u.tn = r / height;
    u.k0 = u.split * g.tiles_per_split;
    u.k1 = min(g.k_tiles, u.k0 + g.tiles_per_split);
    return u;
}

__device__ __forceinline__ float bias_at(const void *bias, int dtype, int i) {
    if (dtype == TH_F32) return static_cast<const float *>(bias)[i];
    if (dtype == TH_F16) return __half2float(static_cast<const __half *>(bias)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16 *>(bias)[i]);
}

__device__ __forceinline__ uint32_t pack_out(float lo, float hi, int dtype) {
    return dtype == TH_F16 ? pack_pair<__half>(lo, hi) : pack_pair<__nv_bfloat16>(lo, hi);
}

// The 32 rows x 128 bytes that a warp has put into its staging box -> rows m0.., columns c0.. of the output.  Where rows do not start on
// 16 bytes a warp writes a row at a time, a word a lane, or two halves: eight rows are read ahead of their stores (3001 x 777 outputs of
// 1000 bfloat16 products: 32 us with each read ahead of its own store only, 16.5 so).
template <typename V, int PER>
__device__ __forceinline__ void copy_rows(unsigned char *to, long long pitch, uint32_t box, int rows, int cols) {
    const int lane = threadIdx.x & 31;
    for (int r0 = 0; r0 < rows; r0 += 8) {
        V v[8][PER];
#pragma unroll
        for (int r = 0; r < 8; ++r)
#pragma unroll
            for (int e = 0; e < PER; ++e) {
                const int at = (lane + 32 * e) * static_cast<int>(sizeof(V));
                const uint32_t from = box + (r0 + r) * 128 + ((((at >> 4) ^ r) << 4) | (at & 15));
                if constexpr (sizeof(V) == 4) asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v[r][e]) : "r"(from) : "memory");
                else asm volatile("ld.shared.b16 %0, [%1];" : "=h"(v[r][e]) : "r"(from) : "memory");
            }
#pragma unroll
        for (int r = 0; r < 8; ++r)
#pragma unroll
            for (int e = 0; e < PER; ++e)
                if (r0 + r < rows && lane + 32 * e < cols) reinterpret_cast<V *>(to + (r0 + r) * pitch)[lane + 32 * e] = v[r][e];
    }
}

__device__ __forceinline__ void store_box(const GemmArgs &g, const CUtensorMap *c_map, uint32_t box, int m0, int c0, int out_bytes) {
    if (g.out_tma) {
        fence_async_smem();
        __syncwarp();
        // a box outside the output is a group of its own all the same: the wait for a box's memory counts groups
        if ((threadIdx.x & 31) == 0) {
            if (m0 < g.m && c0 < g.n) tma_store_2d(c_map, box, c0, m0);
            else asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
        return;
    }
    __syncwarp();
    const int cols = min(128 / out_bytes, g.n - c0), rows = min(32, g.m - m0);
    const long long pitch = g.out_stride * out_bytes;
    unsigned char *to = static_cast<unsigned char *>(g.out) + m0 * pitch + static_cast<long long>(c0) * out_bytes;
    if (out_bytes == 4) copy_rows<uint32_t, 1>(to, pitch, box, rows, cols);
    else if (pitch % 4 == 0 && cols % 2 == 0 && (reinterpret_cast<uintptr_t>(to) & 3) == 0) copy_rows<uint32_t, 1>(to, pitch, box, rows, cols / 2);
    else copy_rows<unsigned short, 2>(to, pitch, box, rows, cols);
    __syncwarp();
}

// A scale as two factors of about its square root: a power of two, and the rest.  A sum takes both scales' powers first, then the product of
// the rests: neither the scales' product (2^-214 to 2^242 for 8-bit rows) nor a sum times one of them has to be a float32, only the result.  Where the
// product is an ordinary float32 the results are the same bits as with it: sum x powers is exact, and rounding the product of the rests rounds it.
__device__ __forceinline__ float2 split_scale(float scale) {
    const uint32_t power = ((__float_as_uint(scale) >> 23 & 255u) + 127u) >> 1;  // the exponents' fields: half of the scale's, with the same bias
    return make_float2(__uint_as_float(power << 23), scale * __uint_as_float((254u - power) << 23));
}

// One result from its sum
template <int EB>
__device__ __forceinline__ float finished(uint32_t raw, float2 row, float2 column, float bias) {
    if constexpr (EB == 1) return fmaf(static_cast<float>(static_cast<int>(raw)) * (row.x * column.x), row.y * column.y, bias);
    else return __uint_as_float(raw) + bias;
}

__device__ __forceinline__ void store_one(void *out, long long at, float v, int dtype) {
    if (dtype == TH_F32) static_cast<float *>(out)[at] = v;
    else if (dtype == TH_F16) static_cast<__half *>(out)[at] = __float2half_rn(v);
    else static_cast<__nv_bfloat16 *>(out)[at] = __float2bfloat16_rn(v);
}

// Sums of a split tile in shared memory, in pieces of four along the output's rows: `line` is an output row of the tile, `piece` four of
// its columns.  Writers have 32 lines (or, transposed, one line and 32 columns) a warp, readers one line: the swizzle serves both.
template <int PIECES>
__device__ __forceinline__ uint32_t exchange_at(uint32_t base, int line, int piece) {
    return base + (line * PIECES + (piece ^ (line & (PIECES < 8 ? PIECES - 1 : 7)))) * 16;
}

__device__ __forceinline__ uint4 ld_cluster_16(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared::cluster.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}

// This CTA's part of a split tile.  A read of another CTA's shared memory takes some 600 cycles, so PIECES_AT_ONCE x RANKS (16) of them are
// on their way together.
template <int EB, int BN, int CG, bool SWAP, int PIECES_AT_ONCE, int RANKS>
__device__ __forceinline__ void finish_split(const GemmArgs &g, const GemmUnit &u, uint32_t rank, uint32_t smem, const float2 *scales, const float *biases) {
    constexpr int kPieces = SWAP ? kGemmRows / 4 : BN / 4;
    const int m0 = (u.tm * CG + static_cast<int>(rank)) * kGemmRows, n0 = u.tn * BN, rows = max(0, min(kGemmRows, g.m - m0)), cols = min(BN, g.n - n0);
    const int lines = SWAP ? cols : rows, along = SWAP ? rows : cols, total = lines * kPieces;
    const int from = total * u.split / g.splits, to = total * (u.split + 1) / g.splits;
    for (int first = from + static_cast<int>(threadIdx.x); first < to; first += PIECES_AT_ONCE * kGemmThreads) {
        uint4 v[PIECES_AT_ONCE][RANKS];
#pragma unroll
        for (int p = 0; p < PIECES_AT_ONCE; ++p) {
            const int i = first + p * kGemmThreads;
            if (i < to) {
                const uint32_t at = exchange_at<kPieces>(smem, i / kPieces, i % kPieces);
#pragma unroll
                for (int r = 0; r < RANKS; ++r)
                    if (r < g.splits) v[p][r] = ld_cluster_16(in_cta(at, CG * r + rank));
            }
        }
#pragma unroll
        for (int p = 0; p < PIECES_AT_ONCE; ++p) {
            const int i = first + p * kGemmThreads, line = i / kPieces, piece = i % kPieces;
            if (i >= to || 4 * piece >= along) continue;
            uint32_t sum[4] = {v[p][0].x, v[p][0].y, v[p][0].z, v[p][0].w};
#pragma unroll
            for (int r = 1; r < RANKS; ++r) {
                if (r < g.splits) {
                    const uint32_t part[4] = {v[p][r].x, v[p][r].y, v[p][r].z, v[p][r].w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum[e] = EB == 1 ? sum[e] + part[e] : __float_as_uint(__uint_as_float(sum[e]) + __uint_as_float(part[e]));
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int c = 4 * piece + e;
                if (c >= along) break;
                const int mi = m0 + (SWAP ? c : line), ni = SWAP ? line : c;
                const float2 scale = EB == 1 ? split_scale(g.lane_scale[mi]) : make_float2(1.f, 1.f);
                const float bias = SWAP ? (g.bias ? bias_at(g.bias, g.bias_dtype, mi) : 0.f) : biases[ni];
                store_one(g.out, SWAP ? static_cast<long long>(n0 + line) * g.out_stride + mi : static_cast<long long>(m0 + line) * g.out_stride + n0 + c,
                          finished<EB>(sum[e], scale, scales[ni], bias), g.out_dtype);
            }
        }
    }
}

// SWAP: the output is C transposed (A's rows are its columns): few tokens, with the weights on the accumulator's rows.
template <int EB, bool A_MN, bool B_MN, int BN, int CG, bool SWAP, int CTAS>
__global__ void __launch_bounds__(kGemmThreads, CTAS)
wide_gemm_kernel(const GemmArgs g, const __grid_constant__ CUtensorMap a_map, const __grid_constant__ CUtensorMap b_map,
                 const __grid_constant__ CUtensorMap c_map) {
    using S = GemmShape<EB, A_MN, B_MN, BN, CG, CTAS>;
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) unsigned long long full[S::kStages], empty[S::kStages], acc_full[2], acc_empty[2];
    __shared__ float2 scales[2][BN];
    __shared__ float biases[2][BN];
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
        for (int b = 0; b < 2; ++b) {
            init(&acc_full[b], 1);
            init(&acc_empty[b], 4 * CG);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if constexpr (CG == 2) {
        // An allocation for a pair takes columns on both SMs: the other CTA must have started.  Without this, with other streams' CTAs starting at the same
        // time, one pair in some 10^5 to 10^6 launches never got past it, and the GPU stood still.  (The meeting costs some 0.2 us a launch.)
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
                    gemm_load<CG>(smem + s * S::kStage, &a_map, (u.k0 + s) * S::kK, u.tm * kGemmRows, bar);
                }
            }
            __syncwarp();
        }
    }
    after_previous();

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
                    const int k = kt * S::kK;
                    if constexpr (A_MN) {
                        gemm_load<CG>(a, &a_map, m0, k, bar);
                        gemm_load<CG>(a + kBoxBytes, &a_map, m0 + 64, k, bar);
                    } else if (it >= ahead) {
                        gemm_load<CG>(a, &a_map, k, m0, bar);
                    }
                    if constexpr (B_MN) {
#pragma unroll
                        for (int j = 0; j < S::kBRows / 64; ++j) gemm_load<CG>(b + j * kBoxBytes, &b_map, n0 + 64 * j, k, bar);
                    } else {
                        gemm_load<CG>(b, &b_map, k, n0, bar);
                    }
                }
                ok = __all_sync(~0u, got);  // the lanes agree behind the issue (one token, 8192 -> 8192 in 8 bits: 14.2 us with the vote ahead of it, 14.0 so)
                if (!ok) break;
            }
        }
    } else if (warp == 1 && rank == 0) {
        // ---- MMAs ----
        int it = 0, done = 0;
        bool ok = true;
        constexpr uint32_t a_step = A_MN ? 2048 : 32, b_step = B_MN ? 2048 : 32;
        for (int unit = first; unit < units && ok; unit += step, ++done) {
            const GemmUnit u = gemm_unit(g, unit);
            const int buf = done & 1;
            ok = gemm_wait(smem_addr(&acc_empty[buf]), ((done >> 1) & 1) ^ 1, &abort_flag);
            if (!ok) break;
            tc_fence_after();
            const uint32_t d = tmem + buf * BN;
            for (int kt = u.k0; kt < u.k1; ++kt, ++it) {
                const int s = it % S::kStages;
                const bool got = lane_wait(smem_addr(&full[s]), (it / S::kStages) & 1, &abort_flag);
                tc_fence_after();
                if (elect_one() && got) {
                    const uint32_t a = smem + s * S::kStage, b = a + S::kABytes;
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        gemm_mma<EB, CG>(d, gemm_desc<A_MN>(a + k * a_step), gemm_desc<B_MN>(b + k * b_step), g.idesc, (kt > u.k0 || k > 0) ? 1u : 0u);
                    gemm_commit<CG>(smem_addr(&empty[s]), leader);
                    if (kt == u.k1 - 1) gemm_commit<CG>(smem_addr(&acc_full[buf]), leader);
                }
                ok = __all_sync(~0u, got);
                if (!ok) break;
            }
        }
    } else if (warp >= 4) {
        // ---- sums -> output ----
        const int quarter = warp & 3, out_bytes = g.out_dtype == TH_F32 ? 4 : 2;
        const uint32_t staging = smem + S::kStages * S::kStage + quarter * kStagingBoxes * kStagingBytes;
        constexpr int kStep = BN < 32 ? BN : 32;
        int done = 0, box = 0;
        for (int unit = first; unit < units; unit += step, ++done) {
            const GemmUnit u = gemm_unit(g, unit);
            const int buf = done & 1;
            const int m0 = (u.tm * CG + static_cast<int>(rank)) * kGemmRows + 32 * quarter, n0 = u.tn * BN, m = m0 + lane;
            float2 lane_scale = make_float2(1.f, 1.f);
            float lane_bias = 0.f;
            if (EB == 1 && m < g.m) lane_scale = split_scale(g.lane_scale[m]);
            if (SWAP && g.bias) lane_bias = m < g.m ? bias_at(g.bias, g.bias_dtype, m) : 0.f;
            // double buffered: a warp that fills the next tile's values has met, at the barrier before, those that read the last but one's
            for (int c = threadIdx.x - 128; c < BN; c += 128) {
                const bool inside = n0 + c < g.n;
                if (EB == 1) scales[buf][c] = split_scale(inside ? g.column_scale[n0 + c] : 0.f);
                biases[buf][c] = !SWAP && g.bias && inside ? bias_at(g.bias, g.bias_dtype, n0 + c) : 0.f;
            }
            asm volatile("bar.sync 1, 128;" ::: "memory");
            if (!gemm_wait(smem_addr(&acc_full[buf]), (done >> 1) & 1, &abort_flag)) {
                // the other warps' waits end too, but they may meet at the barriers of the units before
                for (unit += step; unit < units; unit += step) asm volatile("bar.sync 1, 128;" ::: "memory");
                break;
            }
            tc_fence_after();
            const uint32_t d = tmem + buf * BN + (static_cast<uint32_t>(32 * quarter) << 16);
#pragma unroll 1
            for (int c0 = 0; c0 < BN; c0 += kStep) {
                uint32_t raw[32];
                if constexpr (kStep == 32) tmem_ld32(d + c0, raw);
                else tmem_ld16(d + c0, raw);
                tmem_ld_wait();
                if (c0 + kStep >= BN) {
                    // the accumulator is read: the next tile but one may fill it
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        if constexpr (CG == 2)
                            asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(in_cta(smem_addr(&acc_empty[buf]), leader)) : "memory");
                        else
                            asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(&acc_empty[buf])) : "memory");
                    }
                }
                if (n0 + c0 >= g.n) continue;
                if constexpr (S::kSplits) {
                    if (g.splits > 1) {  // the operands have been read: their shared memory takes the sums
                        if constexpr (SWAP) {
#pragma unroll
                            for (int k = 0; k < kStep; ++k)
                                if (n0 + c0 + k < g.n)
                                    asm volatile("st.shared.b32 [%0], %1;" ::"r"(exchange_at<32>(smem, c0 + k, 8 * quarter + (lane >> 2)) + 4 * (lane & 3)), "r"(raw[k])
                                                 : "memory");
                        } else {
#pragma unroll
                            for (int j = 0; j < kStep / 4; ++j)
                                st_shared_16(exchange_at<BN / 4>(smem, 32 * quarter + lane, c0 / 4 + j), make_uint4(raw[4 * j], raw[4 * j + 1], raw[4 * j + 2], raw[4 * j + 3]));
                        }
                        continue;
                    }
                }
#pragma unroll
                for (int k = 0; k < kStep; ++k)
                    raw[k] = __float_as_uint(finished<EB>(raw[k], lane_scale, scales[buf][c0 + k], SWAP ? lane_bias : biases[buf][c0 + k]));
                if constexpr (SWAP) {
                    if (m < g.m) {
#pragma unroll
                        for (int k = 0; k < kStep; ++k)
                            if (n0 + c0 + k < g.n) store_one(g.out, static_cast<long long>(n0 + c0 + k) * g.out_stride + m, __uint_as_float(raw[k]), g.out_dtype);
                    }
                } else {
                    const uint32_t at = staging + (box % kStagingBoxes) * kStagingBytes + lane * 128;
                    const int half = out_bytes == 2 ? (c0 / 32) & 1 : 0;
                    if (g.out_tma && half == 0) {
                        // the box about to be written was handed to TMA kStagingBoxes stores ago
                        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(kStagingBoxes - 1) : "memory");
                        __syncwarp();
                    }
                    if (out_bytes == 4) {
#pragma unroll
                        for (int j = 0; j < kStep / 4; ++j)
                            st_shared_16(at + ((j ^ (lane & 7)) << 4), make_uint4(raw[4 * j], raw[4 * j + 1], raw[4 * j + 2], raw[4 * j + 3]));
                        store_box(g, &c_map, at - lane * 128, m0, n0 + c0, 4);
                        ++box;
                    } else {
#pragma unroll
                        for (int j = 0; j < kStep / 8; ++j) {
                            uint32_t w[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                w[e] = pack_out(__uint_as_float(raw[8 * j + 2 * e]), __uint_as_float(raw[8 * j + 2 * e + 1]), g.out_dtype);
                            st_shared_16(at + (((4 * half + j) ^ (lane & 7)) << 4), make_uint4(w[0], w[1], w[2], w[3]));
                        }
                        if (half == 1 || n0 + c0 + 32 >= g.n) {
                            store_box(g, &c_map, at - lane * 128, m0, n0 + (c0 & ~63), 2);
                            ++box;
                        }
                    }
                }
            }
        }
        if (!SWAP && g.out_tma && lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    }

    if constexpr (S::kSplits) {
        if (g.splits > 1) {
            // ---- a split tile: this CTA's part of it, from everybody's sums ----
            __syncwarp();
            cluster_sync_all();
            if (!abort_flag) {
                const GemmUnit u = gemm_unit(g, first);
                if (g.splits <= 2) finish_split<EB, BN, CG, SWAP, 8, 2>(g, u, rank, smem, scales[0], biases[0]);
                else if (g.splits <= 4) finish_split<EB, BN, CG, SWAP, 4, 4>(g, u, rank, smem, scales[0], biases[0]);
                else if constexpr (CG == 1) finish_split<EB, BN, CG, SWAP, 2, 8>(g, u, rank, smem, scales[0], biases[0]);
            }
            __syncwarp();
            cluster_sync_all();  // everybody's sums have been read
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

// Rows of `inner` elements, `stride` elements apart; boxes of box_inner x box_outer in the 128-byte swizzle.
bool matrix_map(CUtensorMap *map, const void *base, long long inner, long long outer, long long stride, int elem_bytes, int box_inner, int box_outer) {
    EncodeTiledFn encode = encode_tiled_fn();
    if (!encode || !aligned_to(base, 16) || stride * elem_bytes % 16 != 0) return false;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(outer)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(stride) * elem_bytes};
    const cuuint32_t box[2] = {static_cast<cuuint32_t>(box_inner), static_cast<cuuint32_t>(box_outer)};
    const cuuint32_t elem[2] = {1, 1};
    const CUtensorMapDataType type = elem_bytes == 1   ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                     : elem_bytes == 2 ? CU_TENSOR_MAP_DATA_TYPE_UINT16
                                                       : CU_TENSOR_MAP_DATA_TYPE_UINT32;
    return encode(map, type, 2, const_cast<void *>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Operand {
    const void *base;
    long long stride;  // elements between rows of the matrix as it lies in memory: [rows][k] K-major, [k][rows] MN-major
    int rows;          // extent along m or n
};

template <int EB, bool A_MN, bool B_MN, int BN, int CG, bool SWAP, int CTAS>
int launch_gemm(GemmArgs g, const Operand &a, const Operand &b, int k, bool bf16, cudaStream_t stream) {
    using S = GemmShape<EB, A_MN, B_MN, BN, CG, CTAS>;
    auto kernel = wide_gemm_kernel<EB, A_MN, B_MN, BN, CG, SWAP, CTAS>;
    // Once per thread and device, and ahead of the maps: it also makes the device's context current in this thread, which encoding
    // a map needs and an autograd thread may not have yet.
    static thread_local unsigned long long ready = 0;
    int device = 0;
    if (int rc = cuda_status(cudaGetDevice(&device), "cudaGetDevice")) return rc;
    if (device >= 64 || !(ready >> device & 1)) {
        if (int rc = cuda_status(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes), "cudaFuncSetAttribute(wide_gemm_kernel)"))
            return rc;
        if (device < 64) ready |= 1ull << device;
    }
    CUtensorMap a_map, b_map, c_map;
    const auto operand = [&](CUtensorMap *map, const Operand &o, bool mn, int box_rows) {
        return mn ? matrix_map(map, o.base, o.rows, k, o.stride, EB, 64, 64) : matrix_map(map, o.base, k, o.rows, o.stride, EB, S::kK, box_rows);
    };
    if (!operand(&a_map, a, A_MN, kGemmRows) || !operand(&b_map, b, B_MN, S::kBRows))
        return fail(TH_ERR_ALIGNMENT, "matrix product: operand rows must start on 16 bytes");
    g.m = a.rows;
    g.n = b.rows;
    g.tiles_m = (g.m + CG * kGemmRows - 1) / (CG * kGemmRows);
    g.tiles_n = (g.n + BN - 1) / BN;
    // 32 MB of rows: half of what one die's L2 holds.  Sustained at the power limit, TFLOP/s by rows of a group (MB), 16384 x 4096 -> 16384 float16:
    // 8 (16) 1327, 16 (32) 1345, 32 (64) 1196, a library's 1336; 8192 x 4096 -> 16384 8-bit: 8 (8) 2778, 16 (16) 2882, 32 (32) 2933.
    g.group = static_cast<int>(std::max(4ll, std::min(32ll, (32ll << 20) / (static_cast<long long>(CG) * kGemmRows * k * EB))));
    g.k_tiles = (k + S::kK - 1) / S::kK;
    g.tiles_per_split = (g.k_tiles + g.splits - 1) / g.splits;
    g.splits = (g.k_tiles + g.tiles_per_split - 1) / g.tiles_per_split;
    g.idesc = EB == 1 ? instr_desc_i8(CG * kGemmRows, BN) : instr_desc(CG * kGemmRows, BN, bf16, A_MN, B_MN);
    const int out_bytes = g.out_dtype == TH_F32 ? 4 : 2;
    if (g.splits > (S::kSplits ? 8 / CG : 1)) return fail(TH_ERR_UNSUPPORTED, "matrix product: %d parts", g.splits);
    g.out_tma = !SWAP && g.splits == 1 && matrix_map(&c_map, g.out, g.n, g.m, g.out_stride, out_bytes, 128 / out_bytes, 32);
    if (!g.out_tma) c_map = a_map;  // not looked at
    const long long units = static_cast<long long>(g.tiles_m) * g.tiles_n * g.splits;
    if (units > 0x7fffffffll) return fail(TH_ERR_UNSUPPORTED, "matrix product: too many tiles");
    // a split tile is one unit of every CTA of its cluster; otherwise CTAs go round the tiles
    const long long clusters = g.splits > 1 ? units : std::min<long long>(units, std::max(1, CTAS * sm_count() / CG));
    return launch_chained("wide_gemm_kernel launch", kernel, static_cast<unsigned>(clusters * CG), kGemmThreads, S::kBytes, stream, CG * g.splits, g, a_map, b_map, c_map);
}

}  // namespace
}  // namespace th
