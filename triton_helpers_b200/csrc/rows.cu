// Row kernels of the layers for wide networks: root-mean-square norm (forward, backward, with an 8-bit output),
// 8-bit rows and back, column sums.  All of them are bound by memory: one pass over the data, a row in the registers of
// its team of threads, statistics in float32.
//
// 8-bit rows:  a = max(max_k |x_k|, 2^-100),  q_k = rint(x_k * (127 / a)),  scale = a / 127, all in float32, so that a row is the
// same bits from any kernel (and from elementary operations elsewhere).  The floor keeps 127 / a finite: a row of zeros has zeros and
// a scale of 2^-100 / 127.  A row that holds an infinity or a NaN gets zeros and a NaN as its scale: it reads back as NaN throughout.
#include "common.cuh"

#include <algorithm>

namespace th {
namespace {

constexpr int kMaxTeam = 1024;
constexpr uint32_t kTinyBits = 0x0d800000u;  // 2^-100
constexpr uint32_t kInfBits = 0x7f800000u;

// ---- packets: VB bytes of a row, one access -----------------------------------------------------------

template <int VB>
struct Raw;
template <>
struct Raw<16> { using type = uint4; };
template <>
struct Raw<8> { using type = uint2; };
template <>
struct Raw<4> { using type = uint32_t; };
template <>
struct Raw<2> { using type = unsigned short; };
template <>
struct Raw<1> { using type = unsigned char; };

template <typename T, int VB>
struct Packet {
    static constexpr int N = VB / static_cast<int>(sizeof(T));
    union {
        typename Raw<VB>::type raw;
        T v[N];
    };
    __device__ Packet() {}
};

template <typename T, int VB>
__device__ __forceinline__ void load_values(const T *row, long long packet, float (&f)[VB / sizeof(T)]) {
    Packet<T, VB> p;
    p.raw = reinterpret_cast<const typename Raw<VB>::type *>(row)[packet];
#pragma unroll
    for (int e = 0; e < p.N; ++e) f[e] = to_float<T>(p.v[e]);
}

template <typename T, int VB>
__device__ __forceinline__ void store_values(T *row, long long packet, const float (&f)[VB / sizeof(T)]) {
    Packet<T, VB> p;
#pragma unroll
    for (int e = 0; e < p.N; ++e) p.v[e] = from_float<T>(f[e]);
    reinterpret_cast<typename Raw<VB>::type *>(row)[packet] = p.raw;
}

// The gain of a packet's columns: float32, or the rows' own type
template <typename T, int N>
__device__ __forceinline__ void load_gain(const void *gain, bool gain_f32, long long packet, float (&g)[N]) {
    if (gain_f32) {
        const float *p = static_cast<const float *>(gain) + packet * N;
        if constexpr (N % 4 == 0) {
#pragma unroll
            for (int e = 0; e < N; e += 4) {
                const float4 v = __ldg(reinterpret_cast<const float4 *>(p + e));
                g[e] = v.x; g[e + 1] = v.y; g[e + 2] = v.z; g[e + 3] = v.w;
            }
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) g[e] = __ldg(p + e);
        }
    } else {
        load_values<T, N * static_cast<int>(sizeof(T))>(static_cast<const T *>(gain), packet, g);
    }
}

// ---- sums and maxima over the threads that share a row ---------------------------------------------------

// `red`: 2 x 32 words of shared memory, `turn` flips at every call so that one barrier a call is enough.  The order of a sum is
// fixed, so results repeat.
__device__ __forceinline__ float team_sum(float v, int team, float (*red)[32], int &turn) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    if (team == 32) return v;
    float *slot = red[turn];
    turn ^= 1;
    if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = v;
    __syncthreads();
    v = (threadIdx.x & 31) < team / 32 ? slot[threadIdx.x & 31] : 0.f;
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    return v;
}

__device__ __forceinline__ uint32_t team_max(uint32_t v, int team, float (*red)[32], int &turn) {
    v = __reduce_max_sync(~0u, v);
    if (team == 32) return v;
    uint32_t *slot = reinterpret_cast<uint32_t *>(red[turn]);
    turn ^= 1;
    if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = v;
    __syncthreads();
    return __reduce_max_sync(~0u, (threadIdx.x & 31) < team / 32 ? slot[threadIdx.x & 31] : 0u);
}

// Magnitudes are compared as bit patterns: NaN is larger than infinity, which is larger than every number, so none gets lost.
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

struct RowScale {
    float inverse, scale;
    bool finite;
    __device__ explicit RowScale(uint32_t top_bits) {
        finite = top_bits < kInfBits;
        const float a = __uint_as_float(max(top_bits, kTinyBits));
        inverse = __fdiv_rn(127.f, a);
        scale = finite ? __fdiv_rn(a, 127.f) : __uint_as_float(0x7fc00000u);
    }
};

// rint of a product of at most 127: adding 1.5 * 2^23 leaves the integer in the low byte
__device__ __forceinline__ uint32_t quantum(float v, float inverse) { return __float_as_uint(__fadd_rn(__fmul_rn(v, inverse), 12582912.f)); }

template <int N>
__device__ __forceinline__ void store_quanta(signed char *row, long long packet, const float (&f)[N], const RowScale &s) {
    uint32_t b[N];
#pragma unroll
    for (int e = 0; e < N; ++e) b[e] = s.finite ? quantum(f[e], s.inverse) : 0u;
    if constexpr (N == 1) {
        row[packet] = static_cast<signed char>(b[0]);
    } else {
        uint32_t w[N / 4];
#pragma unroll
        for (int e = 0; e < N; e += 4)
            w[e / 4] = __byte_perm(__byte_perm(b[e], b[e + 1], 0x0040), __byte_perm(b[e + 2], b[e + 3], 0x0040), 0x5410);
        if constexpr (N == 8)
            reinterpret_cast<uint2 *>(row)[packet] = make_uint2(w[0], w[1]);
        else
            reinterpret_cast<uint32_t *>(row)[packet] = w[0];
    }
}

// ---- forward: norm, norm with 8-bit rows, 8-bit rows alone ------------------------------------------------

enum { kNorm = 0, kNormInt8 = 1, kQuantize = 2 };

struct RowFwdArgs {
    const void *x, *residual, *gain;
    void *sum, *y;
    signed char *q;
    float *scale, *rstd;
    long long x_stride, residual_stride, q_stride, rows;
    int d, packets, team, gain_f32;
    float eps;
};

// A team of 32 threads (several rows per CTA) or the whole CTA owns a row and keeps it in registers, P packets a thread; P = 0: rows
// longer than that are read again for every step, by then from L2.  What is normalised is the sum as it is written, rounded, so that
// the backward pass, which reads it, sees the same numbers.
template <typename T, int VB, int P, int MODE, bool RES>
__global__ void __launch_bounds__(kMaxTeam) row_fwd_kernel(const RowFwdArgs a) {
    constexpr int N = VB / static_cast<int>(sizeof(T));
    __shared__ float red[2][32];
    int turn = 0;
    const int team = a.team, t = team == 32 ? threadIdx.x & 31 : threadIdx.x;
    const long long row = team == 32 ? static_cast<long long>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
    if (row >= a.rows) return;  // whole warps, and only where a warp is a team
    const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
    const T *res = RES ? static_cast<const T *>(a.residual) + row * a.residual_stride : nullptr;
    T *sum = RES ? static_cast<T *>(a.sum) + row * a.d : nullptr;
    T *y = MODE == kNorm ? static_cast<T *>(a.y) + row * a.d : nullptr;
    signed char *q = MODE == kNorm ? nullptr : a.q + row * a.q_stride;

    const auto fetch = [&](int i, float (&f)[N]) {
        load_values<T, VB>(x, i, f);
        if constexpr (RES) {
            float r[N];
            load_values<T, VB>(res, i, r);
#pragma unroll
            for (int e = 0; e < N; ++e) f[e] = to_float<T>(from_float<T>(f[e] + r[e]));
        }
    };
    const auto normed = [&](int i, const float (&f)[N], float rstd, float (&o)[N]) {
        float g[N];
        load_gain<T, N>(a.gain, a.gain_f32 != 0, i, g);
#pragma unroll
        for (int e = 0; e < N; ++e) o[e] = f[e] * rstd * g[e];
    };

    if constexpr (P > 0) {
        float f[P][N];
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int i = t + p * team;
            if (i < a.packets) {
                fetch(i, f[p]);
            } else {
#pragma unroll
                for (int e = 0; e < N; ++e) f[p][e] = 0.f;
            }
        }
        if constexpr (RES) {
#pragma unroll
            for (int p = 0; p < P; ++p)
                if (t + p * team < a.packets) store_values<T, VB>(sum, t + p * team, f[p]);
        }
        if constexpr (MODE != kQuantize) {
            float ss = 0.f;
#pragma unroll
            for (int p = 0; p < P; ++p)
#pragma unroll
                for (int e = 0; e < N; ++e) ss = fmaf(f[p][e], f[p][e], ss);
            ss = team_sum(ss, team, red, turn);
            const float rstd = rsqrtf(ss / static_cast<float>(a.d) + a.eps);
            if (a.rstd && t == 0) a.rstd[row] = rstd;
#pragma unroll
            for (int p = 0; p < P; ++p)
                if (t + p * team < a.packets) normed(t + p * team, f[p], rstd, f[p]);
        }
        if constexpr (MODE == kNorm) {
#pragma unroll
            for (int p = 0; p < P; ++p)
                if (t + p * team < a.packets) store_values<T, VB>(y, t + p * team, f[p]);
        } else {
            uint32_t top = 0;
#pragma unroll
            for (int p = 0; p < P; ++p)
#pragma unroll
                for (int e = 0; e < N; ++e) top = max(top, magnitude(f[p][e]));
            const RowScale s(team_max(top, team, red, turn));
            if (t == 0) a.scale[row] = s.scale;
#pragma unroll
            for (int p = 0; p < P; ++p)
                if (t + p * team < a.packets) store_quanta<N>(q, t + p * team, f[p], s);
        }
    } else {
        float f[N], rstd = 1.f;
        if constexpr (MODE != kQuantize) {
            float ss = 0.f;
            for (int i = t; i < a.packets; i += team) {
                fetch(i, f);
                if constexpr (RES) store_values<T, VB>(sum, i, f);
#pragma unroll
                for (int e = 0; e < N; ++e) ss = fmaf(f[e], f[e], ss);
            }
            ss = team_sum(ss, team, red, turn);
            rstd = rsqrtf(ss / static_cast<float>(a.d) + a.eps);
            if (a.rstd && t == 0) a.rstd[row] = rstd;
        }
        const auto again = [&](int i) {
            fetch(i, f);
            if constexpr (MODE != kQuantize) normed(i, f, rstd, f);
        };
        if constexpr (MODE == kNorm) {
            for (int i = t; i < a.packets; i += team) {
                again(i);
                store_values<T, VB>(y, i, f);
            }
        } else {
            uint32_t top = 0;
            for (int i = t; i < a.packets; i += team) {
                again(i);
#pragma unroll
                for (int e = 0; e < N; ++e) top = max(top, magnitude(f[e]));
            }
            const RowScale s(team_max(top, team, red, turn));
            if (t == 0) a.scale[row] = s.scale;
            for (int i = t; i < a.packets; i += team) {
                again(i);
                store_quanta<N>(q, i, f, s);
            }
        }
    }
}

// Threads that share a row and packets each of them holds: a warp up to four packets a lane, then as many threads as give each two,
// up to the CTA's 1024.
struct TeamPlan {
    int team, per_thread, block, rows_per_block;
};
TeamPlan team_plan(int packets, int most) {
    TeamPlan p{};
    if (packets <= 128) {
        p.team = 32;
        p.per_thread = (packets + 31) / 32;
        p.rows_per_block = 4;
        p.block = 128;
    } else {
        p.team = 64;
        while (p.team < kMaxTeam && p.team * 2 < packets) p.team *= 2;
        p.per_thread = (packets + p.team - 1) / p.team;
        p.rows_per_block = 1;
        p.block = p.team;
    }
    int n = 1;
    while (n < p.per_thread) n *= 2;
    p.per_thread = n <= most ? n : 0;
    return p;
}

template <typename T, int VB, int MODE, bool RES>
int launch_row_fwd(RowFwdArgs a, cudaStream_t stream) {
    a.packets = a.d / (VB / static_cast<int>(sizeof(T)));
    const TeamPlan plan = team_plan(a.packets, 8);
    a.team = plan.team;
    const long long blocks = (a.rows + plan.rows_per_block - 1) / plan.rows_per_block;
    if (blocks > 0x7fffffffll) return fail(TH_ERR_UNSUPPORTED, "too many rows: %lld", a.rows);
    const dim3 grid(static_cast<unsigned>(blocks)), block(plan.block);
    switch (plan.per_thread) {
        case 1: row_fwd_kernel<T, VB, 1, MODE, RES><<<grid, block, 0, stream>>>(a); break;
        case 2: row_fwd_kernel<T, VB, 2, MODE, RES><<<grid, block, 0, stream>>>(a); break;
        case 4: row_fwd_kernel<T, VB, 4, MODE, RES><<<grid, block, 0, stream>>>(a); break;
        case 8: row_fwd_kernel<T, VB, 8, MODE, RES><<<grid, block, 0, stream>>>(a); break;
        default: row_fwd_kernel<T, VB, 0, MODE, RES><<<grid, block, 0, stream>>>(a); break;
    }
    return launch_status("row_fwd_kernel");
}

// 16-byte packets where every row of every tensor starts on 16 bytes and ends with a whole packet
template <typename T>
bool packed_rows(const void *p, long long stride, int d) {
    return p == nullptr || (aligned_to(p, 16) && stride * static_cast<long long>(sizeof(T)) % 16 == 0 && d * static_cast<long long>(sizeof(T)) % 16 == 0);
}

template <typename T, int MODE>
int row_fwd(const RowFwdArgs &a, cudaStream_t stream) {
    const bool packed = packed_rows<T>(a.x, a.x_stride, a.d) && packed_rows<T>(a.residual, a.residual_stride, a.d) && packed_rows<T>(a.sum, a.d, a.d) &&
                        packed_rows<T>(a.y, a.d, a.d) && (a.gain == nullptr || aligned_to(a.gain, 16));
    constexpr int E = sizeof(T);
    if constexpr (MODE != kQuantize) {
        if (a.residual) return packed ? launch_row_fwd<T, 16, MODE, true>(a, stream) : launch_row_fwd<T, E, MODE, true>(a, stream);
    }
    return packed ? launch_row_fwd<T, 16, MODE, false>(a, stream) : launch_row_fwd<T, E, MODE, false>(a, stream);
}

template <int MODE>
int row_fwd_of(int dtype, const RowFwdArgs &a, cudaStream_t stream) {
    if (dtype == TH_F32) return row_fwd<float, MODE>(a, stream);
    if (dtype == TH_F16) return row_fwd<__half, MODE>(a, stream);
    return row_fwd<__nv_bfloat16, MODE>(a, stream);
}

// ---- norm, backward -----------------------------------------------------------------------------------------
//
// With h = s * rstd, g = dy * gain and c = mean(g h):  ds = rstd (g - h c) + (gradient of s as an output),  dgain = sum over rows of dy h.
// A team keeps its columns' part of dgain in registers over all the rows it takes, then the CTA adds its teams up and writes one
// partial row; a second kernel adds the partial rows in a fixed order.

struct RowBwdArgs {
    const void *s, *gain, *gy, *gs;
    const float *rstd;
    void *dx;
    float *partial;
    long long s_stride, gy_stride, gs_stride, rows;
    int d, packets, team, gain_f32;
};

template <typename T, int VB, int P, bool GS>
__global__ void __launch_bounds__(kMaxTeam) norm_bwd_kernel(const RowBwdArgs a) {
    constexpr int N = VB / static_cast<int>(sizeof(T));
    __shared__ float red[2][32];
    int turn = 0;
    const int team = a.team, t = team == 32 ? threadIdx.x & 31 : threadIdx.x;
    const int teams = team == 32 ? blockDim.x >> 5 : 1, mine = team == 32 ? threadIdx.x >> 5 : 0;
    const float inv_d = 1.f / static_cast<float>(a.d);
    constexpr int Q = P > 0 ? P : 1;
    float acc[Q][N], gain[Q][N];
#pragma unroll
    for (int p = 0; p < Q; ++p)
#pragma unroll
        for (int e = 0; e < N; ++e) acc[p][e] = gain[p][e] = 0.f;
    if constexpr (P > 0) {
#pragma unroll
        for (int p = 0; p < P; ++p)
            if (t + p * team < a.packets) load_gain<T, N>(a.gain, a.gain_f32 != 0, t + p * team, gain[p]);
    }
    for (long long row = static_cast<long long>(blockIdx.x) * teams + mine; row < a.rows; row += static_cast<long long>(gridDim.x) * teams) {
        const T *s = static_cast<const T *>(a.s) + row * a.s_stride, *gy = static_cast<const T *>(a.gy) + row * a.gy_stride;
        const T *gs = GS ? static_cast<const T *>(a.gs) + row * a.gs_stride : nullptr;
        T *dx = static_cast<T *>(a.dx) + row * a.d;
        const float rstd = a.rstd[row];
        float c = 0.f;
        if constexpr (P > 0) {
            Packet<T, VB> sp[P], yp[P], rp[P];
#pragma unroll
            for (int p = 0; p < P; ++p) {
                const int i = t + p * team;
                if (i < a.packets) {
                    sp[p].raw = reinterpret_cast<const typename Raw<VB>::type *>(s)[i];
                    yp[p].raw = reinterpret_cast<const typename Raw<VB>::type *>(gy)[i];
                    if constexpr (GS) rp[p].raw = reinterpret_cast<const typename Raw<VB>::type *>(gs)[i];
                }
            }
#pragma unroll
            for (int p = 0; p < P; ++p)
                if (t + p * team < a.packets) {
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        const float h = to_float<T>(sp[p].v[e]) * rstd, dy = to_float<T>(yp[p].v[e]);
                        acc[p][e] = fmaf(dy, h, acc[p][e]);
                        c = fmaf(dy * gain[p][e], h, c);
                    }
                }
            c = team_sum(c, team, red, turn) * inv_d;
#pragma unroll
            for (int p = 0; p < P; ++p)
                if (t + p * team < a.packets) {
                    float o[N];
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        const float h = to_float<T>(sp[p].v[e]) * rstd;
                        o[e] = rstd * (to_float<T>(yp[p].v[e]) * gain[p][e] - h * c);
                        if constexpr (GS) o[e] += to_float<T>(rp[p].v[e]);
                    }
                    store_values<T, VB>(dx, t + p * team, o);
                }
        } else {
            float sv[N], yv[N], rv[N];
            for (int i = t; i < a.packets; i += team) {
                load_values<T, VB>(s, i, sv);
                load_values<T, VB>(gy, i, yv);
                load_gain<T, N>(a.gain, a.gain_f32 != 0, i, gain[0]);
#pragma unroll
                for (int e = 0; e < N; ++e) c = fmaf(yv[e] * gain[0][e], sv[e] * rstd, c);
            }
            c = team_sum(c, team, red, turn) * inv_d;
            for (int i = t; i < a.packets; i += team) {
                load_values<T, VB>(s, i, sv);
                load_values<T, VB>(gy, i, yv);
                load_gain<T, N>(a.gain, a.gain_f32 != 0, i, gain[0]);
                if constexpr (GS) load_values<T, VB>(gs, i, rv);
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    yv[e] = rstd * (yv[e] * gain[0][e] - sv[e] * rstd * c);
                    if constexpr (GS) yv[e] += rv[e];
                }
                store_values<T, VB>(dx, i, yv);
            }
        }
    }
    if constexpr (P > 0) {
        if (!a.partial) return;
        float *out = a.partial + static_cast<long long>(blockIdx.x) * a.d;
        if (teams == 1) {
#pragma unroll
            for (int p = 0; p < P; ++p)
                if (t + p * team < a.packets)
#pragma unroll
                    for (int e = 0; e < N; ++e) out[(t + p * team) * N + e] = acc[p][e];
        } else {
            extern __shared__ float columns[];  // d floats: the CTA's teams one after the other
            for (int k = 0; k < teams; ++k) {
                if (k == mine) {
#pragma unroll
                    for (int p = 0; p < P; ++p)
                        if (t + p * team < a.packets)
#pragma unroll
                            for (int e = 0; e < N; ++e) {
                                float *at = columns + (t + p * team) * N + e;
                                *at = k == 0 ? acc[p][e] : *at + acc[p][e];
                            }
                }
                __syncthreads();
            }
            for (int i = threadIdx.x; i < a.d; i += blockDim.x) out[i] = columns[i];
        }
    }
}

// ---- column sums: partial rows per CTA, then their sum ------------------------------------------------------

// partial[block y][column] = sum of g (times s * rstd where s is given) over the block's rows.  A lane has one column, so a warp reads
// 32 neighbours; the rows of a block go round its eight warps.
template <typename T>
__global__ void __launch_bounds__(256) column_sum_kernel(const T *g, long long g_stride, const T *s, long long s_stride, const float *rstd, float *partial,
                                                         long long rows, int d, long long rows_per_block) {
    __shared__ float part[8][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, col = blockIdx.x * 32 + lane;
    const long long first = blockIdx.y * rows_per_block, last = min(rows, first + rows_per_block);
    float v = 0.f;
    if (col < d) {
        for (long long r = first + warp; r < last; r += 8) {
            const float dy = to_float<T>(g[r * g_stride + col]);
            v += s ? dy * to_float<T>(s[r * s_stride + col]) * rstd[r] : dy;
        }
    }
    part[warp][lane] = v;
    __syncthreads();
    if (warp == 0 && col < d) {
#pragma unroll
        for (int k = 1; k < 8; ++k) v += part[k][lane];
        partial[static_cast<long long>(blockIdx.y) * d + col] = v;
    }
}

template <typename O>
__global__ void __launch_bounds__(256) partial_sum_kernel(const float *partial, int count, int d, O *out) {
    __shared__ float part[8][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, col = blockIdx.x * 32 + lane;
    float v = 0.f;
    if (col < d)
        for (int k = warp; k < count; k += 8) v += partial[static_cast<long long>(k) * d + col];
    part[warp][lane] = v;
    __syncthreads();
    if (warp == 0 && col < d) {
#pragma unroll
        for (int k = 1; k < 8; ++k) v += part[k][lane];
        out[col] = from_float<O>(v);
    }
}

int sum_partials(const float *partial, int count, int d, void *out, int out_dtype, cudaStream_t stream) {
    const dim3 grid((d + 31) / 32);
    if (out_dtype == TH_F32)
        partial_sum_kernel<float><<<grid, 256, 0, stream>>>(partial, count, d, static_cast<float *>(out));
    else if (out_dtype == TH_F16)
        partial_sum_kernel<__half><<<grid, 256, 0, stream>>>(partial, count, d, static_cast<__half *>(out));
    else
        partial_sum_kernel<__nv_bfloat16><<<grid, 256, 0, stream>>>(partial, count, d, static_cast<__nv_bfloat16 *>(out));
    return launch_status("partial_sum_kernel");
}

// Partial rows a column sum is cut into: enough blocks for the GPU, at least 32 rows each
int column_parts(long long rows, int d) {
    const long long columns = (d + 31) / 32;
    const long long wanted = std::max(1ll, (8ll * sm_count() + columns - 1) / columns);
    return static_cast<int>(std::max(1ll, std::min({wanted, (rows + 31) / 32, 1024ll})));
}

template <typename T>
int column_sums(const T *g, long long g_stride, const T *s, long long s_stride, const float *rstd, float *partial, int parts, long long rows, int d,
                cudaStream_t stream) {
    const dim3 grid((d + 31) / 32, parts);
    column_sum_kernel<T><<<grid, 256, 0, stream>>>(g, g_stride, s, s_stride, rstd, partial, rows, d, (rows + parts - 1) / parts);
    return launch_status("column_sum_kernel");
}

struct NormBwdPlan {
    TeamPlan team;
    int blocks, parts;  // partial rows: one per CTA, or (rows too long for registers) those of a column sum
};

// `packed`: 16-byte packets.  Registers hold a thread's sums and gains: 32 columns at most.
NormBwdPlan norm_bwd_plan(long long rows, int d, int dtype, bool packed) {
    NormBwdPlan p{};
    const int n = packed ? 16 / static_cast<int>(dtype_bytes(dtype)) : 1;
    p.team = team_plan(d / n, packed ? (dtype == TH_F32 ? 8 : 4) : 8);
    const int per_sm = std::max(1, 1024 / p.team.block);
    p.blocks = static_cast<int>(std::min<long long>((rows + p.team.rows_per_block - 1) / p.team.rows_per_block, static_cast<long long>(sm_count()) * per_sm));
    p.parts = p.team.per_thread ? p.blocks : column_parts(rows, d);
    return p;
}

template <typename T, int VB, bool GS>
int launch_norm_bwd(const RowBwdArgs &a, const NormBwdPlan &plan, cudaStream_t stream) {
    constexpr int N = VB / static_cast<int>(sizeof(T));
    const dim3 grid(plan.blocks), block(plan.team.block);
    const size_t smem = plan.team.team == 32 ? static_cast<size_t>(a.d) * 4 : 0;
    switch (plan.team.per_thread) {
        case 1: norm_bwd_kernel<T, VB, 1, GS><<<grid, block, smem, stream>>>(a); break;
        case 2: norm_bwd_kernel<T, VB, 2, GS><<<grid, block, smem, stream>>>(a); break;
        case 4: norm_bwd_kernel<T, VB, 4, GS><<<grid, block, smem, stream>>>(a); break;
        case 8:
            if constexpr (N < 8) norm_bwd_kernel<T, VB, 8, GS><<<grid, block, smem, stream>>>(a);
            break;
        default: norm_bwd_kernel<T, VB, 0, GS><<<grid, block, 0, stream>>>(a); break;
    }
    return launch_status("norm_bwd_kernel");
}

template <typename T>
int norm_bwd(RowBwdArgs a, void *dgain, int gain_dtype, bool packed, const NormBwdPlan &plan, cudaStream_t stream) {
    constexpr int E = sizeof(T);
    a.packets = packed ? a.d / (16 / E) : a.d;
    a.team = plan.team.team;
    float *partial = a.partial;
    if (!dgain) a.partial = nullptr;
    int rc;
    if (a.gs)
        rc = packed ? launch_norm_bwd<T, 16, true>(a, plan, stream) : launch_norm_bwd<T, E, true>(a, plan, stream);
    else
        rc = packed ? launch_norm_bwd<T, 16, false>(a, plan, stream) : launch_norm_bwd<T, E, false>(a, plan, stream);
    if (rc != TH_OK || !dgain) return rc;
    if (!plan.team.per_thread) {
        rc = column_sums<T>(static_cast<const T *>(a.gy), a.gy_stride, static_cast<const T *>(a.s), a.s_stride, a.rstd, partial, plan.parts, a.rows, a.d, stream);
        if (rc != TH_OK) return rc;
    }
    return sum_partials(partial, plan.parts, a.d, dgain, gain_dtype, stream);
}

// ---- 8-bit rows back to 16 or 32 bits --------------------------------------------------------------------------

// Sixteen columns a thread.  q * scale is rounded once, to T.
template <typename T>
__global__ void __launch_bounds__(256) dequantize_kernel(const signed char *q, long long q_stride, const float *scale, T *out, long long out_stride,
                                                         long long rows, int d, int chunks) {
    const long long id = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
    const long long row = id / chunks;
    if (row >= rows) return;
    const int c = static_cast<int>(id - row * chunks) * 16;
    const float s = scale[row];
    const signed char *src = q + row * q_stride + c;
    T *dst = out + row * out_stride + c;
    const bool whole = c + 16 <= d && ((reinterpret_cast<uintptr_t>(src) | reinterpret_cast<uintptr_t>(dst)) & 15) == 0;
    if (whole) {
        const uint4 raw = *reinterpret_cast<const uint4 *>(src);
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
        Packet<T, 16> p;
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            p.v[k % p.N] = from_float<T>(static_cast<float>(static_cast<signed char>(w[k / 4] >> (8 * (k % 4)))) * s);
            if (k % p.N == p.N - 1) reinterpret_cast<uint4 *>(dst)[k / p.N] = p.raw;
        }
    } else {
        for (int k = 0; k < 16 && c + k < d; ++k) dst[k] = from_float<T>(static_cast<float>(src[k]) * s);
    }
}

bool known_dtype(int dtype) { return dtype == TH_F32 || dtype == TH_F16 || dtype == TH_BF16; }

int check_rows(const char *what, long long rows, int d, int dtype) {
    if (rows < 0 || d < 1) return fail(TH_ERR_BAD_ARG, "%s: %lld rows of %d columns", what, rows, d);
    if (d > (1 << 24)) return fail(TH_ERR_UNSUPPORTED, "%s: %d columns, more than 2^24", what, d);
    if (!known_dtype(dtype)) return fail(TH_ERR_UNSUPPORTED, "%s: unknown dtype code %d", what, dtype);
    return TH_OK;
}

}  // namespace
}  // namespace th

using namespace th;

extern "C" int th_rms_norm_fwd(const void *x_dev, int64_t x_stride, const void *residual_dev, int64_t residual_stride, const void *gain_dev, int gain_dtype,
                               void *sum_dev, void *y_dev, float *rstd_dev, int64_t rows, int d, float eps, int dtype, void *stream) {
    if (int rc = check_rows("th_rms_norm_fwd", rows, d, dtype)) return rc;
    if (gain_dtype != dtype && gain_dtype != TH_F32) return fail(TH_ERR_UNSUPPORTED, "th_rms_norm_fwd: the gain is float32 or of the rows' type");
    if (rows == 0) return TH_OK;
    if (!x_dev || !gain_dev || !y_dev || (residual_dev != nullptr) != (sum_dev != nullptr)) return fail(TH_ERR_BAD_ARG, "th_rms_norm_fwd: null pointer");
    RowFwdArgs a{};
    a.x = x_dev; a.residual = residual_dev; a.gain = gain_dev; a.sum = sum_dev; a.y = y_dev; a.rstd = rstd_dev;
    a.x_stride = x_stride; a.residual_stride = residual_stride; a.rows = rows; a.d = d; a.gain_f32 = gain_dtype == TH_F32; a.eps = eps;
    return row_fwd_of<kNorm>(dtype, a, static_cast<cudaStream_t>(stream));
}

extern "C" int th_rms_norm_int8(const void *x_dev, int64_t x_stride, const void *residual_dev, int64_t residual_stride, const void *gain_dev, int gain_dtype,
                                void *sum_dev, void *q_dev, int64_t q_stride, float *scale_dev, int64_t rows, int d, float eps, int dtype, void *stream) {
    if (int rc = check_rows("th_rms_norm_int8", rows, d, dtype)) return rc;
    if (gain_dtype != dtype && gain_dtype != TH_F32) return fail(TH_ERR_UNSUPPORTED, "th_rms_norm_int8: the gain is float32 or of the rows' type");
    if (rows == 0) return TH_OK;
    if (!x_dev || !gain_dev || !q_dev || !scale_dev || (residual_dev != nullptr) != (sum_dev != nullptr))
        return fail(TH_ERR_BAD_ARG, "th_rms_norm_int8: null pointer");
    if (!aligned_to(q_dev, 16) || q_stride % 16 || q_stride < d) return fail(TH_ERR_ALIGNMENT, "th_rms_norm_int8: 8-bit rows start on 16 bytes");
    RowFwdArgs a{};
    a.x = x_dev; a.residual = residual_dev; a.gain = gain_dev; a.sum = sum_dev; a.q = static_cast<signed char *>(q_dev); a.scale = scale_dev;
    a.x_stride = x_stride; a.residual_stride = residual_stride; a.q_stride = q_stride; a.rows = rows; a.d = d; a.gain_f32 = gain_dtype == TH_F32; a.eps = eps;
    return row_fwd_of<kNormInt8>(dtype, a, static_cast<cudaStream_t>(stream));
}

extern "C" int th_quantize_rows(const void *x_dev, int64_t x_stride, void *q_dev, int64_t q_stride, float *scale_dev, int64_t rows, int d, int dtype,
                                void *stream) {
    if (int rc = check_rows("th_quantize_rows", rows, d, dtype)) return rc;
    if (rows == 0) return TH_OK;
    if (!x_dev || !q_dev || !scale_dev) return fail(TH_ERR_BAD_ARG, "th_quantize_rows: null pointer");
    if (!aligned_to(q_dev, 16) || q_stride % 16 || q_stride < d) return fail(TH_ERR_ALIGNMENT, "th_quantize_rows: 8-bit rows start on 16 bytes");
    RowFwdArgs a{};
    a.x = x_dev; a.q = static_cast<signed char *>(q_dev); a.scale = scale_dev;
    a.x_stride = x_stride; a.q_stride = q_stride; a.rows = rows; a.d = d;
    return row_fwd_of<kQuantize>(dtype, a, static_cast<cudaStream_t>(stream));
}

extern "C" int th_dequantize_rows(const void *q_dev, int64_t q_stride, const float *scale_dev, void *out_dev, int64_t out_stride, int64_t rows, int d,
                                  int dtype, void *stream) {
    if (int rc = check_rows("th_dequantize_rows", rows, d, dtype)) return rc;
    if (rows == 0) return TH_OK;
    if (!q_dev || !scale_dev || !out_dev || q_stride < d || out_stride < d) return fail(TH_ERR_BAD_ARG, "th_dequantize_rows: null pointer or short stride");
    const int chunks = (d + 15) / 16;
    if (rows > (0x7fffffffll * 256) / chunks) return fail(TH_ERR_UNSUPPORTED, "th_dequantize_rows: too many rows: %lld", static_cast<long long>(rows));
    const dim3 grid(static_cast<unsigned>((rows * chunks + 255) / 256));
    cudaStream_t at = static_cast<cudaStream_t>(stream);
    const signed char *q = static_cast<const signed char *>(q_dev);
    if (dtype == TH_F32)
        dequantize_kernel<float><<<grid, 256, 0, at>>>(q, q_stride, scale_dev, static_cast<float *>(out_dev), out_stride, rows, d, chunks);
    else if (dtype == TH_F16)
        dequantize_kernel<__half><<<grid, 256, 0, at>>>(q, q_stride, scale_dev, static_cast<__half *>(out_dev), out_stride, rows, d, chunks);
    else
        dequantize_kernel<__nv_bfloat16><<<grid, 256, 0, at>>>(q, q_stride, scale_dev, static_cast<__nv_bfloat16 *>(out_dev), out_stride, rows, d, chunks);
    return launch_status("dequantize_kernel");
}

// The scratch is the larger of what rows in 16-byte packets and rows read value by value take.
extern "C" int64_t th_rms_norm_bwd_workspace_bytes(int64_t rows, int d, int dtype) {
    if (rows < 1 || d < 1 || !known_dtype(dtype)) return 0;
    const int whole = 16 / static_cast<int>(dtype_bytes(dtype));
    int parts = norm_bwd_plan(rows, d, dtype, false).parts;
    if (d % whole == 0) parts = std::max(parts, norm_bwd_plan(rows, d, dtype, true).parts);
    return static_cast<int64_t>(parts) * d * 4;
}

extern "C" int th_rms_norm_bwd(const void *sum_dev, int64_t sum_stride, const void *gain_dev, int gain_dtype, const float *rstd_dev, const void *grad_y_dev,
                               int64_t gy_stride, const void *grad_sum_dev, int64_t gs_stride, void *grad_x_dev, void *grad_gain_dev, void *workspace_dev,
                               int64_t workspace_bytes, int64_t rows, int d, int dtype, void *stream) {
    if (int rc = check_rows("th_rms_norm_bwd", rows, d, dtype)) return rc;
    if (gain_dtype != dtype && gain_dtype != TH_F32) return fail(TH_ERR_UNSUPPORTED, "th_rms_norm_bwd: the gain is float32 or of the rows' type");
    cudaStream_t at = static_cast<cudaStream_t>(stream);
    if (rows == 0) {
        if (grad_gain_dev) return cuda_status(cudaMemsetAsync(grad_gain_dev, 0, static_cast<size_t>(d) * dtype_bytes(gain_dtype), at), "th_rms_norm_bwd");
        return TH_OK;
    }
    if (!sum_dev || !gain_dev || !rstd_dev || !grad_y_dev || !grad_x_dev) return fail(TH_ERR_BAD_ARG, "th_rms_norm_bwd: null pointer");
    if (grad_gain_dev && (!workspace_dev || workspace_bytes < th_rms_norm_bwd_workspace_bytes(rows, d, dtype) || !aligned_to(workspace_dev, 16)))
        return fail(TH_ERR_WORKSPACE, "th_rms_norm_bwd: scratch missing, too small or off 16 bytes");
    RowBwdArgs a{};
    a.s = sum_dev; a.gain = gain_dev; a.gy = grad_y_dev; a.gs = grad_sum_dev; a.rstd = rstd_dev; a.dx = grad_x_dev;
    a.partial = static_cast<float *>(workspace_dev);
    a.s_stride = sum_stride; a.gy_stride = gy_stride; a.gs_stride = gs_stride; a.rows = rows; a.d = d; a.gain_f32 = gain_dtype == TH_F32;
    const auto run = [&](auto tag) {
        using T = decltype(tag);
        const bool packed = packed_rows<T>(a.s, a.s_stride, d) && packed_rows<T>(a.gy, a.gy_stride, d) && packed_rows<T>(a.gs, a.gs_stride, d) &&
                            packed_rows<T>(a.dx, d, d) && aligned_to(a.gain, 16);
        return norm_bwd<T>(a, grad_gain_dev, gain_dtype, packed, norm_bwd_plan(rows, d, dtype, packed), at);
    };
    if (dtype == TH_F32) return run(float{});
    if (dtype == TH_F16) return run(__half{});
    return run(__nv_bfloat16{});
}

extern "C" int64_t th_column_sum_workspace_bytes(int64_t rows, int d) {
    return rows < 1 || d < 1 ? 0 : static_cast<int64_t>(column_parts(rows, d)) * d * 4;
}

extern "C" int th_column_sum(const void *g_dev, int64_t g_stride, void *out_dev, void *workspace_dev, int64_t workspace_bytes, int64_t rows, int d, int dtype,
                             void *stream) {
    if (int rc = check_rows("th_column_sum", rows, d, dtype)) return rc;
    if (!out_dev) return fail(TH_ERR_BAD_ARG, "th_column_sum: null pointer");
    cudaStream_t at = static_cast<cudaStream_t>(stream);
    if (rows == 0) return cuda_status(cudaMemsetAsync(out_dev, 0, static_cast<size_t>(d) * dtype_bytes(dtype), at), "th_column_sum");
    if (!g_dev) return fail(TH_ERR_BAD_ARG, "th_column_sum: null pointer");
    if (!workspace_dev || workspace_bytes < th_column_sum_workspace_bytes(rows, d) || !aligned_to(workspace_dev, 4))
        return fail(TH_ERR_WORKSPACE, "th_column_sum: scratch missing or too small");
    float *partial = static_cast<float *>(workspace_dev);
    const int parts = column_parts(rows, d);
    int rc;
    if (dtype == TH_F32)
        rc = column_sums<float>(static_cast<const float *>(g_dev), g_stride, nullptr, 0, nullptr, partial, parts, rows, d, at);
    else if (dtype == TH_F16)
        rc = column_sums<__half>(static_cast<const __half *>(g_dev), g_stride, nullptr, 0, nullptr, partial, parts, rows, d, at);
    else
        rc = column_sums<__nv_bfloat16>(static_cast<const __nv_bfloat16 *>(g_dev), g_stride, nullptr, 0, nullptr, partial, parts, rows, d, at);
    return rc != TH_OK ? rc : sum_partials(partial, parts, d, out_dev, dtype, at);
}
