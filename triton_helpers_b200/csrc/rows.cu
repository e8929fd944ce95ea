// Row kernels of the layers for wide networks: root-mean-square norm (forward, backward, with an 8-bit output),
// 8-bit rows and back, column sums.  All of them are bound by memory: one pass over the data, a row in the registers of
// its team of threads, statistics in float32.
//
// 8-bit rows:  a = max(max_k |x_k|, 2^-100),  q_k = rint(x_k * (127 / a)),  scale = a / 127, all in float32, so that a row is the
// same bits from any kernel (and from elementary operations elsewhere).  The floor keeps 127 / a finite: a row of zeros has zeros and
// a scale of 2^-100 / 127.  A row that holds an infinity or a NaN gets zeros and a NaN as its scale: it reads back as NaN throughout.
#include "chained.cuh"
#include "drain.cuh"

#include <algorithm>
#include <utility>

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
struct Raw<4> { using type = uint32_t; };
template <>
struct Raw<2> { using type = unsigned short; };

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

// A row as 16-byte packets that start on 16 bytes, wherever the row itself starts: `shift` elements of the first packet lie ahead of it and
// the last one may reach past it.  A packet holds one element of the row at least, so it lies in memory that is there; elements beside the
// row are read as zeros and never written.  (5000 rows of 3001 bfloat16, us: norm 27 an element at a time, 18.6 so; to 8 bits 26 and 12.4.)
template <typename T, bool SHIFT>
struct Span {
    static constexpr int N = 16 / static_cast<int>(sizeof(T));
    int shift, d, packets;
    __device__ Span(const void *row, int columns) {
        d = columns;
        shift = SHIFT ? static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T)) : 0;
        packets = SHIFT ? (shift + d + N - 1) / N : d / N;
    }
    __device__ __forceinline__ bool edge(int i) const { return SHIFT && (i == 0 || i == packets - 1); }
    __device__ __forceinline__ bool inside(int i, int e) const { return static_cast<unsigned>(i * N + e - shift) < static_cast<unsigned>(d); }
    __device__ __forceinline__ uint4 fetch(const T *row, int i) const { return reinterpret_cast<const uint4 *>(row - shift)[i]; }
    __device__ __forceinline__ void widen(uint4 raw, int i, float (&f)[N]) const {
        Packet<T, 16> p;
        p.raw = raw;
#pragma unroll
        for (int e = 0; e < N; ++e) f[e] = to_float<T>(p.v[e]);
        if (edge(i)) {
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (!inside(i, e)) f[e] = 0.f;
        }
    }
    __device__ __forceinline__ void store(T *row, int i, const float (&f)[N]) const {
        if (edge(i)) {
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (inside(i, e)) row[i * N + e - shift] = from_float<T>(f[e]);
        } else {
            store_values<T, 16>(row - shift, i, f);
        }
    }
    // The gain of a packet's columns: float32, or the rows' own type; it starts on 16 bytes itself
    __device__ __forceinline__ void gains(const void *gain, bool gain_f32, int i, float (&g)[N]) const {
        if constexpr (SHIFT) {
            const int c = i * N - shift;
            if (edge(i)) {
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    const int at = min(max(c + e, 0), d - 1);
                    g[e] = gain_f32 ? static_cast<const float *>(gain)[at] : to_float<T>(static_cast<const T *>(gain)[at]);
                }
            } else if (gain_f32) {
#pragma unroll
                for (int e = 0; e < N; ++e) g[e] = __ldg(static_cast<const float *>(gain) + c + e);
            } else {
#pragma unroll
                for (int e = 0; e < N; ++e) g[e] = to_float<T>(static_cast<const T *>(gain)[c + e]);
            }
        } else if (gain_f32) {
#pragma unroll
            for (int e = 0; e < N; e += 4) {
                const float4 v = __ldg(reinterpret_cast<const float4 *>(static_cast<const float *>(gain) + i * N + e));
                g[e] = v.x; g[e + 1] = v.y; g[e + 2] = v.z; g[e + 3] = v.w;
            }
        } else {
            load_values<T, 16>(static_cast<const T *>(gain), i, g);
        }
    }
};

// ---- sums and maxima over the threads that share a row ---------------------------------------------------

// `red`: 2 x 32 words of shared memory, `turn` flips at every call so that one barrier a call is enough.  The order of a sum is
// fixed, so results repeat.  A team of up to 32 threads is an aligned part of a warp, a larger one the CTA.
__device__ __forceinline__ float team_sum(float v, int team, float (*red)[32], int &turn) {
    if (team <= 32) {
        for (int o = team >> 1; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
        return v;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
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
    if (team < 32) {
        for (int o = team >> 1; o; o >>= 1) v = max(v, __shfl_xor_sync(~0u, v, o));
        return v;
    }
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

// N (4 or 8) of them, the first in the lowest byte
template <int N>
__device__ __forceinline__ unsigned long long quanta(const float (&f)[N], const RowScale &s) {
    uint32_t w[2] = {0, 0};
    if (s.finite) {
#pragma unroll
        for (int e = 0; e < N; e += 4)
            w[e / 4] = __byte_perm(__byte_perm(quantum(f[e], s.inverse), quantum(f[e + 1], s.inverse), 0x0040),
                                   __byte_perm(quantum(f[e + 2], s.inverse), quantum(f[e + 3], s.inverse), 0x0040), 0x5410);
    }
    return w[0] | static_cast<unsigned long long>(w[1]) << 32;
}

template <int N>
__device__ __forceinline__ void store_quanta(signed char *row, int i, unsigned long long b) {
    if constexpr (N == 8) reinterpret_cast<unsigned long long *>(row)[i] = b;
    else reinterpret_cast<uint32_t *>(row)[i] = static_cast<uint32_t>(b);
}

// Packets that lie `shift` columns before their place in the 8-bit row: a lane joins its last columns with its neighbour's first ones, so
// a warp has one packet more than it stores.  Called by whole warps.
template <int N>
__device__ __forceinline__ void store_shifted_quanta(signed char *row, int i, int shift, int d, bool mine, unsigned long long b) {
    const unsigned long long next = __shfl_down_sync(~0u, b, 1);
    if (mine && i * N < d) store_quanta<N>(row, i, shift ? (b >> (8 * shift)) | (next << (8 * (N - shift))) : b);
}

// ---- forward: norm, norm with 8-bit rows, 8-bit rows alone ------------------------------------------------

enum { kNorm = 0, kNormInt8 = 1, kQuantize = 2 };

struct RowFwdArgs {
    const void *x, *residual, *gain;
    void *sum, *y;
    signed char *q;
    float *scale, *rstd;
    long long x_stride, residual_stride, q_stride, rows;
    int d, team, gain_f32;
    float eps;
};

// A team of 4 to 32 threads (several rows per CTA) or the whole CTA owns a row and keeps it in registers, P packets a thread.  What is
// normalised is the sum as it is written, rounded, so that the backward pass, which reads it, sees the same numbers.
template <typename T, int P, int MODE, bool RES, bool SHIFT, int THREADS>
__global__ void __launch_bounds__(THREADS) row_fwd_kernel(const RowFwdArgs a) {
    constexpr int N = 16 / static_cast<int>(sizeof(T));
    __shared__ float red[2][32];
    int turn = 0;
    after_previous();
    const int team = a.team;
    const bool part = team <= 32;  // of a warp
    const int t = part ? threadIdx.x & (team - 1) : threadIdx.x;
    const long long place = part ? static_cast<long long>(blockIdx.x) * (blockDim.x / team) + threadIdx.x / team : blockIdx.x;
    const bool live = place < a.rows;  // teams behind the last row have nothing to load or store, but take part in their warp's sums
    const long long row = live ? place : 0;
    const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
    Span<T, SHIFT> span(x, a.d);
    if (!live) span.packets = 0;

    // shifted 8-bit rows: a warp's (or smaller team's) last lane has the packet that the next one's first lane owns
    constexpr bool kOverlap = SHIFT && MODE != kNorm;
    const int lanes = part ? team : 32, own = kOverlap ? lanes - 1 : lanes;
    const int at = kOverlap && !part ? (t >> 5) * 31 + (t & 31) : t, step = part ? own : team / 32 * own;
    const bool mine = !kOverlap || (t & (lanes - 1)) < own;

    uint4 raw[P], added[P];  // every load is on its way before the first is used
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const int i = at + p * step;
        raw[p] = added[p] = make_uint4(0, 0, 0, 0);
        if (i < span.packets) {
            raw[p] = span.fetch(x, i);
            if constexpr (RES) added[p] = span.fetch(static_cast<const T *>(a.residual) + row * a.residual_stride, i);
        }
    }
    float f[P][N];
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const int i = at + p * step;
        span.widen(raw[p], i, f[p]);
        if constexpr (RES) {
            float r[N];
            span.widen(added[p], i, r);
#pragma unroll
            for (int e = 0; e < N; ++e) f[p][e] = to_float<T>(from_float<T>(f[p][e] + r[e]));
        }
    }
    if constexpr (MODE != kQuantize) {
        float squares = 0.f;
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
            for (int e = 0; e < N; ++e) squares = fmaf(f[p][e], f[p][e], squares);
        const float ss = team_sum(mine ? squares : 0.f, team, red, turn);
        const float rstd = rsqrtf(ss / static_cast<float>(a.d) + a.eps);
        if (a.rstd && t == 0 && live) a.rstd[row] = rstd;
        if constexpr (RES) {
#pragma unroll
            for (int p = 0; p < P; ++p)
                if (mine && at + p * step < span.packets) span.store(static_cast<T *>(a.sum) + row * a.d, at + p * step, f[p]);
        }
#pragma unroll
        for (int p = 0; p < P; ++p) {
            if (at + p * step < span.packets) {
                float g[N];
                span.gains(a.gain, a.gain_f32 != 0, at + p * step, g);
#pragma unroll
                for (int e = 0; e < N; ++e) f[p][e] = f[p][e] * rstd * g[e];
            }
        }
        if constexpr (MODE == kNorm) {
#pragma unroll
            for (int p = 0; p < P; ++p)
                if (at + p * step < span.packets) span.store(static_cast<T *>(a.y) + row * a.d, at + p * step, f[p]);
        }
    }
    if constexpr (MODE != kNorm) {
        uint32_t top = 0;
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
            for (int e = 0; e < N; ++e) top = max(top, magnitude(f[p][e]));
        const RowScale s(team_max(top, team, red, turn));
        if (t == 0 && live) a.scale[row] = s.scale;
        signed char *q = a.q + row * a.q_stride;
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int i = at + p * step;
            const unsigned long long b = quanta<N>(f[p], s);
            if constexpr (SHIFT) store_shifted_quanta<N>(q, i, span.shift, a.d, mine && live, b);
            else if (i < span.packets) store_quanta<N>(q, i, b);
        }
    }
}

// Rows that are too long for registers, or whose tensors do not start alike: read again for every step, by then from L2.  VB = 16 bytes an
// access where everything starts on them, else an element.  A view whose rows start elsewhere than the result's (column 3 of 16384 x 4104 on, 4096
// wide, bfloat16) takes 121 us, packed rows 44.
template <typename T, int VB, int MODE, bool RES>
__global__ void __launch_bounds__(kMaxTeam) row_fwd_stream_kernel(const RowFwdArgs a) {
    constexpr int N = VB / static_cast<int>(sizeof(T));
    __shared__ float red[2][32];
    int turn = 0;
    after_previous();
    const int team = blockDim.x, packets = a.d / N;
    const long long row = blockIdx.x;
    const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
    const T *res = RES ? static_cast<const T *>(a.residual) + row * a.residual_stride : nullptr;
    T *sum = RES ? static_cast<T *>(a.sum) + row * a.d : nullptr;
    float f[N], rstd = 1.f;
    const auto fetch = [&](int i) {
        load_values<T, VB>(x, i, f);
        if constexpr (RES) {
            float r[N];
            load_values<T, VB>(res, i, r);
#pragma unroll
            for (int e = 0; e < N; ++e) f[e] = to_float<T>(from_float<T>(f[e] + r[e]));
        }
    };
    if constexpr (MODE != kQuantize) {
        float ss = 0.f;
        for (int i = threadIdx.x; i < packets; i += team) {
            fetch(i);
            if constexpr (RES) store_values<T, VB>(sum, i, f);
#pragma unroll
            for (int e = 0; e < N; ++e) ss = fmaf(f[e], f[e], ss);
        }
        ss = team_sum(ss, team, red, turn);
        rstd = rsqrtf(ss / static_cast<float>(a.d) + a.eps);
        if (a.rstd && threadIdx.x == 0) a.rstd[row] = rstd;
    }
    const auto value = [&](int i) {
        fetch(i);
        if constexpr (MODE != kQuantize) {
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const long long c = static_cast<long long>(i) * N + e;
                f[e] = f[e] * rstd * (a.gain_f32 ? __ldg(static_cast<const float *>(a.gain) + c) : to_float<T>(static_cast<const T *>(a.gain)[c]));
            }
        }
    };
    if constexpr (MODE == kNorm) {
        T *y = static_cast<T *>(a.y) + row * a.d;
        for (int i = threadIdx.x; i < packets; i += team) {
            value(i);
            store_values<T, VB>(y, i, f);
        }
    } else {
        uint32_t top = 0;
        for (int i = threadIdx.x; i < packets; i += team) {
            value(i);
#pragma unroll
            for (int e = 0; e < N; ++e) top = max(top, magnitude(f[e]));
        }
        const RowScale s(team_max(top, team, red, turn));
        if (threadIdx.x == 0) a.scale[row] = s.scale;
        signed char *q = a.q + row * a.q_stride;
        for (int i = threadIdx.x; i < packets; i += team) {
            value(i);
            if constexpr (N == 1) q[i] = s.finite ? static_cast<signed char>(quantum(f[0], s.inverse)) : 0;
            else store_quanta<N>(q, i, quanta<N>(f, s));
        }
    }
}

// Threads that share a row and packets each of them holds: 4, 8 or 16 lanes for up to two packets each, a warp for up to four, then as many
// threads as give each `wanted`, up to the CTA's 1024 (and eight packets; 0: more than that).  `overlap`: a warp or smaller team shares
// its last packet with the next.  (60000 x 131 bfloat16 to 8 bits: 14.2 us with a warp a row, 13.3 so; norm of 20000 x 512 14.9 and 14.1.)
struct TeamPlan {
    int team, per_thread, block, rows_per_block;
};
TeamPlan team_plan(int packets, int wanted, bool overlap) {
    TeamPlan p{};
    int step = 0;
    for (int lanes = 4; lanes <= 32 && !p.team; lanes *= 2) {
        step = lanes - overlap;
        if (packets <= step * (lanes == 32 ? 4 : 2)) {
            p.team = lanes;
            p.rows_per_block = 128 / lanes;
            p.block = 128;
        }
    }
    if (!p.team) {
        const int own = 32 - overlap;
        p.team = std::min(kMaxTeam, std::max(64, ((packets + wanted - 1) / wanted + own - 1) / own * 32));
        p.rows_per_block = 1;
        p.block = p.team;
        step = p.team / 32 * own;
    }
    p.per_thread = (packets + step - 1) / step;
    int n = 1;
    while (n < p.per_thread) n *= 2;
    p.per_thread = n <= 8 ? n : 0;
    return p;
}

// How the rows of several tensors lie
enum { kPacked, kShifted, kAnyhow };
struct Layout {
    bool packed = true, alike = true;
    uintptr_t start = ~uintptr_t(0), step = 0;
    template <typename T>
    void add(const void *p, long long stride, int d) {
        if (!p) return;
        const uintptr_t at = reinterpret_cast<uintptr_t>(p) & 15, by = static_cast<uintptr_t>(stride * static_cast<long long>(sizeof(T))) & 15;
        packed = packed && at == 0 && by == 0 && d * static_cast<long long>(sizeof(T)) % 16 == 0;
        if (start == ~uintptr_t(0)) {
            start = at;
            step = by;
        }
        alike = alike && at == start && by == step && at % sizeof(T) == 0;
    }
    int kind() const { return packed ? kPacked : alike ? kShifted : kAnyhow; }
};
// Packets of the longest span of d columns
template <typename T>
int span_packets(int d, int kind) {
    constexpr int N = 16 / static_cast<int>(sizeof(T));
    return kind == kPacked ? d / N : (d + 2 * N - 2) / N;
}

// The kernels that team_plan asks for, over all widths: up to 256 threads have one to four packets each, up to 512 four (two where nine to sixteen
// warps overlap and two are wanted), 1024 four or eight.
template <typename T, int MODE, bool RES, bool SHIFT>
int launch_row_fwd(const RowFwdArgs &a, const TeamPlan &plan, unsigned blocks, cudaStream_t stream) {
    const auto run = [&](auto kernel) { return launch_chained("row_fwd_kernel", kernel, blocks, plan.block, 0, stream, 1, a); };
    const int threads = plan.block <= 256 ? 256 : plan.block <= 512 ? 512 : kMaxTeam;
    switch (threads + plan.per_thread) {
        case 256 + 1: return run(row_fwd_kernel<T, 1, MODE, RES, SHIFT, 256>);
        case 256 + 2: return run(row_fwd_kernel<T, 2, MODE, RES, SHIFT, 256>);
        case 256 + 4: return run(row_fwd_kernel<T, 4, MODE, RES, SHIFT, 256>);
        case 512 + 2:
            if constexpr (RES && SHIFT && MODE == kNormInt8) return run(row_fwd_kernel<T, 2, MODE, RES, SHIFT, 512>);
            break;
        case 512 + 4: return run(row_fwd_kernel<T, 4, MODE, RES, SHIFT, 512>);
        case kMaxTeam + 4: return run(row_fwd_kernel<T, 4, MODE, RES, SHIFT, kMaxTeam>);
        case kMaxTeam + 8: return run(row_fwd_kernel<T, 8, MODE, RES, SHIFT, kMaxTeam>);
        default: break;
    }
    return fail(TH_ERR_UNSUPPORTED, "row_fwd_kernel: %d packets for each of %d threads", plan.per_thread, plan.block);
}

template <typename T, int MODE, bool RES>
int plan_row_fwd(RowFwdArgs a, cudaStream_t stream) {
    Layout rows;
    rows.add<T>(a.x, a.x_stride, a.d);
    rows.add<T>(a.residual, a.residual_stride, a.d);
    rows.add<T>(a.sum, a.d, a.d);
    rows.add<T>(a.y, a.d, a.d);
    const bool gain = a.gain == nullptr || aligned_to(a.gain, 16);
    const int kind = gain || rows.kind() == kShifted ? rows.kind() : kAnyhow;
    const int packets = span_packets<T>(a.d, kind);
    // Packets a thread, of 16 bytes each from every input: as many as keep some 64 bytes on their way.  2^26 bfloat16 values, us: without a residual
    // 4096 columns 43.8 with four, 48.7 with two, 63 with one; with one 4096 columns 80.6 with four, 79.8 with two, 86 with one, and off 16 bytes 1537
    // columns 122 and 112, 2500 columns 110 and 100.  Past 512 packets two would ask for CTAs of up to 1024 threads: 5120 to 8192 columns 80.5 with
    // four, 79.7 with two, 12288 columns 82 and 117 (float32 the other way round there, 110 and 91; 4097 bfloat16 columns 122 and 106).
    const TeamPlan plan = team_plan(packets, RES && packets <= 512 ? 2 : 4, kind == kShifted && MODE != kNorm);
    const long long blocks = (a.rows + plan.rows_per_block - 1) / plan.rows_per_block;
    if (a.rows > 0x7fffffffll) return fail(TH_ERR_UNSUPPORTED, "too many rows: %lld", a.rows);
    const unsigned n = static_cast<unsigned>(blocks), all = static_cast<unsigned>(a.rows);
    a.team = plan.team;
    if (kind != kAnyhow && plan.per_thread)
        return kind == kPacked ? launch_row_fwd<T, MODE, RES, false>(a, plan, n, stream) : launch_row_fwd<T, MODE, RES, true>(a, plan, n, stream);
    const int block = std::min(kMaxTeam, std::max(64, (a.d / 8 + 31) / 32 * 32));
    return launch_chained("row_fwd_stream_kernel", kind == kPacked ? row_fwd_stream_kernel<T, 16, MODE, RES> : row_fwd_stream_kernel<T, sizeof(T), MODE, RES>, all,
                          block, 0, stream, 1, a);
}

template <typename T, int MODE>
int row_fwd(const RowFwdArgs &a, cudaStream_t stream) {
    if constexpr (MODE != kQuantize)
        if (a.residual) return plan_row_fwd<T, MODE, true>(a, stream);
    return plan_row_fwd<T, MODE, false>(a, stream);
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
    int d, team, gain_f32;
};

// Rows come through a ring of stages in shared memory, brought by bulk copies of one warp, so that what is in flight does not depend on
// the registers that sums take (16384 x 4096 bfloat16 with a residual: rows held in registers 111 us at best, by launch shape up to 260; a
// ring 93, copied bytes' time 82; float32 16000 x 2048 80 of 80).  16-bit rows are bound by their instructions as well.  Long
// rows are shared by all consumer warps, short ones have a warp each.  A team's rows are a multiple of eight apart, so that each of
// them starts alike and a thread's packets are the same columns in all.
constexpr int kMaxRing = 8;
constexpr unsigned long long kRingWaitNs = 1000000000ull;
__device__ int g_rows_status = 0;  // 1 = a bounded wait ran out

struct RingPlan {
    int stages, rows;          // stages, rows of a stage
    int slot;                  // bytes of one row's place, where rows lie apart
    int tensor_bytes;          // of one tensor's part of a stage
    int whole[3];              // s, gy, gs: a stage's rows are one piece of memory
    long long blocks;          // stages in all
};

// After a wait that ran out (false) nothing more is fetched, and the consumers go on with what is there, so that nobody is left at a barrier;
// the status says so.
__device__ __forceinline__ bool ring_wait(uint32_t bar, uint32_t parity, int *abort_flag) {
    unsigned long long deadline = 0;
    for (unsigned poll = 0;; ++poll) {
        uint32_t done;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
                     : "=r"(done) : "r"(bar), "r"(parity) : "memory");
        if (done) return true;
        if ((poll & 63u) == 63u) {
            if (*reinterpret_cast<volatile int *>(abort_flag)) return false;
            unsigned long long now;
            asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
            if (deadline == 0) deadline = now + kRingWaitNs;
            else if (now > deadline) break;
        }
    }
    *reinterpret_cast<volatile int *>(abort_flag) = 1;
    g_rows_status = 1;
    return false;
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

// The sum over a team: a warp, or all consumers (who meet at barrier 1)
template <int CONSUMERS>
__device__ __forceinline__ float ring_sum(float v, bool wide, float (*red)[32], int &turn) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    if (!wide) return v;
    float *slot = red[turn];
    turn ^= 1;
    if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = v;
    asm volatile("bar.sync 1, %0;" ::"n"(CONSUMERS) : "memory");
    v = (threadIdx.x & 31) < CONSUMERS / 32 ? slot[threadIdx.x & 31] : 0.f;
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    return v;
}

template <typename T, int P, bool GS, bool SHIFT, int CONSUMERS>
__global__ void __launch_bounds__(CONSUMERS + 32, CONSUMERS == 256 ? 2 : 1) norm_bwd_kernel(const RowBwdArgs a, const RingPlan ring) {
    constexpr int N = 16 / static_cast<int>(sizeof(T)), kTensors = GS ? 3 : 2, kWarps = CONSUMERS / 32;
    extern __shared__ __align__(16) unsigned char stages[];
    __shared__ __align__(8) unsigned long long full[kMaxRing], empty[kMaxRing];
    __shared__ float red[2][32];
    __shared__ int abort_flag;
    const auto shared = [](const void *p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); };
    const int stage_bytes = kTensors * ring.tensor_bytes;
    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int i = 0; i < ring.stages; ++i) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(shared(&full[i])), "r"(1u) : "memory");
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(shared(&empty[i])), "r"(static_cast<uint32_t>(kWarps)) : "memory");
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    after_previous();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const char *base[3] = {static_cast<const char *>(a.s), static_cast<const char *>(a.gy), static_cast<const char *>(a.gs)};
    const long long pitch[3] = {a.s_stride * static_cast<long long>(sizeof(T)), a.gy_stride * static_cast<long long>(sizeof(T)),
                                a.gs_stride * static_cast<long long>(sizeof(T))};
    const long long row_bytes = a.d * static_cast<long long>(sizeof(T));
    float acc[P][N];
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
        for (int e = 0; e < N; ++e) acc[p][e] = 0.f;
    const bool wide = a.team > 32;
    const int t = wide ? threadIdx.x : lane;
    int turn = 0, stage = 0;
    uint32_t phase = 0;

    if (warp == kWarps) {
        // ---- rows -> shared memory: whole 16-byte granules that hold a byte of the rows ----
        for (long long block = blockIdx.x; block < ring.blocks; block += gridDim.x) {
            if (!__all_sync(~0u, ring_wait(shared(&empty[stage]), phase ^ 1, &abort_flag))) break;
            const long long row0 = block * ring.rows;
            const int rows = static_cast<int>(min(static_cast<long long>(ring.rows), a.rows - row0));
            const uint32_t bar = shared(&full[stage]);
            uint32_t mine = 0;
            // a piece a lane: one per tensor, or one per row
            const auto pieces = [&](bool send) {
#pragma unroll
                for (int k = 0; k < kTensors; ++k) {
                    const uint32_t to = shared(stages) + stage * stage_bytes + k * ring.tensor_bytes;
                    for (int r = lane; r < (ring.whole[k] ? 1 : rows); r += 32) {
                        const uintptr_t at = reinterpret_cast<uintptr_t>(base[k] + (row0 + r) * pitch[k]);
                        const uintptr_t end = at + (ring.whole[k] ? rows : 1) * row_bytes, from = at & ~uintptr_t(15);
                        const uint32_t bytes = static_cast<uint32_t>((end - from + 15) & ~uintptr_t(15));
                        if (send) bulk_load(to + r * ring.slot, reinterpret_cast<const void *>(from), bytes, bar);
                        else mine += bytes;
                    }
                }
            };
            pieces(false);
            const uint32_t total = __reduce_add_sync(~0u, mine);
            if (lane == 0) asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(total) : "memory");
            __syncwarp();
            pieces(true);
            if (++stage == ring.stages) {
                stage = 0;
                phase ^= 1;
            }
        }
    } else {
        const float inv_d = 1.f / static_cast<float>(a.d);
        const int first = wide ? 0 : warp, apart = wide ? 1 : kWarps;  // a team's rows of a stage
        const long long start = static_cast<long long>(blockIdx.x) * ring.rows;
        // the same for all of the team's rows: where they start in their first packet, and where a stage's first row does
        const Span<T, SHIFT> span(base[0] + (start + first) * pitch[0], a.d);
        const int ahead = SHIFT ? static_cast<int>(reinterpret_cast<uintptr_t>(base[0] + start * pitch[0]) & 15) : 0, bytes = static_cast<int>(row_bytes);
        const long long stride = static_cast<long long>(gridDim.x) * ring.rows;
        // few columns a thread: their gains, and dy * rstd * gain between the two steps, stay in registers
        constexpr bool kHold = P * N <= 16;
        float gain[kHold ? P : 1][N];
        if constexpr (kHold) {
#pragma unroll
            for (int p = 0; p < P; ++p) {
#pragma unroll
                for (int e = 0; e < N; ++e) gain[p][e] = 0.f;
                if (t + p * a.team < span.packets) span.gains(a.gain, a.gain_f32 != 0, t + p * a.team, gain[p]);
            }
        }
        float next_rstd = start + first < a.rows ? a.rstd[start + first] : 0.f;
        for (long long row0 = start; row0 < a.rows; row0 += stride) {
            ring_wait(shared(&full[stage]), phase, &abort_flag);
            const unsigned char *in = stages + stage * stage_bytes;
            const int rows = static_cast<int>(min(static_cast<long long>(ring.rows), a.rows - row0));
            for (int r = first; r < rows; r += apart) {
                const long long row = row0 + r;
                const float rstd = next_rstd;
                const long long following = r + apart < ring.rows ? row + apart : row0 + stride + first;
                if (following < a.rows) next_rstd = a.rstd[following];
                const uint4 *held[3];
#pragma unroll
                for (int k = 0; k < kTensors; ++k)
                    held[k] = reinterpret_cast<const uint4 *>(in + k * ring.tensor_bytes + (ring.whole[k] ? (ahead + r * bytes) & ~15 : r * ring.slot));
                float part = 0.f, w[kHold ? P : 1][N];
#pragma unroll
                for (int p = 0; p < P; ++p) {
                    const int i = t + p * a.team;
                    if (i < span.packets) {
                        float sv[N], (&g)[N] = gain[kHold ? p : 0], (&v)[N] = w[kHold ? p : 0];
                        span.widen(held[0][i], i, sv);
                        span.widen(held[1][i], i, v);
                        if constexpr (!kHold) span.gains(a.gain, a.gain_f32 != 0, i, g);
#pragma unroll
                        for (int e = 0; e < N; ++e) {
                            v[e] *= rstd;
                            acc[p][e] = fmaf(v[e], sv[e], acc[p][e]);
                            v[e] *= g[e];
                            part = fmaf(v[e], sv[e], part);
                        }
                    }
                }
                // part: the sum of dy gain h;  ds = rstd (dy gain - h c) + gs = w - s rstd^2 c + gs
                const float c = ring_sum<CONSUMERS>(part, wide, red, turn) * inv_d, k2 = -rstd * rstd * c;
                T *dx = static_cast<T *>(a.dx) + row * a.d;
#pragma unroll
                for (int p = 0; p < P; ++p) {
                    const int i = t + p * a.team;
                    if (i < span.packets) {
                        float sv[N], o[N], (&v)[N] = w[kHold ? p : 0];
                        if constexpr (!kHold) {
                            span.widen(held[1][i], i, v);
                            span.gains(a.gain, a.gain_f32 != 0, i, sv);
#pragma unroll
                            for (int e = 0; e < N; ++e) v[e] = v[e] * rstd * sv[e];
                        }
                        span.widen(held[0][i], i, sv);
#pragma unroll
                        for (int e = 0; e < N; ++e) o[e] = fmaf(sv[e], k2, v[e]);
                        if constexpr (GS) {
                            span.widen(held[2][i], i, sv);
#pragma unroll
                            for (int e = 0; e < N; ++e) o[e] += sv[e];
                        }
                        span.store(dx, i, o);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(shared(&empty[stage])) : "memory");
            if (++stage == ring.stages) {
                stage = 0;
                phase ^= 1;
            }
        }
    }
    __syncthreads();  // every stage has been read: their memory takes the sums
    if (abort_flag) {  // the same for all threads: nothing may land in this memory once another CTA has it
        if (threadIdx.x == 0) drain_copies(full, ring.stages);
        __syncthreads();
        return;
    }
    if (!a.partial) return;
    float *out = a.partial + static_cast<long long>(blockIdx.x) * a.d;
    const Span<T, SHIFT> span(base[0] + (static_cast<long long>(blockIdx.x) * ring.rows + (wide ? 0 : warp)) * pitch[0], a.d);
    if (wide) {
        if (warp == kWarps) return;
#pragma unroll
        for (int p = 0; p < P; ++p)
            if (t + p * a.team < span.packets)
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (!SHIFT || span.inside(t + p * a.team, e)) out[(t + p * a.team) * N + e - span.shift] = acc[p][e];
    } else {
        float *columns = reinterpret_cast<float *>(stages);  // d floats: the CTA's warps one after the other
        for (int k = 0; k < kWarps; ++k) {
            if (k == warp) {
#pragma unroll
                for (int p = 0; p < P; ++p)
                    if (t + p * 32 < span.packets)
#pragma unroll
                        for (int e = 0; e < N; ++e)
                            if (!SHIFT || span.inside(t + p * 32, e)) {
                                float *at = columns + (t + p * 32) * N + e - span.shift;
                                *at = k == 0 ? acc[p][e] : *at + acc[p][e];
                            }
            }
            __syncthreads();
        }
        for (int i = threadIdx.x; i < a.d; i += blockDim.x) out[i] = columns[i];
    }
}

// Rows that are too long for registers, or whose tensors do not start alike; the gain's gradient is a column sum of its own then.  (16384 rows of
// 4096 bfloat16 that start at another column than the result's: 318 us, packed 84.)
template <typename T, int VB, bool GS>
__global__ void __launch_bounds__(kMaxTeam) norm_bwd_stream_kernel(const RowBwdArgs a) {
    constexpr int N = VB / static_cast<int>(sizeof(T));
    __shared__ float red[2][32];
    int turn = 0;
    after_previous();
    const int team = blockDim.x, packets = a.d / N;
    const long long row = blockIdx.x;
    const T *s = static_cast<const T *>(a.s) + row * a.s_stride, *gy = static_cast<const T *>(a.gy) + row * a.gy_stride;
    const T *gs = GS ? static_cast<const T *>(a.gs) + row * a.gs_stride : nullptr;
    T *dx = static_cast<T *>(a.dx) + row * a.d;
    const float rstd = a.rstd[row];
    float sv[N], w[N], rv[N], c = 0.f;
    const auto fetch = [&](int i) {
        load_values<T, VB>(s, i, sv);
        load_values<T, VB>(gy, i, w);
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const long long col = static_cast<long long>(i) * N + e;
            w[e] = w[e] * rstd * (a.gain_f32 ? __ldg(static_cast<const float *>(a.gain) + col) : to_float<T>(static_cast<const T *>(a.gain)[col]));
        }
    };
    for (int i = threadIdx.x; i < packets; i += team) {
        fetch(i);
#pragma unroll
        for (int e = 0; e < N; ++e) c = fmaf(w[e], sv[e], c);
    }
    const float k = -rstd * rstd * (team_sum(c, team, red, turn) / static_cast<float>(a.d));
    for (int i = threadIdx.x; i < packets; i += team) {
        fetch(i);
        if constexpr (GS) load_values<T, VB>(gs, i, rv);
#pragma unroll
        for (int e = 0; e < N; ++e) {
            w[e] = fmaf(sv[e], k, w[e]);
            if constexpr (GS) w[e] += rv[e];
        }
        store_values<T, VB>(dx, i, w);
    }
}

// ---- column sums: partial rows per CTA, then their sum ------------------------------------------------------

struct ColumnArgs {
    const void *g, *s;       // sums of g, or of g * s * rstd
    const float *rstd;
    void *out;               // [parts][d]: float32 partial rows, or the result itself where there is one part and `whole` is set
    long long g_stride, s_stride, rows, per_part;
    int d, whole;
};

// One block's columns over one part of the rows.  PER columns a lane: 16 bytes where the rows start on them (the last ones may reach past
// the row, to values that no result is made of), else one; the rows go round the block's 32 warps, eight at a time on their way.
template <typename T, int PER>
__device__ __forceinline__ void column_sums_of(const ColumnArgs &a, int block, int part_index, float *part) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, col = (block * 32 + lane) * PER;
    const long long first = part_index * a.per_part, last = min(a.rows, first + a.per_part);
    const T *g = static_cast<const T *>(a.g), *s = static_cast<const T *>(a.s);
    float v[PER] = {};
    if (col < a.d) {
#pragma unroll 8
        for (long long r = first + warp; r < last; r += 32) {
            float x[PER];
            load_values<T, PER * static_cast<int>(sizeof(T))>(g + r * a.g_stride + col, 0, x);
            if (s) {
                float y[PER];
                load_values<T, PER * static_cast<int>(sizeof(T))>(s + r * a.s_stride + col, 0, y);
                const float k = a.rstd[r];
#pragma unroll
                for (int e = 0; e < PER; ++e) x[e] *= y[e] * k;
            }
#pragma unroll
            for (int e = 0; e < PER; ++e) v[e] += x[e];
        }
    }
    // the warps' sums: PER of them a thread, then the 32 / PER groups of every column
    constexpr int kColumns = 32 * PER;
#pragma unroll
    for (int e = 0; e < PER; ++e) part[warp * kColumns + lane * PER + e] = v[e];
    __syncthreads();
    const int c = threadIdx.x % kColumns, group = threadIdx.x / kColumns;
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < PER; ++k) sum += part[(group * PER + k) * kColumns + c];
    __syncthreads();
    part[threadIdx.x] = sum;
    __syncthreads();
    if (threadIdx.x < kColumns && block * kColumns + c < a.d) {
#pragma unroll
        for (int k = 1; k < 32 / PER; ++k) sum += part[k * kColumns + c];
        if (a.whole) static_cast<T *>(a.out)[block * kColumns + c] = from_float<T>(sum);
        else static_cast<float *>(a.out)[static_cast<long long>(part_index) * a.d + block * kColumns + c] = sum;
    }
}

template <typename T, int PER>
__global__ void __launch_bounds__(1024) column_sum_kernel(const ColumnArgs a) {
    __shared__ float part[1024 * PER];
    after_previous();
    column_sums_of<T, PER>(a, blockIdx.x, blockIdx.y, part);
}

template <typename O>
__global__ void __launch_bounds__(1024) partial_sum_kernel(const float *partial, int count, int d, O *out) {
    __shared__ float part[32][33];
    after_previous();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, col = blockIdx.x * 32 + lane;
    float v = 0.f;
    if (col < d) {
#pragma unroll 4
        for (int k = warp; k < count; k += 32) v += partial[static_cast<long long>(k) * d + col];
    }
    part[warp][lane] = v;
    __syncthreads();
    v = part[lane][warp];  // a warp a column
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    if (lane == 0 && blockIdx.x * 32 + warp < d) out[blockIdx.x * 32 + warp] = from_float<O>(v);
}

int sum_partials(const float *partial, int count, int d, void *out, int out_dtype, cudaStream_t stream) {
    const unsigned grid = (d + 31) / 32;
    if (out_dtype == TH_F32) return launch_chained("partial_sum_kernel", partial_sum_kernel<float>, grid, 1024, 0, stream, 1, partial, count, d, static_cast<float *>(out));
    if (out_dtype == TH_F16) return launch_chained("partial_sum_kernel", partial_sum_kernel<__half>, grid, 1024, 0, stream, 1, partial, count, d, static_cast<__half *>(out));
    return launch_chained("partial_sum_kernel", partial_sum_kernel<__nv_bfloat16>, grid, 1024, 0, stream, 1, partial, count, d, static_cast<__nv_bfloat16 *>(out));
}

// Partial rows a column sum is cut into: two blocks an SM, at least 128 rows each; up to 512 rows are summed at once.
int column_parts(long long rows, int d) {
    if (rows <= 512) return 1;
    const long long columns = (d + 255) / 256;
    return static_cast<int>(std::max(1ll, std::min({2ll * sm_count() / std::min<long long>(columns, 2ll * sm_count()), rows / 128, 256ll})));
}

template <typename T>
int column_width(const ColumnArgs &a) {
    constexpr int kWide = 16 / static_cast<int>(sizeof(T));
    const auto whole = [&](const void *p, long long stride) { return aligned_to(p, 16) && stride % kWide == 0; };
    return whole(a.g, a.g_stride) && (!a.s || whole(a.s, a.s_stride)) ? kWide : 1;
}

// Column sums into `out` of the given type, by way of `partial` where there is more than one part
template <typename T>
int column_sums(ColumnArgs a, float *partial, void *out, int out_dtype, cudaStream_t stream) {
    const int parts = column_parts(a.rows, a.d), width = column_width<T>(a);
    a.per_part = (a.rows + parts - 1) / parts;
    a.whole = parts == 1 && (out_dtype == TH_F32) == (sizeof(T) == 4);
    a.out = a.whole ? out : partial;
    const dim3 grid((a.d + 32 * width - 1) / (32 * width), parts);
    const int rc = launch_chained("column_sum_kernel", width > 1 ? column_sum_kernel<T, 16 / sizeof(T)> : column_sum_kernel<T, 1>, grid, 1024, 0, stream, 1, a);
    return rc != TH_OK || a.whole ? rc : sum_partials(partial, parts, a.d, out, out_dtype, stream);
}

struct NormBwdPlan {
    int per_thread, team, consumers;  // packets of a thread (0: the stream kernel), threads of a row, consumer threads
    int parts;                        // partial rows: one per CTA, or those of a column sum
    RingPlan ring;
};

// Dynamic shared memory of a CTA's ring, at most
constexpr int ring_budget(int consumers) { return (consumers == 256 ? 110 : 222) * 1024; }

// A thread sums 32 columns at most.  Up to four packets a lane a row is a warp's; longer ones are shared by 256 threads, with two CTAs an SM, as
// long as a thread has no more than the two packets whose gains and products it can hold, then by 512 with one (2^26 bfloat16 values with the
// sum's gradient, us: 4096 columns 95 with 256 threads, 136 with 512; 4097 columns 389 and 268, 6144 156 and 128, 8192 132 and 114).
template <typename T>
NormBwdPlan norm_bwd_plan(long long rows, int d, int kind, bool gs) {
    constexpr int kMost = sizeof(T) == 4 ? 8 : 4;
    NormBwdPlan p{};
    const int packets = span_packets<T>(d, kind);
    p.parts = column_parts(rows, d);
    if (kind == kAnyhow || packets > 512 * kMost) return p;
    const bool wide = packets > 128;
    p.consumers = packets > 512 ? 512 : 256;
    p.team = wide ? p.consumers : 32;
    RingPlan &r = p.ring;
    r.slot = (packets + 1) * 16;
    const int tensors = gs ? 3 : 2, budget = ring_budget(p.consumers);
    // short rows: eight at a time, and more as long as a stage stays small
    r.rows = wide ? 1 : 8;
    while (!wide && r.rows < 64 && 2 * r.rows * r.slot * tensors <= 16 * 1024) r.rows *= 2;
    r.tensor_bytes = r.rows * r.slot + 16;
    r.stages = std::min(kMaxRing, budget / (tensors * r.tensor_bytes));
    if (r.stages < 2) return p;
    int n = 1;
    while (n * p.team < packets) n *= 2;
    p.per_thread = n;
    r.blocks = (rows + r.rows - 1) / r.rows;
    // one round of CTAs; where a row is a CTA's, a multiple of eight of them
    const long long room = static_cast<long long>(sm_count()) * (p.consumers == 256 ? 2 : 1);
    p.parts = static_cast<int>(wide ? std::min((r.blocks + 7) / 8 * 8, std::max(8ll, room / 8 * 8)) : std::min(r.blocks, room));
    return p;
}

// The function's limit of shared memory is the most that any ring takes, set once per thread and device: it belongs to the device, where another
// thread's launch of the same kernel may have another ring.
template <typename T, int P, bool GS, bool SHIFT, int CONSUMERS>
int launch_norm_bwd_of(const RowBwdArgs &a, const NormBwdPlan &plan, cudaStream_t stream) {
    auto kernel = norm_bwd_kernel<T, P, GS, SHIFT, CONSUMERS>;
    static thread_local unsigned long long ready = 0;
    int device = 0;
    if (int rc = cuda_status(cudaGetDevice(&device), "cudaGetDevice")) return rc;
    if (device >= 64 || !(ready >> device & 1)) {
        if (int rc = cuda_status(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, ring_budget(CONSUMERS)),
                                 "cudaFuncSetAttribute(norm_bwd_kernel)"))
            return rc;
        if (device < 64) ready |= 1ull << device;
    }
    const size_t smem = static_cast<size_t>(plan.ring.stages) * (GS ? 3 : 2) * plan.ring.tensor_bytes;
    return launch_chained("norm_bwd_kernel", kernel, plan.parts, CONSUMERS + 32, smem, stream, 1, a, plan.ring);
}

// A row of one warp or of 256 threads has one to four packets a thread, one of 512 two to four, or eight of float32.
template <typename T, bool GS, bool SHIFT>
int launch_norm_bwd(const RowBwdArgs &a, const NormBwdPlan &plan, cudaStream_t stream) {
    switch (plan.consumers + plan.per_thread) {
        case 256 + 1: return launch_norm_bwd_of<T, 1, GS, SHIFT, 256>(a, plan, stream);
        case 256 + 2: return launch_norm_bwd_of<T, 2, GS, SHIFT, 256>(a, plan, stream);
        case 256 + 4: return launch_norm_bwd_of<T, 4, GS, SHIFT, 256>(a, plan, stream);
        case 512 + 2: return launch_norm_bwd_of<T, 2, GS, SHIFT, 512>(a, plan, stream);
        case 512 + 4: return launch_norm_bwd_of<T, 4, GS, SHIFT, 512>(a, plan, stream);
        case 512 + 8:
            if constexpr (sizeof(T) == 4) return launch_norm_bwd_of<T, 8, GS, SHIFT, 512>(a, plan, stream);
            break;
        default: break;
    }
    return fail(TH_ERR_UNSUPPORTED, "norm_bwd_kernel: %d packets for each of %d threads", plan.per_thread, plan.consumers);
}

template <typename T>
int norm_bwd(RowBwdArgs a, void *dgain, int gain_dtype, cudaStream_t stream) {
    Layout rows;
    rows.add<T>(a.s, a.s_stride, a.d);
    rows.add<T>(a.gy, a.gy_stride, a.d);
    rows.add<T>(a.gs, a.gs_stride, a.d);
    rows.add<T>(a.dx, a.d, a.d);
    const int kind = aligned_to(a.gain, 16) || rows.kind() == kShifted ? rows.kind() : kAnyhow;
    NormBwdPlan plan = norm_bwd_plan<T>(a.rows, a.d, kind, a.gs != nullptr);
    plan.ring.whole[0] = a.s_stride == a.d;
    plan.ring.whole[1] = a.gy_stride == a.d;
    plan.ring.whole[2] = a.gs_stride == a.d;
    float *partial = a.partial;
    a.team = plan.team;
    if (!dgain) a.partial = nullptr;
    int rc;
    if (plan.per_thread) {
        if (kind == kPacked) rc = a.gs ? launch_norm_bwd<T, true, false>(a, plan, stream) : launch_norm_bwd<T, false, false>(a, plan, stream);
        else rc = a.gs ? launch_norm_bwd<T, true, true>(a, plan, stream) : launch_norm_bwd<T, false, true>(a, plan, stream);
        return rc != TH_OK || !dgain ? rc : sum_partials(partial, plan.parts, a.d, dgain, gain_dtype, stream);
    }
    if (a.rows > 0x7fffffffll) return fail(TH_ERR_UNSUPPORTED, "too many rows: %lld", a.rows);
    const unsigned grid = static_cast<unsigned>(a.rows);
    const int block = std::min(kMaxTeam, std::max(64, (a.d / 8 + 31) / 32 * 32));
    if (kind == kPacked) rc = launch_chained("norm_bwd_stream_kernel", a.gs ? norm_bwd_stream_kernel<T, 16, true> : norm_bwd_stream_kernel<T, 16, false>, grid, block, 0, stream, 1, a);
    else rc = launch_chained("norm_bwd_stream_kernel", a.gs ? norm_bwd_stream_kernel<T, sizeof(T), true> : norm_bwd_stream_kernel<T, sizeof(T), false>, grid, block, 0, stream, 1, a);
    if (rc != TH_OK || !dgain) return rc;
    ColumnArgs sums{};
    sums.g = a.gy; sums.s = a.s; sums.rstd = a.rstd;
    sums.g_stride = a.gy_stride; sums.s_stride = a.s_stride; sums.rows = a.rows; sums.d = a.d;
    return column_sums<T>(sums, partial, dgain, gain_dtype, stream);
}

// ---- 8-bit rows back to 16 or 32 bits --------------------------------------------------------------------------

struct DequantizeArgs {
    const signed char *q;
    const float *scale;
    void *out;
    long long q_stride, out_stride, rows;
    int d, chunks;
};

// Sixteen columns a thread.  q * scale is rounded once, to T: in 16 bits it is an operand of the weight's gradient.  Relative to that gradient's
// norm the rounding is 1.6e-3 in bfloat16 and 2.0e-4 in float16, where the 8 bits themselves are 7e-3 to 2e-2.  Keeping what is rounded off would
// take a second product of the weight's gradient's size, over the remainders: 193 us more of 690 at 8192 x 4096 -> 4096.
template <typename T>
__device__ __forceinline__ void dequantize(const DequantizeArgs &a, long long id) {
    const long long row = id / a.chunks;
    if (row >= a.rows) return;
    const int c = static_cast<int>(id - row * a.chunks) * 16;
    const float s = a.scale[row];
    const signed char *src = a.q + row * a.q_stride + c;
    T *dst = static_cast<T *>(a.out) + row * a.out_stride + c;
    const bool whole = c + 16 <= a.d && ((reinterpret_cast<uintptr_t>(src) | reinterpret_cast<uintptr_t>(dst)) & 15) == 0;
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
        for (int k = 0; k < 16 && c + k < a.d; ++k) dst[k] = from_float<T>(static_cast<float>(src[k]) * s);
    }
}

// Results that do not start on 16 bytes: a packet of them a thread, from the two or three words that hold its bytes (5000 x 3001 bfloat16:
// 75 us a value at a time, 12.4 so; for results that do, 16000 x 2048 float32 36.7 with sixteen values a thread, 40.9 so).
template <typename T>
__device__ __forceinline__ void dequantize_shifted(const DequantizeArgs &a, long long id) {
    constexpr int N = Span<T, true>::N;
    const long long row = id / a.chunks;
    if (row >= a.rows) return;
    T *dst = static_cast<T *>(a.out) + row * a.out_stride;
    const Span<T, true> span(dst, a.d);
    const int i = static_cast<int>(id - row * a.chunks), c = i * N - span.shift;
    if (i >= span.packets) return;
    const float s = a.scale[row];
    const signed char *src = a.q + row * a.q_stride;
    float f[N];
    if (span.edge(i)) {
#pragma unroll
        for (int e = 0; e < N; ++e) f[e] = span.inside(i, e) ? static_cast<float>(src[c + e]) * s : 0.f;
    } else {
        const uintptr_t at = reinterpret_cast<uintptr_t>(src + c);
        const uint32_t *words = reinterpret_cast<const uint32_t *>(at & ~uintptr_t(3)), by = 8 * static_cast<uint32_t>(at & 3);
        uint32_t w[N / 4 + 1];
#pragma unroll
        for (int k = 0; k <= N / 4; ++k) w[k] = k < N / 4 || by ? words[k] : 0u;
#pragma unroll
        for (int e = 0; e < N; ++e) f[e] = static_cast<float>(static_cast<signed char>(__funnelshift_r(w[e / 4], w[e / 4 + 1], by) >> (8 * (e % 4)))) * s;
    }
    span.store(dst, i, f);
}

template <typename T, bool SHIFT>
__global__ void __launch_bounds__(256) dequantize_kernel(const DequantizeArgs a) {
    after_previous();
    const long long id = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
    if constexpr (SHIFT) dequantize_shifted<T>(a, id);
    else dequantize<T>(a, id);
}

template <typename T>
int dequantize_rows(DequantizeArgs a, cudaStream_t stream) {
    constexpr int E = sizeof(T), N = 16 / E;
    const bool shifted = !aligned_to(a.out, 16) || a.out_stride * E % 16 != 0;
    a.chunks = shifted ? (a.d + 2 * N - 2) / N : (a.d + 15) / 16;
    if (a.rows > (0x7fffffffll * 256) / a.chunks) return fail(TH_ERR_UNSUPPORTED, "th_dequantize_rows: too many rows: %lld", a.rows);
    const unsigned grid = static_cast<unsigned>((a.rows * a.chunks + 255) / 256);
    return launch_chained("dequantize_kernel", shifted ? dequantize_kernel<T, true> : dequantize_kernel<T, false>, grid, 256, 0, stream, 1, a);
}

// What the weight's gradient reads and the bias's gradient, in one launch: the first blocks sum columns (they take longer), the others turn
// 8-bit rows into T.
template <typename T, int PER>
__global__ void __launch_bounds__(1024) checkpoint_rows_kernel(const DequantizeArgs rows, const ColumnArgs sums, int column_blocks, int sum_blocks) {
    __shared__ float part[1024 * PER];
    after_previous();
    if (blockIdx.x < sum_blocks) column_sums_of<T, PER>(sums, blockIdx.x % column_blocks, blockIdx.x / column_blocks, part);
    else dequantize<T>(rows, static_cast<long long>(blockIdx.x - sum_blocks) * 1024 + threadIdx.x);
}

template <typename T>
int checkpoint_rows(const DequantizeArgs &rows, ColumnArgs sums, float *partial, void *out, int dtype, cudaStream_t stream) {
    const int parts = column_parts(sums.rows, sums.d), width = column_width<T>(sums), columns = (sums.d + 32 * width - 1) / (32 * width);
    sums.per_part = (sums.rows + parts - 1) / parts;
    sums.whole = parts == 1;
    sums.out = sums.whole ? out : partial;
    const long long blocks = static_cast<long long>(columns) * parts + (rows.rows * rows.chunks + 1023) / 1024;
    if (blocks > 0x7fffffffll) return fail(TH_ERR_UNSUPPORTED, "th_checkpoint_rows: too many rows: %lld", rows.rows);
    const int rc = launch_chained("checkpoint_rows_kernel", width > 1 ? checkpoint_rows_kernel<T, 16 / sizeof(T)> : checkpoint_rows_kernel<T, 1>,
                                  static_cast<unsigned>(blocks), 1024, 0, stream, 1, rows, sums, columns, columns * parts);
    return rc != TH_OK || sums.whole ? rc : sum_partials(partial, parts, sums.d, out, dtype, stream);
}

// ---- 16-bit rows to places that start on 16 bytes -----------------------------------------------------------------

constexpr int kMostCopies = 2;
struct CopyArgs {
    const void *src[kMostCopies];
    void *dst[kMostCopies];
    long long src_stride[kMostCopies], dst_stride[kMostCopies], rows[kMostCopies], first_block[kMostCopies + 1];
    int d[kMostCopies];
};

// Sixteen bytes of a destination a thread, from the four or five words that hold them; a word is read only where it holds a byte of the
// row.  Zeros follow a row up to a whole chunk.
__global__ void __launch_bounds__(256) copy_rows_kernel(const CopyArgs a) {
    after_previous();
    const int k = blockIdx.x >= a.first_block[1] ? 1 : 0;
    const int chunks = (a.d[k] + 7) / 8;
    const long long id = (blockIdx.x - a.first_block[k]) * 256 + threadIdx.x, row = id / chunks;
    if (row >= a.rows[k]) return;
    const int c = static_cast<int>(id - row * chunks) * 8;
    const uintptr_t start = reinterpret_cast<uintptr_t>(a.src[k]) + 2 * (row * a.src_stride[k] + c), end = start + 2 * min(8, a.d[k] - c);
    const uintptr_t from = start & ~uintptr_t(3);
    uint32_t w[5];
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = from + 4 * i < end ? reinterpret_cast<const uint32_t *>(from)[i] : 0u;
    if (start & 2) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 16);
    }
    const int left = a.d[k] - c;  // values past the row's end become zeros
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = left >= 2 * i + 2 ? w[i] : left == 2 * i + 1 ? w[i] & 0xffffu : 0u;
    *reinterpret_cast<uint4 *>(static_cast<unsigned short *>(a.dst[k]) + row * a.dst_stride[k] + c) = make_uint4(w[0], w[1], w[2], w[3]);
}

bool known_dtype(int dtype) { return dtype == TH_F32 || dtype == TH_F16 || dtype == TH_BF16; }

int check_rows(const char *what, long long rows, int d, int dtype) {
    if (rows < 0 || d < 1) return fail(TH_ERR_BAD_ARG, "%s: %lld rows of %d columns", what, rows, d);
    if (d > (1 << 24)) return fail(TH_ERR_UNSUPPORTED, "%s: %d columns, more than 2^24", what, d);
    if (!known_dtype(dtype)) return fail(TH_ERR_UNSUPPORTED, "%s: unknown dtype code %d", what, dtype);
    return TH_OK;
}

}  // namespace

int rows_status_word() {
    int status = 0;
    return cudaMemcpyFromSymbol(&status, g_rows_status, sizeof(int)) == cudaSuccess ? status : -1;
}

}  // namespace th

using namespace th;

extern "C" int th_rms_norm_fwd(const void *x_dev, int64_t x_stride, const void *residual_dev, int64_t residual_stride, const void *gain_dev, int gain_dtype,
                               void *sum_dev, void *y_dev, float *rstd_dev, int64_t rows, int d, float eps, int dtype, void *stream) {
    if (int rc = check_rows("th_rms_norm_fwd", rows, d, dtype)) return rc;
    if (gain_dtype != dtype && gain_dtype != TH_F32) return fail(TH_ERR_UNSUPPORTED, "th_rms_norm_fwd: the gain is float32 or of the rows' type");
    if (rows == 0) return TH_OK;
    if (!x_dev || !gain_dev || !y_dev || (residual_dev != nullptr) != (sum_dev != nullptr)) return fail(TH_ERR_BAD_ARG, "th_rms_norm_fwd: null pointer");
    if (int rc = check_elements("th_rms_norm_fwd", dtype, {x_dev, residual_dev, sum_dev, y_dev})) return rc;
    if (int rc = check_elements("th_rms_norm_fwd", gain_dtype, {gain_dev})) return rc;
    if (int rc = check_elements("th_rms_norm_fwd", TH_F32, {rstd_dev})) return rc;
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
    if (int rc = check_elements("th_rms_norm_int8", dtype, {x_dev, residual_dev, sum_dev})) return rc;
    if (int rc = check_elements("th_rms_norm_int8", gain_dtype, {gain_dev})) return rc;
    if (int rc = check_elements("th_rms_norm_int8", TH_F32, {scale_dev})) return rc;
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
    if (int rc = check_elements("th_quantize_rows", dtype, {x_dev})) return rc;
    if (int rc = check_elements("th_quantize_rows", TH_F32, {scale_dev})) return rc;
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
    if (int rc = check_elements("th_dequantize_rows", dtype, {out_dev})) return rc;
    if (int rc = check_elements("th_dequantize_rows", TH_F32, {scale_dev})) return rc;
    const DequantizeArgs a{static_cast<const signed char *>(q_dev), scale_dev, out_dev, q_stride, out_stride, rows, d, 0};
    cudaStream_t at = static_cast<cudaStream_t>(stream);
    if (dtype == TH_F32) return dequantize_rows<float>(a, at);
    if (dtype == TH_F16) return dequantize_rows<__half>(a, at);
    return dequantize_rows<__nv_bfloat16>(a, at);
}

extern "C" int th_copy_rows(int n, const void *const *src_dev, const int64_t *src_stride, void *const *dst_dev, const int64_t *dst_stride, const int64_t *rows,
                            const int *d, void *stream) {
    if (n < 1 || n > kMostCopies || !src_dev || !src_stride || !dst_dev || !dst_stride || !rows || !d) return fail(TH_ERR_BAD_ARG, "th_copy_rows: %d matrices", n);
    CopyArgs a{};
    long long blocks = 0;
    for (int k = 0; k < kMostCopies; ++k) {
        a.first_block[k] = blocks;
        if (k >= n) continue;
        if (int rc = check_rows("th_copy_rows", rows[k], d[k], TH_F16)) return rc;
        if (rows[k] == 0) continue;
        const int pitch = (d[k] + 7) / 8 * 8;
        if (!src_dev[k] || !dst_dev[k] || dst_stride[k] < pitch) return fail(TH_ERR_BAD_ARG, "th_copy_rows: null pointer or short stride");
        if (!aligned_to(dst_dev[k], 16) || dst_stride[k] % 8 || !aligned_to(src_dev[k], 2)) return fail(TH_ERR_ALIGNMENT, "th_copy_rows: destinations start on 16 bytes");
        a.src[k] = src_dev[k]; a.dst[k] = dst_dev[k]; a.src_stride[k] = src_stride[k]; a.dst_stride[k] = dst_stride[k]; a.rows[k] = rows[k]; a.d[k] = d[k];
        blocks += (rows[k] * (pitch / 8) + 255) / 256;
    }
    a.first_block[kMostCopies] = blocks;
    if (a.d[0] == 0) a.d[0] = 8;  // no rows: nothing is read
    if (n < 2 || a.rows[1] == 0) a.first_block[1] = blocks;
    if (blocks == 0) return TH_OK;
    if (blocks > 0x7fffffffll) return fail(TH_ERR_UNSUPPORTED, "th_copy_rows: too many rows");
    return launch_chained("copy_rows_kernel", copy_rows_kernel, static_cast<unsigned>(blocks), 256, 0, static_cast<cudaStream_t>(stream), 1, a);
}

// The most that any layout of the rows takes.
extern "C" int64_t th_rms_norm_bwd_workspace_bytes(int64_t rows, int d, int dtype) {
    if (rows < 1 || d < 1 || !known_dtype(dtype)) return 0;
    int parts = 0;
    for (int kind : {kPacked, kShifted, kAnyhow})
        for (bool gs : {false, true})
            parts = std::max(parts, dtype == TH_F32 ? norm_bwd_plan<float>(rows, d, kind, gs).parts : norm_bwd_plan<__half>(rows, d, kind, gs).parts);
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
    if (int rc = check_elements("th_rms_norm_bwd", dtype, {sum_dev, grad_y_dev, grad_sum_dev, grad_x_dev})) return rc;
    if (int rc = check_elements("th_rms_norm_bwd", gain_dtype, {gain_dev, grad_gain_dev})) return rc;
    if (int rc = check_elements("th_rms_norm_bwd", TH_F32, {rstd_dev})) return rc;
    RowBwdArgs a{};
    a.s = sum_dev; a.gain = gain_dev; a.gy = grad_y_dev; a.gs = grad_sum_dev; a.rstd = rstd_dev; a.dx = grad_x_dev;
    a.partial = static_cast<float *>(workspace_dev);
    a.s_stride = sum_stride; a.gy_stride = gy_stride; a.gs_stride = gs_stride; a.rows = rows; a.d = d; a.gain_f32 = gain_dtype == TH_F32;
    if (dtype == TH_F32) return norm_bwd<float>(a, grad_gain_dev, gain_dtype, at);
    if (dtype == TH_F16) return norm_bwd<__half>(a, grad_gain_dev, gain_dtype, at);
    return norm_bwd<__nv_bfloat16>(a, grad_gain_dev, gain_dtype, at);
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
    if (int rc = check_elements("th_column_sum", dtype, {g_dev, out_dev})) return rc;
    ColumnArgs sums{};
    sums.g = g_dev; sums.g_stride = g_stride; sums.rows = rows; sums.d = d;
    float *partial = static_cast<float *>(workspace_dev);
    if (dtype == TH_F32) return column_sums<float>(sums, partial, out_dev, dtype, at);
    if (dtype == TH_F16) return column_sums<__half>(sums, partial, out_dev, dtype, at);
    return column_sums<__nv_bfloat16>(sums, partial, out_dev, dtype, at);
}

extern "C" int th_checkpoint_rows(const void *q_dev, int64_t q_stride, const float *scale_dev, void *x_dev, int64_t x_stride, int d_in, const void *g_dev,
                                  int64_t g_stride, void *out_dev, int d_out, void *workspace_dev, int64_t workspace_bytes, int64_t rows, int dtype, void *stream) {
    if (int rc = check_rows("th_checkpoint_rows", rows, d_in, dtype)) return rc;
    if (int rc = check_rows("th_checkpoint_rows", rows, d_out, dtype)) return rc;
    if (dtype == TH_F32) return fail(TH_ERR_UNSUPPORTED, "th_checkpoint_rows: float16 or bfloat16");
    if (rows == 0) return th_column_sum(g_dev, g_stride, out_dev, workspace_dev, workspace_bytes, rows, d_out, dtype, stream);
    if (!q_dev || !scale_dev || !x_dev || !g_dev || !out_dev || q_stride < d_in || x_stride < d_in || g_stride < d_out)
        return fail(TH_ERR_BAD_ARG, "th_checkpoint_rows: null pointer or short stride");
    if (!workspace_dev || workspace_bytes < th_column_sum_workspace_bytes(rows, d_out) || !aligned_to(workspace_dev, 4))
        return fail(TH_ERR_WORKSPACE, "th_checkpoint_rows: scratch missing or too small");
    if (int rc = check_elements("th_checkpoint_rows", dtype, {x_dev, g_dev, out_dev})) return rc;
    if (int rc = check_elements("th_checkpoint_rows", TH_F32, {scale_dev})) return rc;
    const DequantizeArgs a{static_cast<const signed char *>(q_dev), scale_dev, x_dev, q_stride, x_stride, rows, d_in, (d_in + 15) / 16};
    ColumnArgs sums{};
    sums.g = g_dev; sums.g_stride = g_stride; sums.rows = rows; sums.d = d_out;
    float *partial = static_cast<float *>(workspace_dev);
    cudaStream_t at = static_cast<cudaStream_t>(stream);
    return dtype == TH_F16 ? checkpoint_rows<__half>(a, sums, partial, out_dev, dtype, at) : checkpoint_rows<__nv_bfloat16>(a, sums, partial, out_dev, dtype, at);
}
