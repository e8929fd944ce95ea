// 8-bit floating-point blocks: rows in blocks of 1 x 128, weights in blocks of 128 x 128, and back.
//
//     a = max(max |x|, 2^-60) over the block      q = e4m3(x * (448 / a))      scale = a / 448
//
// Streaming kernels, bound by memory.  8192 x 4096 bfloat16: rows 19.5 us (100 MB, 5.2 TB/s), back to bfloat16 21 us (4.8); a 4096 x 4096 weight 13 us
// (50 MB, 3.9).  Sixteen lanes hold 128 columns of a row, eight each, so that a block's largest magnitude is one reduction within half a warp.  Magnitudes are compared as integers: a NaN is above infinity, and infinity above every number.
#include "chained.cuh"

#include <algorithm>

namespace th {
namespace {

constexpr int kBlock = 128;
constexpr int kQuantThreads = 256;
constexpr float kLeast = 0x1p-60f, kTop = 448.f;

__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// Four values of e4m3, saturating (x * (448 / a) rounds to at most 448, so nothing does)
__device__ __forceinline__ uint32_t four_e4m3(float a, float b, float c, float d) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return static_cast<uint32_t>(lo) | static_cast<uint32_t>(hi) << 16;
}

__device__ __forceinline__ void four_floats(uint32_t q, float *v) {
    uint32_t lo, hi;  // e4m3 -> f16 is exact
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(lo) : "h"(static_cast<uint16_t>(q)));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(hi) : "h"(static_cast<uint16_t>(q >> 16)));
    const float2 a = __half22float2(*reinterpret_cast<__half2 *>(&lo)), b = __half22float2(*reinterpret_cast<__half2 *>(&hi));
    v[0] = a.x;
    v[1] = a.y;
    v[2] = b.x;
    v[3] = b.y;
}

// Eight elements of a row as they lie in memory, zeros behind its end: 16-bit ones take half the registers that their values would.
// WIDE: they start on 16 bytes.
template <typename T>
struct __align__(16) Eight {
    T v[8];
};

template <typename T, bool WIDE>
__device__ __forceinline__ Eight<T> load8(const T *from, int valid) {
    Eight<T> x;
    if (WIDE && valid >= 8) {
#pragma unroll
        for (unsigned p = 0; p < sizeof(x) / 16; ++p) reinterpret_cast<uint4 *>(&x)[p] = reinterpret_cast<const uint4 *>(from)[p];
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x.v[e] = e < valid ? from[e] : from_float<T>(0.f);
    }
    return x;
}

// The largest magnitude of eight elements, as bits: float32's own, or two 16-bit ones that are compared side by side
template <typename T>
__device__ __forceinline__ uint32_t most_of(const Eight<T> &x) {
    if constexpr (sizeof(T) == 2) {
        const uint4 w = *reinterpret_cast<const uint4 *>(&x);
        constexpr uint32_t kSigns = 0x7fff7fffu;
        return __vmaxu2(__vmaxu2(w.x & kSigns, w.y & kSigns), __vmaxu2(w.z & kSigns, w.w & kSigns));
    } else {
        uint32_t most = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) most = max(most, magnitude(x.v[e]));
        return most;
    }
}
template <typename T>
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    if constexpr (sizeof(T) == 2) return __vmaxu2(a, b);
    else return max(a, b);
}
// The same as the bits of a float32
template <typename T>
__device__ __forceinline__ uint32_t as_float_bits(uint32_t most) {
    if constexpr (sizeof(T) == 4) return most;
    const unsigned short one = static_cast<unsigned short>(max(most & 0xffffu, most >> 16));
    return __float_as_uint(to_float<T>(*reinterpret_cast<const T *>(&one)));
}

// What a block's largest magnitude makes of it, in one division: for even lanes the factor that the block's values take (zero where it is not finite),
// for odd ones its scale (then a NaN)
__device__ __forceinline__ float block_part(uint32_t most) {
    const bool odd = threadIdx.x & 1;
    const float a = fmaxf(__uint_as_float(most), kLeast), part = __fdiv_rn(odd ? a : kTop, odd ? kTop : a);
    return most < 0x7f800000u ? part : odd ? __uint_as_float(0x7fc00000u) : 0.f;
}

template <typename T>
__device__ __forceinline__ void store8(unsigned char *to, int valid, const Eight<T> &from, float factor) {
    const bool finite = factor != 0.f;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = to_float<T>(from.v[e]);
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const float *x = v + 4 * h;
        w[h] = finite ? four_e4m3(__fmul_rn(x[0], factor), __fmul_rn(x[1], factor), __fmul_rn(x[2], factor), __fmul_rn(x[3], factor)) : 0u;
    }
    if (valid >= 8) {
        *reinterpret_cast<uint2 *>(to) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < valid) to[e] = static_cast<unsigned char>(w[e >> 2] >> (8 * (e & 3)));
    }
}

struct QuantArgs {
    const void *x;
    long long x_stride;
    unsigned char *q;
    long long q_stride;
    float *scale;
    long long scale_block;
    long long rows;
    int d, blocks;
    void *copy;  // of 16-bit rows, or null: 3001 x 777 to and from 1000, forward and backward, 89 us with a copy of its own, 87 with this one
    long long copy_stride;
};

// A tile is 16 rows x kAhead column blocks: kAhead loads of each thread are on their way together, those of a CTA's next tile while it works on this one,
// and the scales of neighbouring rows, which lie side by side, leave together.  8192 x 4096 bfloat16: with a tile a CTA 30 us.
constexpr int kAhead = 4;

template <typename T, bool WIDE>
__device__ __forceinline__ void load_tile(const QuantArgs &a, int tile, int columns, Eight<T> (&v)[kAhead]) {
    const int group = tile / columns, first = (tile - group * columns) * kAhead * kBlock + 8 * (threadIdx.x & 15);
    const long long row = static_cast<long long>(group) * 16 + (threadIdx.x >> 4);
    const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) v[i] = load8<T, WIDE>(x + first + i * kBlock, row < a.rows ? a.d - first - i * kBlock : 0);
}

template <typename T>
__device__ __forceinline__ void finish_tile(const QuantArgs &a, int tile, int columns, const Eight<T> (&v)[kAhead]) {
    const int group = tile / columns, first = (tile - group * columns) * kAhead, part = threadIdx.x & 15;
    const long long row = static_cast<long long>(group) * 16 + (threadIdx.x >> 4);
    const unsigned mask = 0xffffu << (threadIdx.x & 16);  // half a warp
    // Four blocks' largest magnitudes at once: lanes hand each other the blocks that the other side goes on with, until four of them have one
    // block to themselves; so the four blocks take one division, with five exchanges for 16 (8192 x 4096 bfloat16: 27.5 us block by block).
    static_assert(kAhead == 4, "four blocks to sixteen lanes");
    const bool high = part & 8, upper = part & 4;
    uint32_t most[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) most[i] = most_of(v[i]);
    const uint32_t first_two = larger<T>(high ? most[2] : most[0], __shfl_xor_sync(mask, high ? most[0] : most[2], 8));
    const uint32_t last_two = larger<T>(high ? most[3] : most[1], __shfl_xor_sync(mask, high ? most[1] : most[3], 8));
    uint32_t mine = larger<T>(upper ? last_two : first_two, __shfl_xor_sync(mask, upper ? first_two : last_two, 4));
    mine = larger<T>(mine, __shfl_xor_sync(mask, mine, 2));
    mine = larger<T>(mine, __shfl_xor_sync(mask, mine, 1));
    const float part_of = block_part(as_float_bits<T>(mine));
    const int b_mine = first + (part >> 2);
    if ((part & 3) == 1 && b_mine < a.blocks && row < a.rows) a.scale[b_mine * a.scale_block + row] = part_of;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
        const float factor = __shfl_sync(mask, part_of, 4 * i, 16);
        const int c = (first + i) * kBlock + 8 * part;
        if (c < a.d && row < a.rows) {
            store8(a.q + row * a.q_stride + c, a.d - c, v[i], factor);
            if constexpr (sizeof(T) == 2)
                if (a.copy)
                    *reinterpret_cast<uint4 *>(static_cast<T *>(a.copy) + row * a.copy_stride + c) = *reinterpret_cast<const uint4 *>(&v[i]);
        }
    }
}

template <typename T, bool WIDE>
__global__ void __launch_bounds__(kQuantThreads, sizeof(T) == 2 ? 4 : 3) float8_rows_kernel(const QuantArgs a, int tiles, int columns) {
    after_previous();
    int tile = blockIdx.x;
    Eight<T> v[kAhead], next[kAhead];
    load_tile<T, WIDE>(a, tile, columns, v);
    while (true) {
        const int then = tile + gridDim.x;
        if (then < tiles) load_tile<T, WIDE>(a, then, columns, next);
        finish_tile(a, tile, columns, v);
        if (then >= tiles) break;
        tile = then;
#pragma unroll
        for (int i = 0; i < kAhead; ++i) v[i] = next[i];
    }
}

// A CTA takes a block of 128 x 128: four rows of each thread in registers
constexpr int kWeightThreads = 512;

template <typename T, bool WIDE>
__global__ void __launch_bounds__(kWeightThreads, sizeof(T) == 2 ? 3 : 2) float8_weight_kernel(const QuantArgs a) {
    __shared__ uint32_t warps[kWeightThreads / 32];
    after_previous();
    constexpr int kRows = kBlock * 16 / kWeightThreads;
    const int c = blockIdx.x * kBlock + 8 * (threadIdx.x & 15), r0 = threadIdx.x >> 4;
    const long long first = static_cast<long long>(blockIdx.y) * kBlock;
    Eight<T> v[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const long long row = first + r0 + kWeightThreads / 16 * i;
        v[i] = load8<T, WIDE>(static_cast<const T *>(a.x) + row * a.x_stride + c, row < a.rows ? a.d - c : 0);
    }
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < kRows; ++i) most = larger<T>(most, most_of(v[i]));
    most = __reduce_max_sync(~0u, as_float_bits<T>(most));
    if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = most;
    __syncthreads();
    most = __reduce_max_sync(~0u, warps[threadIdx.x & (kWeightThreads / 32 - 1)]);
    const float part = block_part(most), factor = __shfl_sync(~0u, part, 0);
    if (threadIdx.x == 1) a.scale[static_cast<long long>(blockIdx.y) * a.blocks + blockIdx.x] = part;
    if (c >= a.d) return;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const long long row = first + r0 + kWeightThreads / 16 * i;
        if (row < a.rows) store8(a.q + row * a.q_stride + c, a.d - c, v[i], factor);
    }
}

struct ValueArgs {
    const unsigned char *q;
    long long q_stride;
    const float *scale;
    long long scale_row, scale_block;
    int block_shift;  // 0 or 7: rows of a block
    void *out;
    long long out_stride;
    long long rows;
    int d;
};

// Sixteen columns a thread: one load of 16 bytes
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kQuantThreads) float8_values_kernel(const ValueArgs a) {
    after_previous();
    const int chunks = (a.d + 15) / 16;
    const long long id = static_cast<long long>(blockIdx.x) * kQuantThreads + threadIdx.x, row = id / chunks;
    if (row >= a.rows) return;
    const int c = static_cast<int>(id - row * chunks) * 16, valid = a.d - c;
    const float s = a.scale[(row >> a.block_shift) * a.scale_row + (c / kBlock) * a.scale_block];
    const unsigned char *q = a.q + row * a.q_stride + c;
    uint32_t w[4] = {0, 0, 0, 0};
    if (valid >= 16) {
        const uint4 in = *reinterpret_cast<const uint4 *>(q);
        w[0] = in.x;
        w[1] = in.y;
        w[2] = in.z;
        w[3] = in.w;
    } else {
#pragma unroll
        for (int e = 0; e < 16; ++e)
            if (e < valid) w[e >> 2] |= static_cast<uint32_t>(q[e]) << (8 * (e & 3));
    }
    T *out = static_cast<T *>(a.out) + row * a.out_stride + c;
    constexpr int N = 16 / static_cast<int>(sizeof(T));
    struct __align__(16) Packet {
        T v[N];
    };
    float v[16];
#pragma unroll
    for (int k = 0; k < 4; ++k) four_floats(w[k], v + 4 * k);
    if (WIDE && valid >= 16) {
#pragma unroll
        for (int p = 0; p < 16 / N; ++p) {
            Packet o;
#pragma unroll
            for (int e = 0; e < N; ++e) o.v[e] = from_float<T>(v[p * N + e] * s);
            reinterpret_cast<Packet *>(out)[p] = o;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 16; ++e)
            if (e < valid) out[e] = from_float<T>(v[e] * s);
    }
}

// least: the smallest stride of the floats' rows (rows that are read may overlap)
int check_blocks(const char *what, const void *x, int64_t x_stride, int64_t least, const void *q, int64_t q_stride, const float *scale, int64_t rows, int d,
                 int dtype) {
    if (rows < 0 || d < 1) return fail(TH_ERR_BAD_ARG, "%s: %lld rows of %d", what, static_cast<long long>(rows), d);
    if (rows > (1ll << 30) || d > (1 << 24)) return fail(TH_ERR_UNSUPPORTED, "%s: %lld rows of %d", what, static_cast<long long>(rows), d);
    if (dtype != TH_F32 && dtype != TH_F16 && dtype != TH_BF16) return fail(TH_ERR_UNSUPPORTED, "%s: unknown dtype code %d", what, dtype);
    if (rows == 0) return TH_OK;
    if (!x || !q || !scale || x_stride < least) return fail(TH_ERR_BAD_ARG, "%s: null pointer or short stride", what);
    if (!aligned_to(q, 16) || q_stride % 16 || q_stride < d) return fail(TH_ERR_ALIGNMENT, "%s: 8-bit rows start on 16 bytes", what);
    if (int rc = check_elements(what, TH_F32, {scale})) return rc;
    return check_elements(what, dtype, {x});
}

bool wide_rows(const void *x, int64_t stride, int dtype) { return aligned_to(x, 16) && stride * static_cast<int64_t>(dtype_bytes(dtype)) % 16 == 0; }

// fn(T{}, std::integral_constant<bool, WIDE>{})
template <typename Fn>
int with_type(int dtype, bool wide, const Fn &fn) {
    const auto at = [&](auto t) { return wide ? fn(t, std::true_type{}) : fn(t, std::false_type{}); };
    return dtype == TH_F32 ? at(float{}) : dtype == TH_F16 ? at(__half{}) : at(__nv_bfloat16{});
}

}  // namespace
}  // namespace th

using namespace th;

static int float8_rows(const char *what, const void *x_dev, int64_t x_stride, void *q_dev, int64_t q_stride, float *scale_dev, int64_t scale_block, void *copy_dev,
                       int64_t copy_stride, int64_t rows, int d, int dtype, void *stream) {
    if (int rc = check_blocks(what, x_dev, x_stride, 0, q_dev, q_stride, scale_dev, rows, d, dtype)) return rc;
    if (rows == 0) return TH_OK;
    if (scale_block < rows) return fail(TH_ERR_BAD_ARG, "%s: short stride of the scales", what);
    const QuantArgs a{x_dev, x_stride, static_cast<unsigned char *>(q_dev), q_stride, scale_dev, scale_block, rows, d, (d + kBlock - 1) / kBlock, copy_dev, copy_stride};
    const int columns = (a.blocks + kAhead - 1) / kAhead;
    const int64_t tiles = (rows + 15) / 16 * columns;
    if (tiles > 0x7fffffff - 0x10000) return fail(TH_ERR_UNSUPPORTED, "%s: %lld rows of %d", what, static_cast<long long>(rows), d);
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>(tiles, static_cast<int64_t>(sm_count()) * (dtype == TH_F32 ? 3 : 4)));
    return with_type(dtype, wide_rows(x_dev, x_stride, dtype), [&](auto t, auto wide) {
        return launch_chained("float8_rows_kernel launch", float8_rows_kernel<decltype(t), decltype(wide)::value>, grid, kQuantThreads, 0,
                              static_cast<cudaStream_t>(stream), 1, a, static_cast<int>(tiles), columns);
    });
}

extern "C" int th_float8_rows(const void *x_dev, int64_t x_stride, void *q_dev, int64_t q_stride, float *scale_dev, int64_t scale_block, int64_t rows, int d,
                              int dtype, void *stream) {
    return float8_rows("th_float8_rows", x_dev, x_stride, q_dev, q_stride, scale_dev, scale_block, nullptr, 0, rows, d, dtype, stream);
}

extern "C" int th_float8_rows_copied(const void *x_dev, int64_t x_stride, void *q_dev, int64_t q_stride, float *scale_dev, int64_t scale_block, void *copy_dev,
                                     int64_t copy_stride, int64_t rows, int d, int dtype, void *stream) {
    if (dtype != TH_F16 && dtype != TH_BF16) return fail(TH_ERR_UNSUPPORTED, "th_float8_rows_copied: float16 or bfloat16, not dtype code %d", dtype);
    if (rows > 0 && (!copy_dev || copy_stride < d)) return fail(TH_ERR_BAD_ARG, "th_float8_rows_copied: null pointer or short stride");
    if (!aligned_to(copy_dev, 16) || copy_stride % 8) return fail(TH_ERR_ALIGNMENT, "th_float8_rows_copied: copied rows start on 16 bytes");
    return float8_rows("th_float8_rows_copied", x_dev, x_stride, q_dev, q_stride, scale_dev, scale_block, copy_dev, copy_stride, rows, d, dtype, stream);
}

extern "C" int th_float8_weight(const void *w_dev, int64_t w_stride, void *q_dev, int64_t q_stride, float *scale_dev, int64_t rows, int d, int dtype,
                                void *stream) {
    if (int rc = check_blocks("th_float8_weight", w_dev, w_stride, 0, q_dev, q_stride, scale_dev, rows, d, dtype)) return rc;
    if (rows == 0) return TH_OK;
    if (rows > 65535ll * kBlock) return fail(TH_ERR_UNSUPPORTED, "th_float8_weight: %lld rows", static_cast<long long>(rows));
    const QuantArgs a{w_dev, w_stride, static_cast<unsigned char *>(q_dev), q_stride, scale_dev, 0, rows, d, (d + kBlock - 1) / kBlock, nullptr, 0};
    const dim3 grid(static_cast<unsigned>(a.blocks), static_cast<unsigned>((rows + kBlock - 1) / kBlock));
    return with_type(dtype, wide_rows(w_dev, w_stride, dtype), [&](auto t, auto wide) {
        return launch_chained("float8_weight_kernel launch", float8_weight_kernel<decltype(t), decltype(wide)::value>, grid, kWeightThreads, 0,
                              static_cast<cudaStream_t>(stream), 1, a);
    });
}

extern "C" int th_float8_values(const void *q_dev, int64_t q_stride, const float *scale_dev, int64_t scale_row, int64_t scale_block, int block_rows,
                                void *out_dev, int64_t out_stride, int64_t rows, int d, int dtype, void *stream) {
    if (block_rows != 1 && block_rows != kBlock) return fail(TH_ERR_BAD_ARG, "th_float8_values: blocks of %d rows", block_rows);
    if (int rc = check_blocks("th_float8_values", out_dev, out_stride, d, q_dev, q_stride, scale_dev, rows, d, dtype)) return rc;
    if (rows == 0) return TH_OK;
    if (scale_row < 0 || scale_block < 0) return fail(TH_ERR_BAD_ARG, "th_float8_values: negative stride of the scales");
    const ValueArgs a{static_cast<const unsigned char *>(q_dev), q_stride, scale_dev, scale_row, scale_block, block_rows == 1 ? 0 : 7, out_dev, out_stride,
                      rows, d};
    const long long blocks = (rows * ((d + 15) / 16) + kQuantThreads - 1) / kQuantThreads;
    if (blocks > 0x7fffffffll) return fail(TH_ERR_UNSUPPORTED, "th_float8_values: %lld rows of %d", static_cast<long long>(rows), d);
    return with_type(dtype, wide_rows(out_dev, out_stride, dtype), [&](auto t, auto wide) {
        return launch_chained("float8_values_kernel launch", float8_values_kernel<decltype(t), decltype(wide)::value>, static_cast<unsigned>(blocks), kQuantThreads,
                              0, static_cast<cudaStream_t>(stream), 1, a);
    });
}
