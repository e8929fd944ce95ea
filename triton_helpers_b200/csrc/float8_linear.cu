// Products of 8-bit floating-point blocks with float32 sums:
//
//     y[m, n] = sum_b a_scale[m, b] b_scale[n / 128, b] sum_{k in b} a[m, k] b[n, k] + bias[n]
//
// and the same over a weight's rows for the input's gradient (b[k, n], scales [k / 128, n / 128]).
#include "chained.cuh"

#include <cuda_fp8.h>

namespace th {
namespace {

constexpr int kBlock = 128;

struct F8Operand {
    const unsigned char *q;
    long long stride;
    const float *scale;
    long long scale_row, scale_block;
};

struct F8Args {
    F8Operand a, b;
    const void *bias;
    void *out;
    long long out_stride;
    long long m;
    int n, k, dtype;
};

__device__ __forceinline__ float f8(unsigned char v) {
    __nv_fp8_e4m3 x;
    x.__x = v;
    return static_cast<float>(x);
}

__device__ __forceinline__ float load_float(const void *p, int i, int dtype) {
    if (dtype == TH_F32) return static_cast<const float *>(p)[i];
    if (dtype == TH_F16) return __half2float(static_cast<const __half *>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}
__device__ __forceinline__ void store_float(void *p, long long i, float v, int dtype) {
    if (dtype == TH_F32) static_cast<float *>(p)[i] = v;
    else if (dtype == TH_F16) static_cast<__half *>(p)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
}

// 64 x 64 results a CTA, 4 x 4 a thread, 32 of K in shared memory at a time.  ALONG_N: b lies [k][n].
template <bool ALONG_N>
__global__ void __launch_bounds__(256) float8_product_kernel(const F8Args g) {
    __shared__ float as[32][65], bs[32][65];
    after_previous();
    const long long m0 = static_cast<long long>(blockIdx.y) * 64;
    const int n0 = blockIdx.x * 64, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    float sum[4][4] = {}, part[4][4] = {};
    for (int k0 = 0; k0 < g.k; k0 += 32) {
        for (int i = threadIdx.x; i < 64 * 32; i += 256) {
            const int r = i / 32, k = i % 32;
            as[k][r] = m0 + r < g.m && k0 + k < g.k ? f8(g.a.q[(m0 + r) * g.a.stride + k0 + k]) : 0.f;
            const int c = ALONG_N ? i % 64 : r, kk = ALONG_N ? i / 64 : k;
            bs[kk][c] = n0 + c < g.n && k0 + kk < g.k ? f8(ALONG_N ? g.b.q[(k0 + kk) * g.b.stride + n0 + c] : g.b.q[(n0 + c) * g.b.stride + k0 + kk]) : 0.f;
        }
        __syncthreads();
        for (int k = 0; k < 32; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) part[i][j] = fmaf(as[k][ty + 16 * i], bs[k][tx + 16 * j], part[i][j]);
        __syncthreads();
        if ((k0 + 32) % kBlock == 0 || k0 + 32 >= g.k) {
            const int b = k0 / kBlock;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const long long m = m0 + ty + 16 * i;
                    const int n = n0 + tx + 16 * j;
                    if (m < g.m && n < g.n) {
                        const float sb = ALONG_N ? g.b.scale[b * g.b.scale_row + (n / kBlock) * g.b.scale_block]
                                                 : g.b.scale[(n / kBlock) * g.b.scale_row + b * g.b.scale_block];
                        sum[i][j] += part[i][j] * g.a.scale[m * g.a.scale_row + b * g.a.scale_block] * sb;
                    }
                    part[i][j] = 0.f;
                }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const long long m = m0 + ty + 16 * i;
            const int n = n0 + tx + 16 * j;
            if (m < g.m && n < g.n) store_float(g.out, m * g.out_stride + n, sum[i][j] + (g.bias ? load_float(g.bias, n, g.dtype) : 0.f), g.dtype);
        }
}

template <bool ALONG_N>
int run_float8(const F8Args &g, cudaStream_t stream) {
    const dim3 grid((g.n + 63) / 64, static_cast<unsigned>((g.m + 63) / 64));
    return launch_chained("float8_product_kernel launch", float8_product_kernel<ALONG_N>, grid, 256, 0, stream, 1, g);
}

int check_f8_shape(const char *what, int64_t rows, int d_in, int d_out, int dtype) {
    if (rows < 0 || d_in < 1 || d_out < 1) return fail(TH_ERR_BAD_ARG, "%s: %lld rows, %d -> %d", what, static_cast<long long>(rows), d_in, d_out);
    if (rows > (1ll << 30) || d_in > (1 << 24) || d_out > (1 << 24))
        return fail(TH_ERR_UNSUPPORTED, "%s: %lld rows, %d -> %d", what, static_cast<long long>(rows), d_in, d_out);
    if (dtype != TH_F32 && dtype != TH_F16 && dtype != TH_BF16) return fail(TH_ERR_UNSUPPORTED, "%s: unknown dtype code %d", what, dtype);
    return TH_OK;
}

int check_f8_operand(const char *what, const F8Operand &o, int d) {
    if (!o.q || !o.scale || o.scale_row < 0 || o.scale_block < 0) return fail(TH_ERR_BAD_ARG, "%s: null pointer or negative stride of the scales", what);
    if (!aligned_to(o.q, 16) || o.stride % 16 || o.stride < d) return fail(TH_ERR_ALIGNMENT, "%s: 8-bit rows start on 16 bytes", what);
    return check_elements(what, TH_F32, {o.scale});
}

int check_f8_output(const char *what, const void *bias, const void *out, int64_t stride, int d, int dtype) {
    if (!out || stride < d) return fail(TH_ERR_BAD_ARG, "%s: null pointer or short stride", what);
    return check_elements(what, dtype, {bias, out});
}

F8Operand f8_operand(const void *q, int64_t stride, const float *scale, int64_t row, int64_t block) {
    return {static_cast<const unsigned char *>(q), stride, scale, row, block};
}

}  // namespace
}  // namespace th

using namespace th;

extern "C" int th_float8_linear(const void *q_dev, int64_t q_stride, const float *scale_dev, int64_t scale_row, int64_t scale_block, const void *weight_dev,
                                int64_t weight_stride, const float *weight_scale_dev, int64_t weight_scale_row, int64_t weight_scale_block,
                                const void *bias_dev, void *y_dev, int64_t y_stride, int64_t rows, int d_in, int d_out, int dtype, void *stream) {
    if (int rc = check_f8_shape("th_float8_linear", rows, d_in, d_out, dtype)) return rc;
    if (rows == 0) return TH_OK;
    F8Args g{f8_operand(q_dev, q_stride, scale_dev, scale_row, scale_block),
             f8_operand(weight_dev, weight_stride, weight_scale_dev, weight_scale_row, weight_scale_block), bias_dev, y_dev, y_stride, rows, d_out, d_in, dtype};
    if (int rc = check_f8_operand("th_float8_linear", g.a, d_in)) return rc;
    if (int rc = check_f8_operand("th_float8_linear", g.b, d_in)) return rc;
    if (int rc = check_f8_output("th_float8_linear", bias_dev, y_dev, y_stride, d_out, dtype)) return rc;
    return run_float8<false>(g, static_cast<cudaStream_t>(stream));
}

// Scratch: the rows' 8-bit values, then their scales, a column block after the other
static int64_t pitch_of(int d) { return (static_cast<int64_t>(d) + 15) / 16 * 16; }

extern "C" int64_t th_float8_quantized_linear_workspace_bytes(int64_t rows, int d_in) {
    return rows < 1 || d_in < 1 ? 0 : rows * (pitch_of(d_in) + 4ll * ((d_in + kBlock - 1) / kBlock)) + 16;
}

extern "C" int th_float8_quantized_linear(const void *x_dev, int64_t x_stride, int x_dtype, const void *weight_dev, int64_t weight_stride,
                                          const float *weight_scale_dev, int64_t weight_scale_row, int64_t weight_scale_block, const void *bias_dev,
                                          void *y_dev, int64_t y_stride, void *workspace_dev, int64_t workspace_bytes, int64_t rows, int d_in, int d_out,
                                          int dtype, void *stream) {
    if (int rc = check_f8_shape("th_float8_quantized_linear", rows, d_in, d_out, dtype)) return rc;
    if (rows == 0) return TH_OK;
    if (!workspace_dev || workspace_bytes < th_float8_quantized_linear_workspace_bytes(rows, d_in) || !aligned_to(workspace_dev, 16))
        return fail(TH_ERR_WORKSPACE, "th_float8_quantized_linear: scratch missing, too small or off 16 bytes");
    char *q = static_cast<char *>(workspace_dev);
    float *scale = reinterpret_cast<float *>(q + rows * pitch_of(d_in));
    F8Args g{f8_operand(q, pitch_of(d_in), scale, 1, rows),
             f8_operand(weight_dev, weight_stride, weight_scale_dev, weight_scale_row, weight_scale_block), bias_dev, y_dev, y_stride, rows, d_out, d_in, dtype};
    // the product's refusals first: nothing is launched for a call that it does not take
    if (int rc = check_f8_operand("th_float8_quantized_linear", g.b, d_in)) return rc;
    if (int rc = check_f8_output("th_float8_quantized_linear", bias_dev, y_dev, y_stride, d_out, dtype)) return rc;
    if (int rc = th_float8_rows(x_dev, x_stride, q, pitch_of(d_in), scale, rows, rows, d_in, x_dtype, stream)) return rc;
    return run_float8<false>(g, static_cast<cudaStream_t>(stream));
}

extern "C" int th_float8_bwd_input(const void *grad_q_dev, int64_t grad_q_stride, const float *grad_scale_dev, int64_t grad_scale_row,
                                   int64_t grad_scale_block, const void *weight_dev, int64_t weight_stride, const float *weight_scale_dev,
                                   int64_t weight_scale_row, int64_t weight_scale_block, void *grad_x_dev, int64_t gx_stride, int64_t rows, int d_in,
                                   int d_out, int dtype, void *stream) {
    if (int rc = check_f8_shape("th_float8_bwd_input", rows, d_in, d_out, dtype)) return rc;
    if (rows == 0) return TH_OK;
    F8Args g{f8_operand(grad_q_dev, grad_q_stride, grad_scale_dev, grad_scale_row, grad_scale_block),
             f8_operand(weight_dev, weight_stride, weight_scale_dev, weight_scale_row, weight_scale_block), nullptr, grad_x_dev, gx_stride, rows, d_in, d_out, dtype};
    if (int rc = check_f8_operand("th_float8_bwd_input", g.a, d_out)) return rc;
    if (int rc = check_f8_operand("th_float8_bwd_input", g.b, d_in)) return rc;
    if (int rc = check_f8_output("th_float8_bwd_input", nullptr, grad_x_dev, gx_stride, d_in, dtype)) return rc;
    return run_float8<true>(g, static_cast<cudaStream_t>(stream));
}
