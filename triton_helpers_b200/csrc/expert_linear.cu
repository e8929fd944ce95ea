// Linear layers of several experts on rows sorted by expert, with float32 sums:
//
//     y[r] = x[r] W_e^T      grad_x[r] = grad_y[r] W_e      grad_W_e = sum_r grad_y[r]^T x[r]      for rows r of expert e
//
// The rows' ends are read on the device.
#include "chained.cuh"

#include <algorithm>

namespace th {
namespace {

struct ExpertArgs {
    const void *x, *w;        // along the output's rows, and along its columns
    long long x_stride, w_stride, expert_stride;
    const int32_t *ends;
    void *out;
    long long out_stride;
    int rows, experts, n, k;  // of the output's columns and of what is summed over
};

// First row behind expert e; the row that it starts at is that of the expert before
__device__ __forceinline__ int end_of(const int32_t *ends, int e, int rows) {
    int end = 0;
    for (int i = 0; i <= e; ++i) end = max(end, min(ends[i], rows));
    return end;
}

// 64 x 64 results a CTA, 4 x 4 a thread, 32 of K in shared memory at a time.  ALONG_N: the weight lies [k][n].
// The z axis goes over experts, and one more for the rows behind the last end.
template <typename T, bool ALONG_N>
__global__ void __launch_bounds__(256) expert_product_kernel(const ExpertArgs g) {
    __shared__ float as[32][65], bs[32][65];
    after_previous();
    const int e = blockIdx.z, tx = threadIdx.x & 15, ty = threadIdx.x >> 4, n0 = blockIdx.x * 64;
    const bool behind = e == g.experts;
    const int first = e ? end_of(g.ends, e - 1, g.rows) : 0, end = behind ? g.rows : end_of(g.ends, e, g.rows);
    const T *w = static_cast<const T *>(g.w) + (behind ? 0 : e) * g.expert_stride;
    for (int m0 = first + blockIdx.y * 64; m0 < end; m0 += gridDim.y * 64) {
        float sum[4][4] = {};
        for (int k0 = 0; k0 < g.k && !behind; k0 += 32) {
            for (int i = threadIdx.x; i < 64 * 32; i += 256) {
                const int r = i / 32, k = i % 32;
                as[k][r] = m0 + r < end && k0 + k < g.k ? to_float<T>(static_cast<const T *>(g.x)[(m0 + r) * g.x_stride + k0 + k]) : 0.f;
                const int c = ALONG_N ? i % 64 : r, kk = ALONG_N ? i / 64 : k;
                bs[kk][c] = n0 + c < g.n && k0 + kk < g.k ? to_float<T>(ALONG_N ? w[(k0 + kk) * g.w_stride + n0 + c] : w[(n0 + c) * g.w_stride + k0 + kk]) : 0.f;
            }
            __syncthreads();
            for (int k = 0; k < 32; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) sum[i][j] = fmaf(as[k][ty + 16 * i], bs[k][tx + 16 * j], sum[i][j]);
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
                if (m < end && n < g.n) static_cast<T *>(g.out)[m * g.out_stride + n] = from_float<T>(sum[i][j]);
            }
    }
}

// grad_W: x is grad_y (its columns are the output's rows), w is x
template <typename T>
__global__ void __launch_bounds__(256) expert_weight_kernel(const ExpertArgs g, int m_size) {
    __shared__ float as[32][65], bs[32][65];
    after_previous();
    const int e = blockIdx.z, tx = threadIdx.x & 15, ty = threadIdx.x >> 4, n0 = blockIdx.x * 64, m0 = blockIdx.y * 64;
    const int first = e ? end_of(g.ends, e - 1, g.rows) : 0, end = end_of(g.ends, e, g.rows);
    float sum[4][4] = {};
    for (int r0 = first; r0 < end; r0 += 32) {
        for (int i = threadIdx.x; i < 64 * 32; i += 256) {
            const int r = r0 + i / 64, c = i % 64;
            as[i / 64][c] = r < end && m0 + c < m_size ? to_float<T>(static_cast<const T *>(g.x)[r * g.x_stride + m0 + c]) : 0.f;
            bs[i / 64][c] = r < end && n0 + c < g.n ? to_float<T>(static_cast<const T *>(g.w)[r * g.w_stride + n0 + c]) : 0.f;
        }
        __syncthreads();
        for (int k = 0; k < 32; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) sum[i][j] = fmaf(as[k][ty + 16 * i], bs[k][tx + 16 * j], sum[i][j]);
        __syncthreads();
    }
    T *out = static_cast<T *>(g.out) + static_cast<long long>(e) * m_size * g.n;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
            if (m < m_size && n < g.n) out[static_cast<long long>(m) * g.n + n] = from_float<T>(sum[i][j]);
        }
}

constexpr int kMostExperts = 1024;

int check_experts(const char *what, int64_t rows, int experts, int d_in, int d_out, int dtype, const int32_t *ends) {
    if (rows < 0 || experts < 1 || d_in < 1 || d_out < 1)
        return fail(TH_ERR_BAD_ARG, "%s: %lld rows, %d experts, %d -> %d", what, static_cast<long long>(rows), experts, d_in, d_out);
    if (rows > (1ll << 30) || d_in > (1 << 24) || d_out > (1 << 24) || experts > kMostExperts)
        return fail(TH_ERR_UNSUPPORTED, "%s: %lld rows, %d experts, %d -> %d", what, static_cast<long long>(rows), experts, d_in, d_out);
    if (dtype != TH_F16 && dtype != TH_BF16) return fail(TH_ERR_UNSUPPORTED, "%s: float16 or bfloat16, not dtype code %d", what, dtype);
    if (!ends) return fail(TH_ERR_BAD_ARG, "%s: null pointer", what);
    return check_elements(what, TH_F32, {ends});
}

int check_16(const char *what, const void *p, int64_t stride, int d) {
    if (!p || stride < d) return fail(TH_ERR_BAD_ARG, "%s: null pointer or short stride", what);
    if (!aligned_to(p, 16) || stride % 8) return fail(TH_ERR_ALIGNMENT, "%s: operand rows start on 16 bytes", what);
    return TH_OK;
}

template <bool ALONG_N>
int run_experts(const ExpertArgs &g, int dtype, cudaStream_t stream) {
    const dim3 grid((g.n + 63) / 64, std::min(64, (g.rows + 63) / 64), g.experts + 1);
    return launch_chained("expert_product_kernel launch", dtype == TH_F16 ? expert_product_kernel<__half, ALONG_N> : expert_product_kernel<__nv_bfloat16, ALONG_N>, grid,
                          256, 0, stream, 1, g);
}

int check_weight(const char *what, const void *w, int64_t stride, int64_t expert_stride, int d_in, int d_out) {
    if (int rc = check_16(what, w, stride, d_in)) return rc;
    if (expert_stride < stride * (d_out - 1) + d_in) return fail(TH_ERR_BAD_ARG, "%s: experts overlap", what);
    return expert_stride % 8 ? fail(TH_ERR_ALIGNMENT, "%s: experts start on 16 bytes", what) : TH_OK;
}

}  // namespace
}  // namespace th

using namespace th;

extern "C" int th_expert_linear_fwd(const void *x_dev, int64_t x_stride, const void *weight_dev, int64_t weight_stride, int64_t expert_stride,
                                    const int32_t *ends_dev, void *y_dev, int64_t y_stride, int64_t rows, int experts, int d_in, int d_out, int dtype,
                                    void *stream) {
    if (int rc = check_experts("th_expert_linear_fwd", rows, experts, d_in, d_out, dtype, ends_dev)) return rc;
    if (rows == 0) return TH_OK;
    if (int rc = check_16("th_expert_linear_fwd", x_dev, x_stride, d_in)) return rc;
    if (int rc = check_weight("th_expert_linear_fwd", weight_dev, weight_stride, expert_stride, d_in, d_out)) return rc;
    if (!y_dev || y_stride < d_out) return fail(TH_ERR_BAD_ARG, "th_expert_linear_fwd: null pointer or short stride");
    if (int rc = check_elements("th_expert_linear_fwd", dtype, {y_dev})) return rc;
    const ExpertArgs g{x_dev, weight_dev, x_stride, weight_stride, expert_stride, ends_dev, y_dev, y_stride, static_cast<int>(rows), experts, d_out, d_in};
    return run_experts<false>(g, dtype, static_cast<cudaStream_t>(stream));
}

extern "C" int th_expert_linear_bwd_input(const void *grad_y_dev, int64_t gy_stride, const void *weight_dev, int64_t weight_stride, int64_t expert_stride,
                                          const int32_t *ends_dev, void *grad_x_dev, int64_t gx_stride, int64_t rows, int experts, int d_in, int d_out,
                                          int dtype, void *stream) {
    if (int rc = check_experts("th_expert_linear_bwd_input", rows, experts, d_in, d_out, dtype, ends_dev)) return rc;
    if (rows == 0) return TH_OK;
    if (int rc = check_16("th_expert_linear_bwd_input", grad_y_dev, gy_stride, d_out)) return rc;
    if (int rc = check_weight("th_expert_linear_bwd_input", weight_dev, weight_stride, expert_stride, d_in, d_out)) return rc;
    if (!grad_x_dev || gx_stride < d_in) return fail(TH_ERR_BAD_ARG, "th_expert_linear_bwd_input: null pointer or short stride");
    if (int rc = check_elements("th_expert_linear_bwd_input", dtype, {grad_x_dev})) return rc;
    const ExpertArgs g{grad_y_dev, weight_dev, gy_stride, weight_stride, expert_stride, ends_dev, grad_x_dev, gx_stride, static_cast<int>(rows), experts, d_in, d_out};
    return run_experts<true>(g, dtype, static_cast<cudaStream_t>(stream));
}

extern "C" int th_expert_linear_bwd_weight(const void *grad_y_dev, int64_t gy_stride, const void *x_dev, int64_t x_stride, const int32_t *ends_dev,
                                           void *grad_weight_dev, int64_t rows, int experts, int d_in, int d_out, int dtype, void *stream) {
    if (int rc = check_experts("th_expert_linear_bwd_weight", rows, experts, d_in, d_out, dtype, ends_dev)) return rc;
    if (!grad_weight_dev) return fail(TH_ERR_BAD_ARG, "th_expert_linear_bwd_weight: null pointer");
    if (int rc = check_elements("th_expert_linear_bwd_weight", dtype, {grad_weight_dev})) return rc;
    cudaStream_t at = static_cast<cudaStream_t>(stream);
    if (rows == 0) return cuda_status(cudaMemsetAsync(grad_weight_dev, 0, static_cast<size_t>(experts) * d_in * d_out * 2, at), "th_expert_linear_bwd_weight");
    if (int rc = check_16("th_expert_linear_bwd_weight", grad_y_dev, gy_stride, d_out)) return rc;
    if (int rc = check_16("th_expert_linear_bwd_weight", x_dev, x_stride, d_in)) return rc;
    const ExpertArgs g{grad_y_dev, x_dev, gy_stride, x_stride, 0, ends_dev, grad_weight_dev, d_in, static_cast<int>(rows), experts, d_in, 0};
    const dim3 grid((d_in + 63) / 64, (d_out + 63) / 64, experts);
    return launch_chained("expert_weight_kernel launch", dtype == TH_F16 ? expert_weight_kernel<__half> : expert_weight_kernel<__nv_bfloat16>, grid, 256, 0, at, 1, g,
                          d_out);
}
