// Linear layers of any width: 8-bit integers with a scale per token and per channel, and 16-bit products in the three forms that a
// layer's forward and backward pass take.  The products are wide_gemm_kernel's; what is here chooses its tile and adds up split sums.
#include "wide_gemm.cuh"

#include <algorithm>

namespace th {
namespace {

// How a product is cut: tile width, CTAs per tile, transposed or not, and the parts that K is split into.
struct ProductPlan {
    int bn, cg;
    bool swap;
    int splits;
};

int divide_up(long long a, long long b) { return static_cast<int>((a + b - 1) / b); }

// Parts of K so that tiles x parts fill the GPU, each of at least `least` stages
int split_count(long long tiles, int k_tiles, int least) {
    const long long want = std::max(1ll, sm_count() / std::max(1ll, tiles));
    const int parts = static_cast<int>(std::min<long long>(want, std::max(1, k_tiles / least)));
    const int per = divide_up(k_tiles, parts);
    return divide_up(k_tiles, per);
}

ProductPlan plan_product(int m, int n, int k, int elem_bytes) {
    ProductPlan p{};
    const int k_tiles = divide_up(k, 128 / elem_bytes);
    if (elem_bytes == 1 && m <= 128) {
        p.swap = true;
        p.cg = 1;
        p.bn = m <= 16 ? 16 : m <= 32 ? 32 : m <= 64 ? 64 : 128;
        p.splits = split_count(divide_up(n, kGemmRows), k_tiles, 4);
        return p;
    }
    const long long pairs = static_cast<long long>(divide_up(m, 256)) * divide_up(n, 256);
    if (pairs >= 40) {
        p.bn = 256;
        p.cg = 2;
        p.splits = 1;
    } else {
        p.bn = 128;
        p.cg = 1;
        p.splits = split_count(static_cast<long long>(divide_up(m, 128)) * divide_up(n, 128), k_tiles, 8);
    }
    return p;
}

int64_t product_workspace(int64_t m, int n, int k, int elem_bytes) {
    if (m < 1 || n < 1 || k < 1 || m > 0x7fffffffll) return 0;
    const ProductPlan p = plan_product(static_cast<int>(m), n, k, elem_bytes);
    return p.splits > 1 ? static_cast<int64_t>(p.splits) * m * n * 4 : 0;
}

// ---- sums of a split product ------------------------------------------------------------------------------

struct SplitArgs {
    const uint32_t *partial;
    int splits;
    long long rows, split_elems;
    int n;
    const float *row_scale, *column_scale;
    const void *bias;
    int bias_dtype;
    void *out;
    long long out_stride;
    int out_dtype;
};

// The parts are added in their order: integers exactly, float32 sums the same way at every call.
template <bool INT>
__global__ void __launch_bounds__(256) split_sum_kernel(const SplitArgs a) {
    const int n = blockIdx.x * 256 + threadIdx.x;
    const long long row = blockIdx.y + static_cast<long long>(blockIdx.z) * gridDim.y;
    if (n >= a.n || row >= a.rows) return;
    const uint32_t *p = a.partial + row * a.n + n;
    float v;
    if constexpr (INT) {
        int sum = 0;
        for (int s = 0; s < a.splits; ++s) sum += static_cast<int>(p[s * a.split_elems]);
        v = static_cast<float>(sum) * (a.row_scale[row] * a.column_scale[n]);
    } else {
        v = 0.f;
        for (int s = 0; s < a.splits; ++s) v += __uint_as_float(p[s * a.split_elems]);
    }
    if (a.bias) v += bias_at(a.bias, a.bias_dtype, n);
    const long long at = row * a.out_stride + n;
    if (a.out_dtype == TH_F32) static_cast<float *>(a.out)[at] = v;
    else if (a.out_dtype == TH_F16) static_cast<__half *>(a.out)[at] = __float2half_rn(v);
    else static_cast<__nv_bfloat16 *>(a.out)[at] = __float2bfloat16_rn(v);
}

// ---- one product ------------------------------------------------------------------------------------------

struct Product {
    Operand a, b;  // a along the output's rows, b along its columns
    int k;
    const float *row_scale, *column_scale;
    const void *bias;
    void *out;
    long long out_stride;
    int out_dtype, bias_dtype;
    void *workspace;
    long long workspace_bytes;
};

template <int EB, bool A_MN, bool B_MN>
int run_product(const char *what, const Product &p, bool bf16, cudaStream_t stream) {
    const ProductPlan plan = plan_product(p.a.rows, p.b.rows, p.k, EB);
    GemmArgs g{};
    g.splits = plan.splits;
    g.out = p.out;
    g.out_stride = p.out_stride;
    g.out_dtype = p.out_dtype;
    g.lane_scale = plan.swap ? p.column_scale : p.row_scale;
    g.column_scale = plan.swap ? p.row_scale : p.column_scale;
    g.bias = p.bias;
    g.bias_dtype = p.bias_dtype;
    if (plan.splits > 1) {
        const long long elems = static_cast<long long>(p.a.rows) * p.b.rows;
        if (!p.workspace || p.workspace_bytes < plan.splits * elems * 4 || !aligned_to(p.workspace, 16))
            return fail(TH_ERR_WORKSPACE, "%s: scratch missing, too small or off 16 bytes", what);
        g.out = p.workspace;
        g.out_stride = p.b.rows;
        g.split_stride = elems * 4;
        g.out_dtype = kRaw32;
    }
    int rc = TH_ERR_UNSUPPORTED;
    if constexpr (EB == 1) {
        if (plan.swap) {
            switch (plan.bn) {
                case 16: rc = launch_gemm<1, false, false, 16, 1, true>(g, p.b, p.a, p.k, false, stream); break;
                case 32: rc = launch_gemm<1, false, false, 32, 1, true>(g, p.b, p.a, p.k, false, stream); break;
                case 64: rc = launch_gemm<1, false, false, 64, 1, true>(g, p.b, p.a, p.k, false, stream); break;
                default: rc = launch_gemm<1, false, false, 128, 1, true>(g, p.b, p.a, p.k, false, stream); break;
            }
        }
    }
    if (!plan.swap) {
        rc = plan.cg == 2 ? launch_gemm<EB, A_MN, B_MN, 256, 2, false>(g, p.a, p.b, p.k, bf16, stream)
                          : launch_gemm<EB, A_MN, B_MN, 128, 1, false>(g, p.a, p.b, p.k, bf16, stream);
    }
    if (rc != TH_OK || plan.splits == 1) return rc;
    SplitArgs s{};
    s.partial = static_cast<const uint32_t *>(p.workspace);
    s.splits = plan.splits;
    s.rows = p.a.rows;
    s.n = p.b.rows;
    s.split_elems = s.rows * s.n;
    s.row_scale = p.row_scale;
    s.column_scale = p.column_scale;
    s.bias = p.bias;
    s.bias_dtype = p.bias_dtype;
    s.out = p.out;
    s.out_stride = p.out_stride;
    s.out_dtype = p.out_dtype;
    const unsigned gy = static_cast<unsigned>(std::min<long long>(s.rows, 32768));
    const dim3 grid(divide_up(s.n, 256), gy, divide_up(s.rows, gy));
    split_sum_kernel<EB == 1><<<grid, 256, 0, stream>>>(s);
    return launch_status("split_sum_kernel");
}

int check_shape(const char *what, int64_t rows, int d_in, int d_out) {
    if (rows < 0 || d_in < 1 || d_out < 1) return fail(TH_ERR_BAD_ARG, "%s: %lld rows, %d -> %d", what, static_cast<long long>(rows), d_in, d_out);
    if (rows > (1ll << 30) || d_in > (1 << 24) || d_out > (1 << 24))
        return fail(TH_ERR_UNSUPPORTED, "%s: %lld rows, %d -> %d", what, static_cast<long long>(rows), d_in, d_out);
    return TH_OK;
}

int check_16bit(const char *what, int dtype) {
    return dtype == TH_F16 || dtype == TH_BF16 ? TH_OK : fail(TH_ERR_UNSUPPORTED, "%s: float16 or bfloat16, not dtype code %d", what, dtype);
}

}  // namespace
}  // namespace th

using namespace th;

extern "C" int th_linear_tc_status(void) {
    int status = 0;
    if (cudaMemcpyFromSymbol(&status, g_tc_status, sizeof(int)) != cudaSuccess) return -1;
    return status;
}

extern "C" int64_t th_int8_linear_workspace_bytes(int64_t rows, int d_in, int d_out) { return product_workspace(rows, d_out, d_in, 1); }

extern "C" int th_int8_linear(const void *q_dev, int64_t q_stride, const float *scale_dev, const void *weight_dev, int64_t weight_stride,
                              const float *weight_scale_dev, const void *bias_dev, void *y_dev, int64_t y_stride, void *workspace_dev, int64_t workspace_bytes,
                              int64_t rows, int d_in, int d_out, int dtype, void *stream) {
    if (int rc = check_shape("th_int8_linear", rows, d_in, d_out)) return rc;
    // 128 x 128 x 131071 is the largest sum that 32 bits are sure to hold
    if (d_in > 131071) return fail(TH_ERR_UNSUPPORTED, "th_int8_linear: %d inputs, more than a 32-bit sum holds", d_in);
    if (dtype != TH_F32 && dtype != TH_F16 && dtype != TH_BF16) return fail(TH_ERR_UNSUPPORTED, "th_int8_linear: unknown dtype code %d", dtype);
    if (rows == 0) return TH_OK;
    if (!q_dev || !scale_dev || !weight_dev || !weight_scale_dev || !y_dev) return fail(TH_ERR_BAD_ARG, "th_int8_linear: null pointer");
    if (!aligned_to(q_dev, 16) || q_stride % 16 || q_stride < d_in || !aligned_to(weight_dev, 16) || weight_stride % 16 || weight_stride < d_in)
        return fail(TH_ERR_ALIGNMENT, "th_int8_linear: 8-bit rows start on 16 bytes");
    Product p{};
    p.a = {q_dev, q_stride, static_cast<int>(rows)};
    p.b = {weight_dev, weight_stride, d_out};
    p.k = d_in;
    p.row_scale = scale_dev;
    p.column_scale = weight_scale_dev;
    p.bias = bias_dev;
    p.out = y_dev;
    p.out_stride = y_stride;
    p.out_dtype = p.bias_dtype = dtype;
    p.workspace = workspace_dev;
    p.workspace_bytes = workspace_bytes;
    return run_product<1, false, false>("th_int8_linear", p, false, static_cast<cudaStream_t>(stream));
}

extern "C" int64_t th_linear_workspace_bytes(int64_t rows, int d_in, int d_out) {
    if (rows < 1 || rows > (1ll << 30)) return 0;
    return std::max({product_workspace(rows, d_out, d_in, 2), product_workspace(rows, d_in, d_out, 2), product_workspace(d_out, d_in, static_cast<int>(rows), 2)});
}

extern "C" int th_linear_fwd(const void *x_dev, int64_t x_stride, const void *weight_dev, int64_t weight_stride, const void *bias_dev, void *y_dev,
                             int64_t y_stride, void *workspace_dev, int64_t workspace_bytes, int64_t rows, int d_in, int d_out, int dtype, void *stream) {
    if (int rc = check_shape("th_linear_fwd", rows, d_in, d_out)) return rc;
    if (int rc = check_16bit("th_linear_fwd", dtype)) return rc;
    if (rows == 0) return TH_OK;
    if (!x_dev || !weight_dev || !y_dev || x_stride < d_in || weight_stride < d_in || y_stride < d_out)
        return fail(TH_ERR_BAD_ARG, "th_linear_fwd: null pointer or short stride");
    Product p{};
    p.a = {x_dev, x_stride, static_cast<int>(rows)};
    p.b = {weight_dev, weight_stride, d_out};
    p.k = d_in;
    p.bias = bias_dev;
    p.out = y_dev;
    p.out_stride = y_stride;
    p.out_dtype = p.bias_dtype = dtype;
    p.workspace = workspace_dev;
    p.workspace_bytes = workspace_bytes;
    return run_product<2, false, false>("th_linear_fwd", p, dtype == TH_BF16, static_cast<cudaStream_t>(stream));
}

extern "C" int th_linear_bwd_input(const void *grad_y_dev, int64_t gy_stride, const void *weight_dev, int64_t weight_stride, void *grad_x_dev,
                                   int64_t gx_stride, void *workspace_dev, int64_t workspace_bytes, int64_t rows, int d_in, int d_out, int dtype,
                                   void *stream) {
    if (int rc = check_shape("th_linear_bwd_input", rows, d_in, d_out)) return rc;
    if (int rc = check_16bit("th_linear_bwd_input", dtype)) return rc;
    if (rows == 0) return TH_OK;
    if (!grad_y_dev || !weight_dev || !grad_x_dev || gy_stride < d_out || weight_stride < d_in || gx_stride < d_in)
        return fail(TH_ERR_BAD_ARG, "th_linear_bwd_input: null pointer or short stride");
    Product p{};
    p.a = {grad_y_dev, gy_stride, static_cast<int>(rows)};
    p.b = {weight_dev, weight_stride, d_in};
    p.k = d_out;
    p.out = grad_x_dev;
    p.out_stride = gx_stride;
    p.out_dtype = dtype;
    p.workspace = workspace_dev;
    p.workspace_bytes = workspace_bytes;
    return run_product<2, false, true>("th_linear_bwd_input", p, dtype == TH_BF16, static_cast<cudaStream_t>(stream));
}

extern "C" int th_linear_bwd_weight(const void *grad_y_dev, int64_t gy_stride, const void *x_dev, int64_t x_stride, void *grad_weight_dev,
                                    void *workspace_dev, int64_t workspace_bytes, int64_t rows, int d_in, int d_out, int dtype, void *stream) {
    if (int rc = check_shape("th_linear_bwd_weight", rows, d_in, d_out)) return rc;
    if (int rc = check_16bit("th_linear_bwd_weight", dtype)) return rc;
    if (!grad_weight_dev) return fail(TH_ERR_BAD_ARG, "th_linear_bwd_weight: null pointer");
    cudaStream_t at = static_cast<cudaStream_t>(stream);
    if (rows == 0) return cuda_status(cudaMemsetAsync(grad_weight_dev, 0, static_cast<size_t>(d_in) * d_out * 2, at), "th_linear_bwd_weight");
    if (!grad_y_dev || !x_dev || gy_stride < d_out || x_stride < d_in) return fail(TH_ERR_BAD_ARG, "th_linear_bwd_weight: null pointer or short stride");
    Product p{};
    p.a = {grad_y_dev, gy_stride, d_out};
    p.b = {x_dev, x_stride, d_in};
    p.k = static_cast<int>(rows);
    p.out = grad_weight_dev;
    p.out_stride = d_in;
    p.out_dtype = dtype;
    p.workspace = workspace_dev;
    p.workspace_bytes = workspace_bytes;
    return run_product<2, true, true>("th_linear_bwd_weight", p, dtype == TH_BF16, at);
}
