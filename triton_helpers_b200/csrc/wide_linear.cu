// Linear layers of any width: 8-bit integers with a scale per token and per channel, and 16-bit products in the three forms that a
// layer's forward and backward pass take.  The products are wide_gemm_kernel's; what is here chooses how they are cut.
#include "wide_gemm.cuh"

namespace th {
namespace {

// How a product is cut: tile width, CTAs per tile, transposed or not, and the parts that K is split into (within a cluster).
struct ProductPlan {
    int bn, cg;
    bool swap;
    int splits;
};

// The cheapest cut by an estimate in cycles: rounds of tiles x stages x cycles a stage (what its bytes take into the SM), what a pair
// takes longer to start, and for split tiles the exchange of their sums.  All cuts measured on a B200, us (tile columns x CTAs x parts;
// * is the one taken): 2048 x 2048 -> 2048 256x2x1* 17.9, 128x2x1 21, 128x1x1 26; 512 x 4096 -> 4096 128x2x1* 20.3, 256x2x2 21.9, 128x1x1
// 25.5; gradient of 777 x 1000 weights from 3001 rows 128x2x2* 15.3, 128x1x2 16.5, 128x2x1 19.3, 256x2x1 24.6; of 512 x 512 weights from
// 16384 rows 128x2x4* 22, 128x1x4 26, 256x2x1 79; 300 x 256 -> 512 128x1x1* 5.7, 128x2x1 6.8, 256x2x1 8.2.
ProductPlan plan_product(int m, int n, int k, int elem_bytes) {
    const int k_tiles = divide_up(k, 128 / elem_bytes);
    ProductPlan best{};
    double least = 0;
    const auto consider = [&](int bn, int cg, bool swap, int per_sm, double stage, double exchange) {
        const long long tiles = swap ? static_cast<long long>(divide_up(n, kGemmRows)) * divide_up(m, bn)
                                     : static_cast<long long>(divide_up(m, cg * kGemmRows)) * divide_up(n, bn);
        for (int s = 1; s * cg <= 8 && s <= k_tiles; ++s) {
            const int per = divide_up(k_tiles, s);
            if (divide_up(k_tiles, per) != s) continue;
            const int slots = cluster_slots(s * cg, per_sm);
            if (s > 1 && tiles > slots) break;
            // CTAs that share an SM share its way in
            const double rounds = per_sm == 1 ? divide_up(tiles, slots) : static_cast<double>(divide_up(tiles * s, sm_count()));
            const double cost = rounds * per * stage + (cg == 2 ? 1800 : 0) + (s > 1 ? exchange : 0);
            if (best.bn == 0 || cost < least) {
                best = {bn, cg, swap, s};
                least = cost;
            }
        }
    };
    if (elem_bytes == 1 && m <= 128) {  // tokens along the accumulator's columns: tiles no wider than they are
        const int bn = m <= 16 ? 16 : m <= 32 ? 32 : m <= 64 ? 64 : 128;
        consider(bn, 1, true, 2, 2.0 * (kGemmRows + bn), 1500 + 8 * bn);
        return best;
    }
    consider(256, 2, false, 1, 540, 9000);
    consider(128, 2, false, 1, 410, 4500);
    consider(128, 1, false, 1, 540, 4500);
    return best;
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
    int weights_settled;  // b was complete before the kernel ahead of this one began
};

template <int EB, bool A_MN, bool B_MN>
int run_product(const Product &p, bool bf16, cudaStream_t stream) {
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
    g.early = p.weights_settled;
    if constexpr (EB == 1) {
        if (plan.swap) {
            switch (plan.bn) {
                case 16: return launch_gemm<1, false, false, 16, 1, true, 2>(g, p.b, p.a, p.k, false, stream);
                case 32: return launch_gemm<1, false, false, 32, 1, true, 2>(g, p.b, p.a, p.k, false, stream);
                case 64: return launch_gemm<1, false, false, 64, 1, true, 2>(g, p.b, p.a, p.k, false, stream);
                default: return launch_gemm<1, false, false, 128, 1, true, 2>(g, p.b, p.a, p.k, false, stream);
            }
        }
    }
    if (plan.cg == 1) return launch_gemm<EB, A_MN, B_MN, 128, 1, false, 1>(g, p.a, p.b, p.k, bf16, stream);
    return plan.bn == 256 ? launch_gemm<EB, A_MN, B_MN, 256, 2, false, 1>(g, p.a, p.b, p.k, bf16, stream)
                          : launch_gemm<EB, A_MN, B_MN, 128, 2, false, 1>(g, p.a, p.b, p.k, bf16, stream);
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

bool known_dtype(int dtype) { return dtype == TH_F32 || dtype == TH_F16 || dtype == TH_BF16; }

int check_int8(const void *weight, int64_t weight_stride, const float *weight_scale, const void *bias, const void *y, int64_t y_stride, int d_in, int d_out, int dtype) {
    // 128 x 128 x 131071 is the largest sum that 32 bits are sure to hold
    if (d_in > 131071) return fail(TH_ERR_UNSUPPORTED, "th_int8_linear: %d inputs, more than a 32-bit sum holds", d_in);
    if (!known_dtype(dtype)) return fail(TH_ERR_UNSUPPORTED, "th_int8_linear: unknown dtype code %d", dtype);
    if (!weight || !weight_scale || !y || y_stride < d_out) return fail(TH_ERR_BAD_ARG, "th_int8_linear: null pointer or short stride");
    if (!aligned_to(weight, 16) || weight_stride % 16 || weight_stride < d_in) return fail(TH_ERR_ALIGNMENT, "th_int8_linear: 8-bit rows start on 16 bytes");
    if (int rc = check_elements("th_int8_linear", TH_F32, {weight_scale})) return rc;
    return check_elements("th_int8_linear", dtype, {bias, y});
}

}  // namespace
}  // namespace th

namespace th {
int rows_status_word();  // rows.cu
int float8_status_word();  // float8_linear.cu
int expert_status_word();  // expert_linear.cu
}

using namespace th;

extern "C" int th_linear_tc_status(void) {
    int status = 0;
    if (cudaMemcpyFromSymbol(&status, g_tc_status, sizeof(int)) != cudaSuccess) return -1;
    const int rows = rows_status_word(), blocks = float8_status_word(), experts = expert_status_word();
    return rows < 0 || blocks < 0 || experts < 0 ? -1 : status | rows | blocks | experts;
}

static int int8_linear(const void *q_dev, int64_t q_stride, const float *scale_dev, const void *weight_dev, int64_t weight_stride, const float *weight_scale_dev,
                       const void *bias_dev, void *y_dev, int64_t y_stride, int64_t rows, int d_in, int d_out, int dtype, int weights_settled, void *stream) {
    if (int rc = check_shape("th_int8_linear", rows, d_in, d_out)) return rc;
    if (rows == 0 && d_in <= 131071 && known_dtype(dtype)) return TH_OK;
    if (int rc = check_int8(weight_dev, weight_stride, weight_scale_dev, bias_dev, y_dev, y_stride, d_in, d_out, dtype)) return rc;
    if (!q_dev || !scale_dev) return fail(TH_ERR_BAD_ARG, "th_int8_linear: null pointer");
    if (!aligned_to(q_dev, 16) || q_stride % 16 || q_stride < d_in) return fail(TH_ERR_ALIGNMENT, "th_int8_linear: 8-bit rows start on 16 bytes");
    if (int rc = check_elements("th_int8_linear", TH_F32, {scale_dev})) return rc;
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
    p.weights_settled = weights_settled;
    return run_product<1, false, false>(p, false, static_cast<cudaStream_t>(stream));
}

extern "C" int th_int8_linear(const void *q_dev, int64_t q_stride, const float *scale_dev, const void *weight_dev, int64_t weight_stride,
                              const float *weight_scale_dev, const void *bias_dev, void *y_dev, int64_t y_stride, int64_t rows, int d_in, int d_out,
                              int dtype, void *stream) {
    return int8_linear(q_dev, q_stride, scale_dev, weight_dev, weight_stride, weight_scale_dev, bias_dev, y_dev, y_stride, rows, d_in, d_out, dtype, 0, stream);
}

extern "C" int64_t th_quantized_linear_workspace_bytes(int64_t rows, int d_in) {
    return rows < 1 || d_in < 1 ? 0 : rows * ((d_in + 15) / 16 * 16 + 4ll) + 16;
}

// The quantising kernel lets the product start only once everything ahead of itself has finished, the weights included, so the product may
// fetch its first weights while the rows are being quantised (one token, 8192 -> 8192, weights from memory: 17.0 -> 16.7 us captured).
extern "C" int th_quantized_linear(const void *x_dev, int64_t x_stride, int x_dtype, const void *weight_dev, int64_t weight_stride, const float *weight_scale_dev,
                                   const void *bias_dev, void *y_dev, int64_t y_stride, void *workspace_dev, int64_t workspace_bytes, int64_t rows, int d_in,
                                   int d_out, int dtype, void *stream) {
    if (rows > 0 && (!workspace_dev || workspace_bytes < th_quantized_linear_workspace_bytes(rows, d_in) || !aligned_to(workspace_dev, 16)))
        return fail(TH_ERR_WORKSPACE, "th_quantized_linear: scratch missing, too small or off 16 bytes");
    const int64_t pitch = (d_in + 15) / 16 * 16;
    char *q = static_cast<char *>(workspace_dev);
    float *scale = reinterpret_cast<float *>(q + rows * pitch);
    // the product's refusals first: nothing is launched for a call that it does not take
    if (int rc = check_shape("th_quantized_linear", rows, d_in, d_out)) return rc;
    if (rows == 0) return int8_linear(q, pitch, scale, weight_dev, weight_stride, weight_scale_dev, bias_dev, y_dev, y_stride, 0, d_in, d_out, dtype, 0, stream);
    if (int rc = check_int8(weight_dev, weight_stride, weight_scale_dev, bias_dev, y_dev, y_stride, d_in, d_out, dtype)) return rc;
    if (int rc = th_quantize_rows(x_dev, x_stride, q, pitch, scale, rows, d_in, x_dtype, stream)) return rc;
    return int8_linear(q, pitch, scale, weight_dev, weight_stride, weight_scale_dev, bias_dev, y_dev, y_stride, rows, d_in, d_out, dtype, 1, stream);
}

extern "C" int th_linear_fwd(const void *x_dev, int64_t x_stride, const void *weight_dev, int64_t weight_stride, const void *bias_dev, void *y_dev,
                             int64_t y_stride, int64_t rows, int d_in, int d_out, int dtype, void *stream) {
    if (int rc = check_shape("th_linear_fwd", rows, d_in, d_out)) return rc;
    if (int rc = check_16bit("th_linear_fwd", dtype)) return rc;
    if (rows == 0) return TH_OK;
    if (!x_dev || !weight_dev || !y_dev || x_stride < d_in || weight_stride < d_in || y_stride < d_out)
        return fail(TH_ERR_BAD_ARG, "th_linear_fwd: null pointer or short stride");
    if (int rc = check_elements("th_linear_fwd", dtype, {bias_dev, y_dev})) return rc;
    Product p{};
    p.a = {x_dev, x_stride, static_cast<int>(rows)};
    p.b = {weight_dev, weight_stride, d_out};
    p.k = d_in;
    p.bias = bias_dev;
    p.out = y_dev;
    p.out_stride = y_stride;
    p.out_dtype = p.bias_dtype = dtype;
    return run_product<2, false, false>(p, dtype == TH_BF16, static_cast<cudaStream_t>(stream));
}

extern "C" int th_linear_bwd_input(const void *grad_y_dev, int64_t gy_stride, const void *weight_dev, int64_t weight_stride, void *grad_x_dev,
                                   int64_t gx_stride, int64_t rows, int d_in, int d_out, int dtype, void *stream) {
    if (int rc = check_shape("th_linear_bwd_input", rows, d_in, d_out)) return rc;
    if (int rc = check_16bit("th_linear_bwd_input", dtype)) return rc;
    if (rows == 0) return TH_OK;
    if (!grad_y_dev || !weight_dev || !grad_x_dev || gy_stride < d_out || weight_stride < d_in || gx_stride < d_in)
        return fail(TH_ERR_BAD_ARG, "th_linear_bwd_input: null pointer or short stride");
    if (int rc = check_elements("th_linear_bwd_input", dtype, {grad_x_dev})) return rc;
    Product p{};
    p.a = {grad_y_dev, gy_stride, static_cast<int>(rows)};
    p.b = {weight_dev, weight_stride, d_in};
    p.k = d_out;
    p.out = grad_x_dev;
    p.out_stride = gx_stride;
    p.out_dtype = dtype;
    return run_product<2, false, true>(p, dtype == TH_BF16, static_cast<cudaStream_t>(stream));
}

extern "C" int th_linear_bwd_weight(const void *grad_y_dev, int64_t gy_stride, const void *x_dev, int64_t x_stride, void *grad_weight_dev,
                                    int64_t rows, int d_in, int d_out, int dtype, void *stream) {
    if (int rc = check_shape("th_linear_bwd_weight", rows, d_in, d_out)) return rc;
    if (int rc = check_16bit("th_linear_bwd_weight", dtype)) return rc;
    if (!grad_weight_dev) return fail(TH_ERR_BAD_ARG, "th_linear_bwd_weight: null pointer");
    cudaStream_t at = static_cast<cudaStream_t>(stream);
    if (rows == 0) return cuda_status(cudaMemsetAsync(grad_weight_dev, 0, static_cast<size_t>(d_in) * d_out * 2, at), "th_linear_bwd_weight");
    if (!grad_y_dev || !x_dev || gy_stride < d_out || x_stride < d_in) return fail(TH_ERR_BAD_ARG, "th_linear_bwd_weight: null pointer or short stride");
    if (int rc = check_elements("th_linear_bwd_weight", dtype, {grad_weight_dev})) return rc;
    Product p{};
    p.a = {grad_y_dev, gy_stride, d_out};
    p.b = {x_dev, x_stride, d_in};
    p.k = static_cast<int>(rows);
    p.out = grad_weight_dev;
    p.out_stride = d_in;
    p.out_dtype = dtype;
    return run_product<2, true, true>(p, dtype == TH_BF16, at);
}
