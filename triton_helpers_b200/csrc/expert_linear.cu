// Linear layers of several experts on rows sorted by expert: the products are expert_gemm_kernel's; what is here chooses their tiles.
// The ends are on the device, so that the choice goes by the average number of rows.
#include "expert_gemm.cuh"

#include <cmath>

namespace th {
namespace {

// Columns of the accumulator for few rows an expert; 0 where rows fill tiles of their own.  64 experts, 2048 -> 1024 (268 MB of weights), us with 16, 32 and 64
// columns and with 128-row tiles: 8 rows an expert 45.4, 46.0, 46.8, 50.3; 16 rows 48.0, 47.3, 48.0, 51.1; 32 rows 57.3, 49.8, 48.8, 51.6; 64 rows 80, 59.6, 52.8, 51.3.
int few_rows(int rows, int experts) {
    const int average = divide_up(rows, experts);
    return average > 48 ? 0 : average <= 8 ? 16 : average <= 20 ? 32 : 64;
}

// Whether pairs of CTAs on 256 x 256 tiles are quicker than single ones on 128 x 128, by an estimate in cycles: rounds of tiles x (stages x cycles a
// stage + what a tile takes besides).  Pairs against single ones, us: 16384 rows of 32 experts 2048 -> 4096 249 / 304, its weights' gradient 266 / 356; 128 rows
// for each of 64 experts 2048 -> 1024 63 / 67, 64 rows 59 / 51; 3001 rows of 7 experts 520 -> 336 10.2 / 8.8, the gradient 13.2 / 11.5.
bool pairs_pay(double tiles_256, double tiles_128, double stages) {
    const double rounds_256 = std::ceil(tiles_256 / (sm_count() / 2)), rounds_128 = std::ceil(tiles_128 / sm_count());
    return rounds_256 * (stages * 520 + 1500) + 1800 < rounds_128 * (stages * 560 + 800);
}

// Rows of an operand and one of the weight's two sides
template <bool B_MN>
int run_rows(ExpertArgs x, const ExpertOperand &rows, const ExpertOperand &weight, bool bf16, cudaStream_t stream) {
    switch (few_rows(x.rows, x.experts)) {
        case 16: return launch_experts<B_MN, false, 16, 1, true, false, 2>(x, weight, rows, bf16, stream);
        case 32: return launch_experts<B_MN, false, 32, 1, true, false, 2>(x, weight, rows, bf16, stream);
        case 64: return launch_experts<B_MN, false, 64, 1, true, false, 2>(x, weight, rows, bf16, stream);
        default: break;
    }
    // of an expert's tiles the last one is half empty on average; where its rows fit 128, a pair's tile would be so for sure
    const double average = static_cast<double>(x.rows) / x.experts, half = 0.5 * x.experts;
    if (average > 96 && pairs_pay((x.rows / 256.0 + half) * divide_up(x.g.n, 256), (x.rows / 128.0 + half) * divide_up(x.g.n, 128), divide_up(x.k, 64)))
        return launch_experts<false, B_MN, 256, 2, false, false, 1>(x, rows, weight, bf16, stream);
    return launch_experts<false, B_MN, 128, 1, false, false, 1>(x, rows, weight, bf16, stream);
}

int run_weights(ExpertArgs x, const ExpertOperand &a, const ExpertOperand &b, bool bf16, cudaStream_t stream) {
    const double e = x.experts;
    if (pairs_pay(e * divide_up(x.g.m, 256) * divide_up(x.g.n, 256), e * divide_up(x.g.m, 128) * divide_up(x.g.n, 128), divide_up(divide_up(x.rows, x.experts), 64)))
        return launch_experts<true, true, 256, 2, false, true, 1>(x, a, b, bf16, stream);
    return launch_experts<true, true, 128, 1, false, true, 1>(x, a, b, bf16, stream);
}

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

int check_weight(const char *what, const void *w, int64_t stride, int64_t expert_stride, int d_in, int d_out) {
    if (int rc = check_16(what, w, stride, d_in)) return rc;
    if (expert_stride < stride * (d_out - 1) + d_in) return fail(TH_ERR_BAD_ARG, "%s: experts overlap", what);
    return expert_stride % 8 ? fail(TH_ERR_ALIGNMENT, "%s: experts start on 16 bytes", what) : TH_OK;
}

}  // namespace
}  // namespace th

namespace th {
int expert_status_word() {
    int status = 0;
    return cudaMemcpyFromSymbol(&status, g_tc_status, sizeof(int)) == cudaSuccess ? status : -1;
}
}  // namespace th

using namespace th;

static ExpertArgs expert_args(const int32_t *ends, int64_t rows, int experts, int m, int n, int k, void *out, int64_t out_stride, int dtype) {
    ExpertArgs x{};
    x.ends = ends;
    x.experts = experts;
    x.rows = static_cast<int>(rows);
    x.k = k;
    x.g.m = m;
    x.g.n = n;
    x.g.out = out;
    x.g.out_stride = out_stride;
    x.g.out_dtype = dtype;
    return x;
}

extern "C" int th_expert_linear_fwd(const void *x_dev, int64_t x_stride, const void *weight_dev, int64_t weight_stride, int64_t expert_stride,
                                    const int32_t *ends_dev, void *y_dev, int64_t y_stride, int64_t rows, int experts, int d_in, int d_out, int dtype,
                                    void *stream) {
    if (int rc = check_experts("th_expert_linear_fwd", rows, experts, d_in, d_out, dtype, ends_dev)) return rc;
    if (rows == 0) return TH_OK;
    if (int rc = check_16("th_expert_linear_fwd", x_dev, x_stride, d_in)) return rc;
    if (int rc = check_weight("th_expert_linear_fwd", weight_dev, weight_stride, expert_stride, d_in, d_out)) return rc;
    if (!y_dev || y_stride < d_out) return fail(TH_ERR_BAD_ARG, "th_expert_linear_fwd: null pointer or short stride");
    if (int rc = check_elements("th_expert_linear_fwd", dtype, {y_dev})) return rc;
    return run_rows<false>(expert_args(ends_dev, rows, experts, static_cast<int>(rows), d_out, d_in, y_dev, y_stride, dtype), {x_dev, d_in, rows, x_stride, 1, 8},
                           {weight_dev, d_in, d_out, weight_stride, experts, expert_stride}, dtype == TH_BF16, static_cast<cudaStream_t>(stream));
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
    return run_rows<true>(expert_args(ends_dev, rows, experts, static_cast<int>(rows), d_in, d_out, grad_x_dev, gx_stride, dtype),
                          {grad_y_dev, d_out, rows, gy_stride, 1, 8}, {weight_dev, d_in, d_out, weight_stride, experts, expert_stride}, dtype == TH_BF16,
                          static_cast<cudaStream_t>(stream));
}

extern "C" int th_expert_linear_bwd_weight(const void *grad_y_dev, int64_t gy_stride, const void *x_dev, int64_t x_stride, const int32_t *ends_dev,
                                           void *grad_weight_dev, int64_t rows, int experts, int d_in, int d_out, int dtype, void *stream) {
    if (int rc = check_experts("th_expert_linear_bwd_weight", rows, experts, d_in, d_out, dtype, ends_dev)) return rc;
    // rows of all experts' gradients are counted in 32 bits, those behind the end of the last tile (256 rows at most) with them
    if (static_cast<int64_t>(experts) * d_out > 0x7fffffffll - 256) return fail(TH_ERR_UNSUPPORTED, "th_expert_linear_bwd_weight: %d experts, %d -> %d", experts, d_in, d_out);
    if (!grad_weight_dev) return fail(TH_ERR_BAD_ARG, "th_expert_linear_bwd_weight: null pointer");
    if (int rc = check_elements("th_expert_linear_bwd_weight", dtype, {grad_weight_dev})) return rc;
    cudaStream_t at = static_cast<cudaStream_t>(stream);
    if (rows == 0) return cuda_status(cudaMemsetAsync(grad_weight_dev, 0, static_cast<size_t>(experts) * d_in * d_out * 2, at), "th_expert_linear_bwd_weight");
    if (int rc = check_16("th_expert_linear_bwd_weight", grad_y_dev, gy_stride, d_out)) return rc;
    if (int rc = check_16("th_expert_linear_bwd_weight", x_dev, x_stride, d_in)) return rc;
    return run_weights(expert_args(ends_dev, rows, experts, d_out, d_in, 0, grad_weight_dev, d_in, dtype), {grad_y_dev, d_out, rows, gy_stride, 1, 8},
                       {x_dev, d_in, rows, x_stride, 1, 8}, dtype == TH_BF16, at);
}
