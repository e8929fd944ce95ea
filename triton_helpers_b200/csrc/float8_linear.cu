// Linear layers on 8-bit floating-point blocks: the products are float8_gemm_kernel's; what is here chooses how they are cut.
#include "float8_gemm.cuh"

namespace th {
namespace {

struct F8Plan {
    int bn, cg;
    bool swap;
    int splits;
};

// The cheapest cut by an estimate in cycles, as for the products without scales (wide_linear.cu): rounds of tiles x blocks of K x cycles a
// block, what a pair takes longer to start, and for split tiles the exchange of their sums.  Cuts measured on a B200, us (tile columns x CTAs x parts; * is
// the one taken): 8192 x 4096 -> 4096 256x2x1* 142, 128x2x1 180, 128x1x1 181; 2048 x 2048 -> 2048 256x2x1* 17.2, 128x1x1 20.3, 128x2x1 20.9; 512 x 4096 -> 4096
// 128x1x1* 18.4, 128x2x1 19.8, 256x2x2 22.2; 256 x 8192 -> 1024 128x1x5* 13.9, 128x1x4 14.5, 128x2x4 16.1, 256x2x1 36.9; 1023 x 2500 -> 1111 128x1x2* 14.7,
// 128x2x1 15.5, 256x2x1 18.8; one token 4096 -> 4096 in 1, 2, 3, 4*, 8 parts 14.6, 11.9, 10.2, 9.7, 9.9; 100 tokens in 1, 2, 4*, 8 parts 29, 20.5, 16.6, 35.
F8Plan plan_float8(int m, int n, int k, bool b_mn) {
    const int k_tiles = divide_up(k, kF8Block);
    F8Plan best{};
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
    if (!b_mn && m <= 128) {  // tokens along the accumulator's columns: tiles no wider than they are
        const int bn = m <= 16 ? 16 : m <= 32 ? 32 : m <= 64 ? 64 : 128;
        consider(bn, 1, true, bn == 128 ? 1 : 2, 2.0 * (kGemmRows + bn), 1500 + 8 * bn);
        return best;
    }
    consider(256, 2, false, 1, 960, 9000);
    if (!b_mn) consider(128, 2, false, 1, 720, 4500);  // an MN-major weight comes 128 columns a CTA
    consider(128, 1, false, 1, 680, 4500);
    return best;
}

template <bool B_MN>
int run_float8(const F8Product &p, cudaStream_t stream) {
    const F8Plan plan = plan_float8(p.tokens.rows, p.weight.rows, p.k, B_MN);
    if constexpr (!B_MN) {
        if (plan.swap) {
            switch (plan.bn) {
                case 16: return launch_float8<false, 16, 1, true, 2>(p, plan.splits, stream);
                case 32: return launch_float8<false, 32, 1, true, 2>(p, plan.splits, stream);
                case 64: return launch_float8<false, 64, 1, true, 2>(p, plan.splits, stream);
                default: return launch_float8<false, 128, 1, true, 1>(p, plan.splits, stream);
            }
        }
        if (plan.cg == 2 && plan.bn == 128) return launch_float8<false, 128, 2, false, 1>(p, plan.splits, stream);
    }
    return plan.cg == 1 ? launch_float8<B_MN, 128, 1, false, 1>(p, plan.splits, stream) : launch_float8<B_MN, 256, 2, false, 1>(p, plan.splits, stream);
}

int check_f8_shape(const char *what, int64_t rows, int d_in, int d_out, int dtype) {
    if (rows < 0 || d_in < 1 || d_out < 1) return fail(TH_ERR_BAD_ARG, "%s: %lld rows, %d -> %d", what, static_cast<long long>(rows), d_in, d_out);
    if (rows > (1ll << 30) || d_in > (1 << 24) || d_out > (1 << 24))
        return fail(TH_ERR_UNSUPPORTED, "%s: %lld rows, %d -> %d", what, static_cast<long long>(rows), d_in, d_out);
    if (dtype != TH_F32 && dtype != TH_F16 && dtype != TH_BF16) return fail(TH_ERR_UNSUPPORTED, "%s: unknown dtype code %d", what, dtype);
    return TH_OK;
}

int check_f8_operand(const char *what, const Operand &o, const F8Scale &scale, int d) {
    if (!o.base || !scale.at || scale.row < 0 || scale.block < 0) return fail(TH_ERR_BAD_ARG, "%s: null pointer or negative stride of the scales", what);
    if (!aligned_to(o.base, 16) || o.stride % 16 || o.stride < d) return fail(TH_ERR_ALIGNMENT, "%s: 8-bit rows start on 16 bytes", what);
    return check_elements(what, TH_F32, {scale.at});
}

int check_f8_output(const char *what, const void *bias, const void *out, int64_t stride, int d, int dtype) {
    if (!out || stride < d) return fail(TH_ERR_BAD_ARG, "%s: null pointer or short stride", what);
    return check_elements(what, dtype, {bias, out});
}

}  // namespace
}  // namespace th

namespace th {
int float8_status_word() {
    int status = 0;
    return cudaMemcpyFromSymbol(&status, g_tc_status, sizeof(int)) == cudaSuccess ? status : -1;
}
}  // namespace th

using namespace th;

extern "C" int th_float8_linear(const void *q_dev, int64_t q_stride, const float *scale_dev, int64_t scale_row, int64_t scale_block, const void *weight_dev,
                                int64_t weight_stride, const float *weight_scale_dev, int64_t weight_scale_row, int64_t weight_scale_block,
                                const void *bias_dev, void *y_dev, int64_t y_stride, int64_t rows, int d_in, int d_out, int dtype, void *stream) {
    if (int rc = check_f8_shape("th_float8_linear", rows, d_in, d_out, dtype)) return rc;
    if (rows == 0) return TH_OK;
    const F8Product p{{q_dev, q_stride, static_cast<int>(rows)}, {weight_dev, weight_stride, d_out}, {scale_dev, scale_row, scale_block},
                      {weight_scale_dev, weight_scale_row, weight_scale_block}, d_in, bias_dev, y_dev, y_stride, dtype, 0};
    if (int rc = check_f8_operand("th_float8_linear", p.tokens, p.token_scale, d_in)) return rc;
    if (int rc = check_f8_operand("th_float8_linear", p.weight, p.weight_scale, d_in)) return rc;
    if (int rc = check_f8_output("th_float8_linear", bias_dev, y_dev, y_stride, d_out, dtype)) return rc;
    return run_float8<false>(p, static_cast<cudaStream_t>(stream));
}

// Scratch: the rows' 8-bit values, then their scales, a column block after the other
static int64_t pitch_of(int d) { return (static_cast<int64_t>(d) + 15) / 16 * 16; }

extern "C" int64_t th_float8_quantized_linear_workspace_bytes(int64_t rows, int d_in) {
    return rows < 1 || d_in < 1 ? 0 : rows * (pitch_of(d_in) + 4ll * ((d_in + kF8Block - 1) / kF8Block)) + 16;
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
    const F8Product p{{q, pitch_of(d_in), static_cast<int>(rows)}, {weight_dev, weight_stride, d_out}, {scale, 1, rows},
                      {weight_scale_dev, weight_scale_row, weight_scale_block}, d_in, bias_dev, y_dev, y_stride, dtype, 1};
    // the product's refusals first: nothing is launched for a call that it does not take
    if (int rc = check_f8_operand("th_float8_quantized_linear", p.weight, p.weight_scale, d_in)) return rc;
    if (int rc = check_f8_output("th_float8_quantized_linear", bias_dev, y_dev, y_stride, d_out, dtype)) return rc;
    if (int rc = th_float8_rows(x_dev, x_stride, q, pitch_of(d_in), scale, rows, rows, d_in, x_dtype, stream)) return rc;
    return run_float8<false>(p, static_cast<cudaStream_t>(stream));
}

extern "C" int th_float8_bwd_input(const void *grad_q_dev, int64_t grad_q_stride, const float *grad_scale_dev, int64_t grad_scale_row,
                                   int64_t grad_scale_block, const void *weight_dev, int64_t weight_stride, const float *weight_scale_dev,
                                   int64_t weight_scale_row, int64_t weight_scale_block, void *grad_x_dev, int64_t gx_stride, int64_t rows, int d_in,
                                   int d_out, int dtype, void *stream) {
    if (int rc = check_f8_shape("th_float8_bwd_input", rows, d_in, d_out, dtype)) return rc;
    if (rows == 0) return TH_OK;
    const F8Product p{{grad_q_dev, grad_q_stride, static_cast<int>(rows)}, {weight_dev, weight_stride, d_in}, {grad_scale_dev, grad_scale_row, grad_scale_block},
                      {weight_scale_dev, weight_scale_row, weight_scale_block}, d_out, nullptr, grad_x_dev, gx_stride, dtype, 0};
    if (int rc = check_f8_operand("th_float8_bwd_input", p.tokens, p.token_scale, d_out)) return rc;
    if (int rc = check_f8_operand("th_float8_bwd_input", p.weight, p.weight_scale, d_in)) return rc;
    if (int rc = check_f8_output("th_float8_bwd_input", nullptr, grad_x_dev, gx_stride, d_in, dtype)) return rc;
    return run_float8<true>(p, static_cast<cudaStream_t>(stream));
}
