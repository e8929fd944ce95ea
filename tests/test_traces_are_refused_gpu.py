r"""Functions that launch kernels outside of an autograd node refuse torch.jit.trace: it would record the empty result alone."""
import pytest
import torch

from triton_helpers_b200.layers.float8_linear import Float8Blocks, dequantize_float8, float8_linear, quantize_float8_rows, quantize_float8_weight
from triton_helpers_b200.layers.int8_linear import Int8Rows, dequantize_rows, int8_linear, quantize_rows
from triton_helpers_b200.layers.rms_norm import rms_norm_int8
from triton_helpers_b200.optim import grad_norm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize(
    "name",
    ["float8_linear", "float8_linear of blocks", "quantize_float8_rows", "quantize_float8_weight", "dequantize_float8", "int8_linear", "int8_linear of rows",
     "quantize_rows", "dequantize_rows", "rms_norm_int8", "grad_norm"],
)  # fmt: skip
def test_a_trace_is_refused(name):
    g = torch.Generator(device="cuda").manual_seed(0)
    x, weight = (torch.randn(n, 256, device="cuda", generator=g).half() for n in (20, 72))
    w8, wi, gain = quantize_float8_weight(weight), quantize_rows(weight), torch.ones(256, device="cuda").half()
    x8, xi = quantize_float8_rows(x), quantize_rows(x)
    call, given = {
        "float8_linear": (lambda x: float8_linear(x, w8), x),
        "float8_linear of blocks": (lambda s: float8_linear(Float8Blocks(x8.q, s), w8, dtype=torch.float16), x8.scale),
        "quantize_float8_rows": (lambda x: quantize_float8_rows(x).scale, x),
        "quantize_float8_weight": (lambda x: quantize_float8_weight(x).scale, x),
        "dequantize_float8": (lambda s: dequantize_float8(Float8Blocks(x8.q, s)), x8.scale),
        "int8_linear": (lambda x: int8_linear(x, wi), x),
        "int8_linear of rows": (lambda s: int8_linear(Int8Rows(xi.q, s), wi, dtype=torch.float16), xi.scale),
        "quantize_rows": (lambda x: quantize_rows(x).scale, x),
        "dequantize_rows": (lambda s: dequantize_rows(Int8Rows(xi.q, s)), xi.scale),
        "rms_norm_int8": (lambda x: rms_norm_int8(x, gain).scale, x),
        "grad_norm": (lambda x: grad_norm([x]), x),
    }[name]
    want = call(given)
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(call, given, check_trace=False)
    assert torch.equal(call(given), want)  # and the calls behind it are as before
