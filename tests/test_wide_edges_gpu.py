r"""Layers for wide networks where a definition has to hold at its edges: roundings, layouts, scales, threads, modes."""
import pytest
import torch

from triton_helpers_b200.layers.checkpointed_linear import checkpointed_linear
from triton_helpers_b200.layers.int8_linear import dequantize_rows, quantize_rows

pytestmark = pytest.mark.gpu


def normal(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,d_in,d_out", [(300, 256, 512), (3001, 100, 77), (2048, 512, 640)])
def test_weight_gradient_is_that_of_the_rows_back_in_16_bits(rows, d_in, d_out, dtype):
    # the operand's one rounding to 16 bits is all that is lost: float32 sums of the rounded rows, and the result's half step
    x, w = normal(rows, d_in, dtype=dtype), normal(d_out, d_in, seed=1, dtype=dtype).requires_grad_(True)
    gy = normal(rows, d_out, seed=2, dtype=dtype)
    (got,) = torch.autograd.grad(checkpointed_linear(x, w), [w], gy)
    x16 = dequantize_rows(quantize_rows(x), dtype).double()
    want, reach = gy.double().t() @ x16, gy.double().abs().t() @ x16.abs()
    assert bool(((got.double() - want).abs() <= (rows + 2) * 2.0**-23 * reach + 1.01 * torch.finfo(dtype).eps / 2 * want.abs() + 2.0**-24).all())
