r"""Layers for wide networks where a definition has to hold at its edges: roundings, layouts, scales, threads, modes."""
import pytest
import torch

from triton_helpers_b200.layers.checkpointed_linear import checkpointed_linear
from triton_helpers_b200.layers.int8_linear import Int8Rows, dequantize_rows, int8_linear, quantize_rows

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


@pytest.mark.parametrize("lead", [(4, 3), (3, 4), (2, 4, 3), (4, 2, 3), (4, 1, 3)])
def test_expanded_8_bit_rows(lead):
    # rows that share memory along any leading dimension: what they hold is what counts, and nothing past them is read
    rows, weight = quantize_rows(normal(4, 40)), quantize_rows(normal(24, 40, seed=1))
    shape = [4 if n == 4 else 1 for n in lead]
    q, scale = rows.q.view(*shape, 40).expand(*lead, 40), rows.scale.view(shape).expand(lead).contiguous()
    want = int8_linear(Int8Rows(q.contiguous(), scale), weight, dtype=torch.float32)
    assert torch.equal(int8_linear(Int8Rows(q, scale), weight, dtype=torch.float32), want)
    assert torch.equal(want, int8_linear(rows, weight, dtype=torch.float32).view(*shape, 24).expand(*lead, 24))
    assert torch.equal(dequantize_rows(Int8Rows(q, scale)), q.float() * scale[..., None])


def test_expanded_8_bit_weights():
    rows, one = quantize_rows(normal(5, 48)), quantize_rows(normal(1, 48, seed=1))
    weight = Int8Rows(one.q.expand(7, 48), one.scale.expand(7).contiguous())
    assert torch.equal(int8_linear(rows, weight, dtype=torch.float32), int8_linear(rows, one, dtype=torch.float32).expand(5, 7))
