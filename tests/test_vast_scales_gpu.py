r"""8-bit floating-point products with scales at the end of float32's range: a block whose products sum to zero adds nothing, whatever its scales."""
import pytest
import torch

from triton_helpers_b200 import _lib
from triton_helpers_b200.layers.float8_linear import Float8Blocks, float8_linear

pytestmark = pytest.mark.gpu

MOST = torch.finfo(torch.float32).max
PAIRS = [(MOST, MOST), (-MOST, MOST), (2.0**127, -(2.0**127)), (MOST, 2.0**126), (1.9 * 2.0**126, MOST)]


def e4m3(*shape, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-4, 5, shape, device="cuda", generator=g).to(torch.float8_e4m3fn)


def operands(rows, n, blocks):
    r"""Tokens and a weight of small whole numbers, scales of one."""
    k = 128 * blocks
    x = Float8Blocks(e4m3(rows, k), torch.ones(rows, blocks, device="cuda"))
    return x, Float8Blocks(e4m3(n, k, seed=1), torch.ones(-(-n // 128), blocks, device="cuda"))


# few tokens along the accumulator's columns, single CTAs, K in parts, pairs of CTAs
@pytest.mark.parametrize("rows,n,blocks", [(1, 200, 2), (20, 130, 3), (100, 300, 8), (150, 200, 2), (300, 256, 40), (2100, 2304, 3)])
@pytest.mark.parametrize("pair", PAIRS)
def test_float8_blocks_without_products(pair, rows, n, blocks):
    x, w = operands(rows, n, blocks)
    want = x.q[:, 128:].double() @ w.q[:, 128:].double().t()  # whole numbers below 2^24: exact
    bias = torch.arange(n, device="cuda").float()
    # the first block: nothing but zeros in the tokens' odd rows, products that cancel in the even ones
    first = torch.zeros(rows, 128, device="cuda")
    first[::2, 3], first[::2, 90] = 2.0, -2.0
    x.q[:, :128] = first.to(torch.float8_e4m3fn)
    w.q[:, 90] = w.q[:, 3]
    x.scale[:, 0], w.scale[:, 0] = pair
    got = float8_linear(x, w, bias, torch.float32)
    assert torch.equal(got.double(), want + bias.double()) and _lib.lib().th_linear_tc_status() == 0


@pytest.mark.parametrize("rows,n", [(3, 40), (150, 200), (2100, 2304)])
def test_float8_products_beyond_float32_are_infinite(rows, n):
    x, w = operands(rows, n, 2)
    x.scale[:, 0], w.scale[:, 0] = MOST, -MOST
    far = x.q[:, :128].double() @ w.q[:, :128].double().t()
    near = x.q[:, 128:].double() @ w.q[:, 128:].double().t()
    got = float8_linear(x, w, dtype=torch.float32)
    assert torch.equal(got.double(), torch.where(far == 0, near, far * float("-inf"))) and bool((far == 0).any())


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("other", [MOST, 1.0, 0.0, 2.0**-149])
def test_float8_scales_that_are_not_finite_stay_so(bad, other):
    # as the definition has it: a zero block times an infinite scale is a NaN, other products are infinite
    for rows, n in ((3, 40), (150, 200)):
        x, w = operands(rows, n, 2)
        x.q[::2, :128] = torch.zeros(128, device="cuda").to(torch.float8_e4m3fn)
        x.scale[:, 0], w.scale[:, 0] = bad, other
        blocks = [x.q[:, i : i + 128].double() @ w.q[:, i : i + 128].double().t() for i in (0, 128)]
        want = blocks[0] * (bad * other) + blocks[1]
        got = float8_linear(x, w, dtype=torch.float32)
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.double().nan_to_num(0, 1, -1), want.nan_to_num(0, 1, -1))
