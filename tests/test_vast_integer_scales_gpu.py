r"""8-bit integer products with scales at the end of float32's range: a sum of zero stays zero, whatever its scales."""
import pytest
import torch

from triton_helpers_b200 import _lib
from triton_helpers_b200.layers.int8_linear import Int8Rows, int8_linear, quantize_rows

pytestmark = pytest.mark.gpu

MOST = torch.finfo(torch.float32).max
PAIRS = [(MOST, MOST), (-MOST, MOST), (2.0**127, -(2.0**127)), (MOST, 2.0**126), (1.9 * 2.0**126, MOST), (MOST, 2.0**-149), (2.0**-149, MOST)]


def rows_of(rows, k, scale, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return Int8Rows(torch.randint(-5, 6, (rows, k), device="cuda", generator=g).to(torch.int8), torch.full((rows,), scale, device="cuda"))


# few tokens along the accumulator's columns, K in parts, single CTAs, pairs of CTAs
@pytest.mark.parametrize("rows,n,k", [(1, 200, 256), (20, 130, 384), (100, 300, 2048), (150, 200, 256), (300, 256, 4096), (2100, 2304, 384)])
@pytest.mark.parametrize("pair", PAIRS)
def test_sums_of_zero(pair, rows, n, k):
    x, w = rows_of(rows, k, pair[0]), rows_of(n, k, pair[1], seed=1)
    # nothing but zeros in the tokens' odd rows, products that cancel in the even ones
    x.q.zero_()
    x.q[::2, 3], x.q[::2, 90] = 2, -2
    w.q[:, 90] = w.q[:, 3]
    bias = torch.arange(n, device="cuda").float()
    got = int8_linear(x, w, bias, torch.float32)
    assert torch.equal(got, bias.expand(rows, n)) and _lib.lib().th_linear_tc_status() == 0


@pytest.mark.parametrize("rows,n,k", [(3, 40, 256), (150, 200, 256), (300, 256, 4096), (2100, 2304, 384)])
@pytest.mark.parametrize("pair", PAIRS)
def test_other_sums(pair, rows, n, k):
    x, w = rows_of(rows, k, pair[0]), rows_of(n, k, pair[1], seed=1)
    sums = x.q.double() @ w.q.double().t()
    # the scales' product is a float32 where it is finite (a power of two times a scale): one rounding of it, one of the result
    want = sums * (pair[0] * pair[1])
    got = int8_linear(x, w, dtype=torch.float32).double()
    if abs(pair[0] * pair[1]) > MOST:
        assert torch.equal(got, torch.where(sums == 0, torch.zeros_like(sums), sums.sign() * float("inf") * (1 if pair[0] * pair[1] > 0 else -1)).nan_to_num(0, float("inf"), float("-inf")))
    else:
        assert float(((got - want).abs() - 2.0**-23 * 1.01 * want.abs()).max()) <= 0


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("other", [MOST, 1.0, 0.0, 2.0**-149])
@pytest.mark.parametrize("swapped", [False, True])
def test_scales_that_are_not_finite_stay_so(bad, other, swapped):
    for rows, n in ((3, 40), (150, 200)):
        x, w = rows_of(rows, 256, other if swapped else bad), rows_of(n, 256, bad if swapped else other, seed=1)
        x.q[::2] = 0
        want = (x.q.double() @ w.q.double().t()) * (bad * other)
        got = int8_linear(x, w, dtype=torch.float32).double()
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0, 1, -1), want.nan_to_num(0, 1, -1))


@pytest.mark.parametrize("rows,n,k", [(3, 40, 256), (150, 200, 256), (300, 256, 4096), (2100, 2304, 384)])
@pytest.mark.parametrize("power", [0, 60, -60])
def test_ordinary_scales_give_the_bits_of_their_product(rows, n, k, power):
    g = torch.Generator(device="cuda").manual_seed(2)
    x, w = (quantize_rows(torch.randn(m, k, device="cuda", generator=g) * 2.0**p) for m, p in ((rows, power), (n, -power / 2)))
    sums = (x.q.double() @ w.q.double().t()).float()
    assert torch.equal(int8_linear(x, w, dtype=torch.float32), sums * (x.scale[:, None] * w.scale[None, :]))
