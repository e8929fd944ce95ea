r"""Layers of experts at sizes where pairs of CTAs share a tile: the rows of an expert's last stage that are not its own are cleared in both CTAs' shared memory."""
import pytest
import torch

from triton_helpers_b200 import _lib
from triton_helpers_b200.layers.expert_linear import expert_linear

pytestmark = pytest.mark.gpu

WIDTH = 1024  # with some thousand rows of a few experts the estimate takes pairs of 256 x 256 in every direction (profiled: expert_gemm_kernel<..., 256, 2, ...>)


def normal(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def gradients(x, w, ends, gy):
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    y = expert_linear(x, w, ends)
    return [y.detach(), *torch.autograd.grad(y, (x, w), gy)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("counts", [[1000, 1001, 999, 1063], [1, 2047, 1500, 600], [1300, 63, 65, 2700], [1024, 1087, 961, 1000]])
@pytest.mark.parametrize("who", [1, 2])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_bad_expert_keeps_to_itself(counts, who, bad, dtype):
    rows = sum(counts) + 40
    x, w, gy = normal(rows, WIDTH, dtype=dtype), normal(4, WIDTH, WIDTH, seed=1, dtype=dtype) * WIDTH**-0.5, normal(rows, WIDTH, seed=2, dtype=dtype)
    ends = torch.tensor(counts, device="cuda").cumsum(0).to(torch.int32)
    clean = gradients(x, w, ends, gy)
    mine = slice(sum(counts[:who]), sum(counts[: who + 1]))
    x[mine], gy[mine] = bad, bad
    x[sum(counts) :], gy[sum(counts) :] = bad, bad  # nobody's rows as well
    got = gradients(x, w, ends, gy)
    keep = torch.ones(rows, dtype=torch.bool, device="cuda")
    keep[mine] = False
    for i in (0, 1):
        assert torch.equal(got[i][keep], clean[i][keep]) and bool((got[i][sum(counts) :] == 0).all()) and not bool(got[i][mine].isfinite().all())
    others = [e for e in range(4) if e != who]
    assert torch.equal(got[2][others], clean[2][others]) and not bool(got[2][who].isfinite().any())
    assert _lib.lib().th_linear_tc_status() == 0


def test_many_passes_give_the_same_bits():
    # the last stages of eight uneven experts, again and again beside another stream's products
    counts = [700, 641, 1, 1030, 333, 800, 511, 449]
    x, w = normal(sum(counts), WIDTH, dtype=torch.bfloat16), normal(8, WIDTH, WIDTH, seed=1, dtype=torch.bfloat16)
    gy, ends = normal(sum(counts), WIDTH, seed=2, dtype=torch.bfloat16), torch.tensor(counts, device="cuda").cumsum(0).to(torch.int32)
    want = gradients(x, w, ends, gy)
    side, others = torch.cuda.Stream(), []
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(30):
        with torch.cuda.stream(side):
            others.append(gradients(x, w, ends, gy))
        got = gradients(x, w, ends, gy)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for got in others for a, b in zip(got, want))
