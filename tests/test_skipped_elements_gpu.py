r"""The count of elements that Adam passes over: a 32-bit counter that stays at its most instead of turning negative."""
import pytest
import torch

from triton_helpers_b200 import _lib
from triton_helpers_b200.optim import FusedAdam, adam_update, adam_updates, clipped_adam_updates

pytestmark = pytest.mark.gpu

MOST = 2**31 - 1
HYPER = (1, 1e-3, (0.9, 0.99), 1e-8)


def tensors(n, dtype=torch.float32, bad=float("nan")):
    p, g = torch.ones(n, device="cuda", dtype=dtype), torch.full((n,), bad, device="cuda", dtype=dtype)
    return p, g, torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")


def counter(value):
    return torch.tensor([value], dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("before,n", [(0, 1000), (MOST - 1000, 1000), (MOST - 999, 1000), (MOST - 3, 100_003), (MOST, 5), (MOST - 1, 3_000_000)])
def test_updates_count_up_to_the_most(before, n, dtype):
    want = min(before + n, MOST)
    held = counter(before)
    adam_update(*tensors(n, dtype), *HYPER, skipped=held)
    assert int(held) == want
    for deferred in (False, True):  # the native path and the Python one
        _lib.native().defer(deferred)
        try:
            held = counter(before)
            adam_updates(*[[t] for t in tensors(n, dtype)], [1.0], [False], *HYPER, held)
            assert int(held) == want
            held = counter(before)
            clipped_adam_updates(*[[t] for t in tensors(n, dtype)], 1.0, *HYPER, skipped=held)
            assert int(held) == want
        finally:
            _lib.native().defer(False)


def test_many_steps_of_a_norm_that_is_not_finite():
    p = torch.nn.Parameter(torch.ones(3_000_000, device="cuda"))
    opt = FusedAdam([p], lr=0.1)
    p.grad = torch.zeros_like(p)
    p.grad[7] = float("inf")
    for step in range(1, 721):  # 2.16e9 elements
        opt.step(max_norm=1.0)
        if step in (1, 700):
            assert opt.skipped_elements() == step * 3_000_000
    assert opt.skipped_elements() == MOST and bool((p == 1).all())
