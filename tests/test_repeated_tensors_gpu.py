r"""Clipping where a tensor is given more than once: a gradient that several parameters hold is scaled once, a parameter is updated once or refused."""
import pytest
import torch

from triton_helpers_b200 import _lib
from triton_helpers_b200.optim import clip_grad_norm_, clipped_adam_updates

pytestmark = pytest.mark.gpu


@pytest.fixture(params=[False, True], ids=["native", "python"])
def path(request):
    _lib.native().defer(request.param)
    yield
    _lib.native().defer(False)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 1000, 300_001])
def test_a_shared_gradient_is_scaled_once(path, n, dtype):
    params = [torch.nn.Parameter(torch.zeros(m, device="cuda", dtype=dtype)) for m in (n, n, 77, n)]
    shared = torch.full((n,), 3.0, device="cuda", dtype=dtype)
    for p in (params[0], params[1], params[3]):
        p.grad = shared
    params[2].grad = torch.full((77,), 3.0, device="cuda", dtype=dtype)
    norm = clip_grad_norm_(params, 1.0)
    want = 3.0 * (3 * n + 77) ** 0.5
    assert abs(float(norm) / want - 1) <= 2.0**-20
    # the factor in float32, then one rounding to the gradient's type
    half = torch.finfo(dtype).eps / 2
    for g in (shared, params[2].grad):
        assert float((g.double() * want / 3 - 1).abs().max()) <= 1.01 * (half + 2.0**-19)


def test_a_strided_shared_gradient_is_scaled_once(path):
    params = [torch.nn.Parameter(torch.zeros(30, 20, device="cuda")) for _ in range(2)]
    shared = torch.full((20, 30), 2.0, device="cuda").t()
    for p in params:
        p.grad = shared
    want = 2.0 * 1200**0.5
    assert abs(float(clip_grad_norm_(params, 1.0)) / want - 1) <= 2.0**-20
    assert float((shared * want / 2 - 1).abs().max()) <= 2.0**-19


def test_many_gradients_are_all_scaled(path):
    # more than a launch's list, neighbours in one buffer among them, and empty ones, which begin where their neighbours do
    flat = torch.ones(700 * 16, device="cuda")
    params = [torch.nn.Parameter(torch.zeros(16, device="cuda")) for _ in range(700)] + [torch.nn.Parameter(torch.zeros(0, device="cuda")) for _ in range(3)]
    for i, p in enumerate(params):
        p.grad = flat[16 * i : 16 * i + 16] if i < 700 else flat[16 * (i - 700) :][:0]
    norm = clip_grad_norm_(params, 1.0)
    assert abs(float(norm) ** 2 / flat.numel() - 1) <= 2.0**-19 and float((flat * float(norm) - 1).abs().max()) <= 2.0**-19


def test_an_update_takes_a_parameter_once(path):
    p, g, m, v = (torch.ones(50, device="cuda") for _ in range(4))
    with pytest.raises(ValueError, match="once"):
        clipped_adam_updates([p, p], [g, g], [m, m.clone()], [v, v.clone()], 1.0, 1, 1e-3, (0.9, 0.99), 1e-8)
    assert bool((p == 1).all())
    empty = torch.ones(0, device="cuda")
    clipped_adam_updates([p, empty, empty], [g, empty, empty], [m, empty, empty], [v, empty, empty], 1.0, 1, 1e-3, (0.9, 0.99), 1e-8)
    assert bool((p != 1).all())
