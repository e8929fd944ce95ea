r"""The host path in C++ of the layers for wide networks against their Python functions: the same bits, gradients and errors."""
import pytest
import torch

from triton_helpers_b200 import _lib
from triton_helpers_b200.layers.checkpointed_linear import checkpointed_linear
from triton_helpers_b200.layers.int8_linear import Int8Rows, int8_linear, quantize_rows
from triton_helpers_b200.layers.rms_norm import rms_norm, rms_norm_int8

pytestmark = pytest.mark.gpu


def normal(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def flat(out):
    for t in out if isinstance(out, (tuple, list)) else [out]:
        yield from flat(t) if isinstance(t, tuple) else [t.detach()]


def both(call):
    r"""``call``'s outputs: native, then Python."""
    results = []
    for deferred in (False, True):
        _lib.native().defer(deferred)
        try:
            results.append(list(flat(call())))
        finally:
            _lib.native().defer(False)
    assert len(results[0]) == len(results[1])
    for a, b in zip(*results):
        assert a.dtype == b.dtype and a.shape == b.shape and a.device == b.device and torch.equal(a, b)
    return results[0]


@pytest.mark.parametrize("shape", [(1, 8), (33,), (2, 5, 100), (300, 257)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("added", [False, True])
def test_rms_norm(shape, dtype, added):
    x, gain = normal(*shape, dtype=dtype).requires_grad_(True), normal(shape[-1], seed=1, dtype=dtype).requires_grad_(True)
    residual = normal(*shape, seed=2, dtype=dtype).requires_grad_(True) if added else None
    gy, gs = normal(*shape, seed=3, dtype=dtype), normal(*shape, seed=4, dtype=dtype)
    wanted = [t for t in (x, gain, residual) if t is not None]

    def call():
        out = rms_norm(x, gain, residual)
        return list(flat(out)) + list(torch.autograd.grad(out, wanted, [gy, gs] if added else [gy]))

    both(call)
    with torch.no_grad():
        both(lambda: rms_norm(x, gain, residual))
        both(lambda: rms_norm_int8(x, gain, residual))


@pytest.mark.parametrize("shape", [(1, 16), (20,), (2, 3, 50), (140, 300)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_int8_linear(shape, dtype):
    x, weight, bias = normal(*shape, dtype=dtype), quantize_rows(normal(70, shape[-1], seed=1)), normal(70, seed=2, dtype=dtype)
    both(lambda: int8_linear(x, weight))
    both(lambda: int8_linear(x, weight, bias))
    rows = quantize_rows(x)
    both(lambda: int8_linear(rows, weight, bias, dtype))
    both(lambda: int8_linear(x, weight, dtype=torch.float32))
    both(lambda: int8_linear(Int8Rows(rows.q.contiguous(), rows.scale), weight, dtype=dtype))  # Python's: rows are copied


@pytest.mark.parametrize("shape", [(1, 16), (20,), (2, 3, 50), (140, 300)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_checkpointed_linear(shape, dtype):
    for d_out in (24, 31):
        x, w, b = normal(*shape, dtype=dtype).requires_grad_(True), normal(d_out, shape[-1], seed=1, dtype=dtype).requires_grad_(True), normal(d_out, seed=2, dtype=dtype).requires_grad_(True)
        gy = normal(*shape[:-1], d_out, seed=3, dtype=dtype)
        for bias in (None, b):

            def call(wanted):
                y = checkpointed_linear(x, w, bias)
                return [y, *torch.autograd.grad(y, wanted, gy)]

            leaves = [t for t in (x, w, bias) if t is not None]
            both(lambda: call(leaves))
            for t in leaves:
                both(lambda: call([t]))


def test_saved_tensor_hooks():
    # tensors that went to the host and came back, packed as the host left them
    x, w = normal(30, 50, dtype=torch.float16).requires_grad_(True), normal(20, 50, seed=1, dtype=torch.float16).requires_grad_(True)
    gain = normal(50, seed=2).requires_grad_(True)

    def call():
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.cuda()):
            y = checkpointed_linear(x, w)
            z, s = rms_norm(x, gain, x.detach())
        return [*torch.autograd.grad(y.sum(), [x, w]), *torch.autograd.grad(z.sum() + s.sum(), [x, gain])]

    both(call)


def test_hooks_and_shared_leaves():
    x, gain = normal(6, 32).requires_grad_(True), normal(32, seed=1).requires_grad_(True)

    def call():
        y, s = rms_norm(x, gain, x)  # the same tensor on both sides: its gradient is added up
        return torch.autograd.grad((y * s).sum(), [x, gain])

    both(call)
    w = normal(32, 32, dtype=torch.float16).requires_grad_(True)
    both(lambda: torch.autograd.grad(checkpointed_linear(w, w).sum(), [w]))


def test_an_input_changed_in_place_is_noticed():
    x, gain = normal(6, 32), normal(32, seed=1).requires_grad_(True)
    for deferred in (False, True):
        _lib.native().defer(deferred)
        try:
            y = rms_norm(x, gain)
        finally:
            _lib.native().defer(False)
        x.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
