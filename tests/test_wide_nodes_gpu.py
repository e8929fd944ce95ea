r"""The 8-bit training layer and the layers of experts where autograd is asked for more than a backward pass: saved-tensor hooks, function transforms, forward
mode, tracing, subclasses, freed and repeated graphs; and a clipped update that sees the sum over ranks."""
import math

import pytest
import torch

from triton_helpers_b200 import _lib
from triton_helpers_b200.layers.expert_linear import expert_linear
from triton_helpers_b200.layers.float8_linear import float8_linear, float8_training_linear, quantize_float8_weight
from triton_helpers_b200.layers.fully_fused_mlp import FullyFusedMLP
from triton_helpers_b200.layers.hash_encoding import HashEncoding
from triton_helpers_b200.layers.int8_linear import Int8Rows, int8_linear, quantize_rows
from triton_helpers_b200.training import NeuralFieldTrainer

pytestmark = pytest.mark.gpu

OPERATORS = ["float8", "float8 bias", "experts", "experts off 16 bytes"]


def normal(*shape, seed=0, dtype=torch.float16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def operator(name):
    r"""(function of its leaves, the leaves, an incoming gradient)"""
    if name.startswith("float8"):
        leaves = [normal(150, 200), normal(136, 200, seed=1)] + ([normal(136, seed=2)] if "bias" in name else [])
        return float8_training_linear, [t.requires_grad_() for t in leaves], normal(150, 136, seed=3)
    d = 203 if "off" in name else 200
    ends = torch.tensor([40, 40, 130], device="cuda", dtype=torch.int32)
    leaves = [normal(150, d), normal(3, 136, d, seed=1)]
    return lambda x, w: expert_linear(x, w, ends), [t.requires_grad_() for t in leaves], normal(150, 136, seed=3)


def gradients(call, leaves, gy):
    y = call(*leaves)
    return [y.detach(), *torch.autograd.grad(y, leaves, gy)]


def equal(got, want):
    return len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("name", OPERATORS)
def test_native_and_python_paths_agree(name):
    call, leaves, gy = operator(name)
    want = gradients(call, leaves, gy)
    _lib.native().defer(True)
    try:
        assert equal(gradients(call, leaves, gy), want)
    finally:
        _lib.native().defer(False)


@pytest.mark.parametrize("python", [False, True])
@pytest.mark.parametrize("name", OPERATORS)
def test_saved_tensors_go_through_their_hooks(name, python):
    call, leaves, gy = operator(name)
    want = gradients(call, leaves, gy)
    _lib.native().defer(python)
    try:
        with torch.autograd.graph.save_on_cpu():
            y = call(*leaves)
        assert equal(torch.autograd.grad(y, leaves, gy), want[1:])
        packed = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: packed.append(t.shape) or t.clone(), lambda t: t.clone()):
            y = call(*leaves)
        assert packed and equal(torch.autograd.grad(y, leaves, gy), want[1:])
    finally:
        _lib.native().defer(False)


@pytest.mark.parametrize("name", OPERATORS)
def test_a_hook_that_returns_less_is_refused(name):
    call, leaves, gy = operator(name)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t[..., : t.shape[-1] // 2]):
        y = call(*leaves)
    with pytest.raises(RuntimeError, match="saved-tensor hook"):
        torch.autograd.grad(y, leaves, gy)


@pytest.mark.parametrize("name", OPERATORS)
def test_function_transforms_are_refused_or_right(name):
    call, leaves, gy = operator(name)
    x, *rest = [t.detach() for t in leaves]
    want = gradients(call, leaves, gy)
    with pytest.raises(RuntimeError):  # no rule for a batch dimension
        torch.func.vmap(lambda x: call(x, *rest))(x.expand(2, *x.shape))
    with torch.autograd.forward_ad.dual_level():  # no rule for tangents
        with pytest.raises((RuntimeError, NotImplementedError)):
            call(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)), *rest)
    # and neither leaves anything behind
    assert equal(gradients(call, leaves, gy), want)


@pytest.mark.parametrize("name", OPERATORS)
def test_a_trace_follows_its_input(name):
    call, leaves, _ = operator(name)
    x, *rest = [t.detach() for t in leaves]
    with torch.no_grad():
        traced = torch.jit.trace(call, (x, *rest), check_trace=False)
        assert torch.equal(traced(x * 0.5, *rest), call(x * 0.5, *rest))


@pytest.mark.parametrize("name", OPERATORS)
def test_a_tensor_subclass(name):
    class Rows(torch.Tensor):
        pass

    call, leaves, _ = operator(name)
    x, *rest = [t.detach() for t in leaves]
    y = call(x.as_subclass(Rows), *rest)
    assert torch.equal(y.as_subclass(torch.Tensor), call(x, *rest))


@pytest.mark.parametrize("name", OPERATORS)
def test_a_freed_graph_and_changed_tensors_are_errors(name):
    call, leaves, gy = operator(name)
    y = call(*leaves)
    first = torch.autograd.grad(y, leaves, gy, retain_graph=True)
    assert equal(torch.autograd.grad(y, leaves, gy), first)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y, leaves, gy)
    if name.startswith("experts"):  # which keep the tensors themselves
        y = call(*leaves)
        with torch.no_grad():
            leaves[1].mul_(1.0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(y, leaves, gy)


@pytest.mark.parametrize("name", OPERATORS)
def test_each_gradient_by_itself(name):
    call, leaves, gy = operator(name)
    want = gradients(call, leaves, gy)
    for i in range(len(leaves)):
        some = [t.detach().requires_grad_(i == j) for j, t in enumerate(leaves)]
        y = call(*some)
        (got,) = torch.autograd.grad(y, [some[i]], gy)
        assert torch.equal(got, want[1 + i])
        (got,) = torch.autograd.grad(call(*leaves), [leaves[i]], gy)
        assert torch.equal(got, want[1 + i])


@pytest.mark.parametrize("name", OPERATORS)
def test_an_expanded_gradient(name):
    call, leaves, gy = operator(name)
    want = gradients(call, leaves, torch.ones_like(gy))
    assert equal(torch.autograd.grad(call(*leaves).sum(), leaves), want[1:])
    want = gradients(call, leaves, gy[:1].expand_as(gy).contiguous())
    assert equal(torch.autograd.grad(call(*leaves), leaves, gy[:1].expand_as(gy)), want[1:])


def test_a_serving_layer_of_a_subclass():
    class Rows(torch.Tensor):
        pass

    x, w = normal(20, 300), quantize_float8_weight(normal(70, 300, seed=1))
    assert torch.equal(float8_linear(x.as_subclass(Rows), w).as_subclass(torch.Tensor), float8_linear(x, w))


@pytest.mark.parametrize("n", [333, 330, 300, 136])
@pytest.mark.parametrize("rows", [3, 150])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_integer_products_into_a_part_have_their_values(rows, n, dtype):
    d, lib = 264, _lib.lib()
    x, w = quantize_rows(normal(rows, d, dtype=torch.float32)), quantize_rows(normal(n, d, seed=1, dtype=torch.float32))
    out = torch.full((rows + 10, 400), 7.0, device="cuda", dtype=dtype)
    _lib.check(
        lib.th_int8_linear(x.q.data_ptr(), x.q.stride(0), x.scale.data_ptr(), w.q.data_ptr(), w.q.stride(0), w.scale.data_ptr(), None, out.data_ptr(), 400, rows, d,
                           n, _lib.DTYPE_CODE[dtype], _lib.stream_ptr(out.device)),
        "th_int8_linear",
    )  # fmt: skip
    sums = (x.q.double() @ w.q.double().t()).float()  # exact
    assert torch.equal(out[:rows, :n], (sums * (x.scale[:, None] * w.scale[None, :])).to(dtype))
    assert torch.equal(out[:rows, :n], int8_linear(Int8Rows(x.q, x.scale), w, dtype=dtype))
    assert bool((out[rows:] == 7).all()) and bool((out[:, n:] == 7).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_a_trainer_clips_the_gradient_of_all_ranks(dtype, monkeypatch):
    # a second rank with the same points, as the sum over ranks sees it: the mean over the global batch, its norm and the update are one rank's
    from triton_helpers_b200 import training

    def make():
        torch.manual_seed(0)
        encoding, mlp = HashEncoding(2**10, 4, 2, 2, 4, 64).cuda().to(dtype), FullyFusedMLP(8, 16, 8, 2).cuda().to(dtype)
        return NeuralFieldTrainer(encoding, mlp, lr=1e-2, eps=1e-8, grad_out_scale=64.0, max_grad_norm=1e-3)

    class TwoRanks:
        def __init__(self, *_, **__):
            self.held = []

        def start(self, grads):
            self.held += list(grads)

        def finish(self):
            for g in self.held:
                g.mul_(2)

    def moments(t):
        return [t.optimizer.state[p]["exp_avg"] for p in t.parameters()] if t.optimizer is not None else [t._state.table_m, t._state.mlp_m]

    g = torch.Generator(device="cuda").manual_seed(1)
    x, target = torch.rand(512, 2, device="cuda", generator=g) * 2 - 1, torch.randn(512, 8, device="cuda", generator=g, dtype=dtype)
    one, two = make(), make()
    one.step(x, target)
    monkeypatch.setattr(training, "PendingReduce", TwoRanks)
    monkeypatch.setattr(training, "allreduce_gradients", lambda grads, group=None: [t.mul_(2) for t in grads])
    monkeypatch.setattr(NeuralFieldTrainer, "world_size", lambda self: 2)
    two.step(x, target)
    # doubled gradients at half the scale: the same numbers but for sums in any order, in the table's own type
    allowed = 64 * torch.finfo(dtype).eps
    assert abs(float(two.last_grad_norm) / float(one.last_grad_norm) - 1) <= allowed and math.isfinite(float(one.last_grad_norm))
    for a, b in zip(moments(one), moments(two)):
        assert float((a - b).abs().max()) <= allowed * float(a.abs().max())
    norm = math.sqrt(sum(float(m.double().square().sum()) for m in moments(two)))
    assert abs(norm / 1e-4 - 1) < 1e-2  # a tenth of what the bound lets through
