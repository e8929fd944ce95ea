r"""A trainer whose optimizer's ``step`` was replaced, by a function that knows nothing of clipping."""
import pytest
import torch

from triton_helpers_b200.layers.fully_fused_mlp import FullyFusedMLP
from triton_helpers_b200.layers.hash_encoding import HashEncoding
from triton_helpers_b200.training import NeuralFieldTrainer

pytestmark = pytest.mark.gpu


def trainer(**kwargs):
    torch.manual_seed(0)
    encoding = HashEncoding(2**10, 4, 2, 2, 4, 64).cuda()
    return NeuralFieldTrainer(encoding, FullyFusedMLP(8, 16, 8, 2).cuda(), lr=1e-2, eps=1e-8, **kwargs)


def batch():
    g = torch.Generator(device="cuda").manual_seed(1)
    return torch.rand(512, 2, device="cuda", generator=g) * 2 - 1, torch.randn(512, 8, device="cuda", generator=g)


@pytest.mark.parametrize("graph", [False, True])
def test_a_step_of_the_former_signature_is_called(graph):
    seen = {}
    for replaced in (False, True):
        t = trainer()
        if graph:  # a hook of a module has the step go through the autograd graph
            t.mlp.register_forward_hook(lambda *_: None)
        if replaced:
            inner, calls = t.optimizer.step, []

            def step(grad_scale=1.0, zero_grad=False):
                calls.append((grad_scale, zero_grad))
                return inner(grad_scale, zero_grad)

            t.optimizer.step = step
        t.step(*batch())
        assert t.last_grad_norm is None
        seen[replaced] = [t.optimizer.state[p]["exp_avg"] for p in t.parameters()]
    assert len(calls) == 1 and calls[0][0] > 0 and calls[0][1] != graph
    # a tenth of the gradients, which are summed in any order: some tens of additions' roundings, each of half a step of the largest at most
    assert all(float((a - b).abs().max()) <= 64 * torch.finfo(torch.float32).eps * float(a.abs().max()) for a, b in zip(seen[False], seen[True]))


@pytest.mark.parametrize("graph", [False, True])
def test_a_replaced_step_is_told_of_clipping_that_was_asked_for(graph):
    t, asked = trainer(max_grad_norm=0.5), []
    if graph:
        t.mlp.register_forward_hook(lambda *_: None)
    inner = t.optimizer.step

    def step(grad_scale=1.0, zero_grad=False, max_norm=None):
        asked.append(max_norm)
        return inner(grad_scale, zero_grad, max_norm)

    t.optimizer.step = step
    t.step(*batch())
    assert asked == [0.5] and float(t.last_grad_norm) > 0


@pytest.mark.parametrize("graph", [False, True])
def test_an_update_of_the_former_signature_is_called(graph):
    t, calls = trainer(), []
    if graph:
        t.mlp.register_forward_hook(lambda *_: None)
    inner = t.optimizer.update

    def update(group, params, grads, grad_scales, zero_grads):
        calls.append(len(params))
        return inner(group, params, grads, grad_scales, zero_grads)

    t.optimizer.update = update
    before = [p.detach().clone() for p in t.parameters()]
    t.step(*batch())
    assert calls == [len(before)] and t.last_grad_norm is None
    assert not any(torch.equal(a, b) for a, b in zip(before, t.parameters()))
