r"""The global norm of gradients, clipping by it, and the clipped update against float64."""
import math

import pytest
import torch

from triton_helpers_b200 import _lib
from triton_helpers_b200.layers.expert_linear import ExpertLinear
from triton_helpers_b200.layers.float8_linear import Float8TrainingLinear
from triton_helpers_b200.layers.fully_fused_mlp import FullyFusedMLP
from triton_helpers_b200.layers.hash_encoding import HashEncoding
from triton_helpers_b200.layers.rms_norm import RMSNorm
from triton_helpers_b200.optim import FusedAdam, adam_update, clip_grad_norm_, clipped_adam_updates, grad_norm
from triton_helpers_b200.training import NeuralFieldTrainer

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
# float32 sums of eight squares at most (8 roundings of 2^-24), float64 from there; a square root halves that; one rounding of the norm
NORM = 1.01 * (4 + 1) * 2.0**-24


def normal(*shape, seed=0, dtype=torch.float32, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)


def exact_norm(tensors, scales=None):
    scales = scales or [1.0] * len(tensors)
    return math.sqrt(sum(s * s * float(t.double().square().sum()) for t, s in zip(tensors, scales)))


def factor_of(norm, max_norm):
    r"""As the kernel computes it, from its own norm, in float32."""
    f = torch.tensor(max_norm, dtype=torch.float32) / (norm.cpu() + torch.tensor(1e-6, dtype=torch.float32))
    return float(f.clamp_max(1.0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes", [[1], [7], [0, 5], [4096], [4097, 3, 8191], [100_003], [3_000_001, 17], [33] * 700, [5000] * 40])
def test_norm(sizes, dtype):
    tensors = [normal(n, seed=i, dtype=dtype) for i, n in enumerate(sizes)]
    want = exact_norm(tensors)
    got = grad_norm(tensors)
    assert got.dtype == torch.float32 and got.shape == () and abs(float(got) - want) <= NORM * want
    assert torch.equal(grad_norm(tensors), got)
    scales = [0.5 + i % 3 for i in range(len(sizes))]
    want = exact_norm(tensors, scales)
    assert abs(float(grad_norm(tensors, scales)) - want) <= NORM * want
    with _lib.KernelTimer():  # leaves the call to Python
        assert torch.equal(grad_norm(tensors), got)


@pytest.mark.parametrize("dtype", DTYPES)
def test_norm_of_views_and_strides(dtype):
    flat = normal(5000, dtype=dtype)
    for tensors in ([flat[1:], flat[3:4000], flat[:1], flat[7:9]], [flat.view(50, 100).t(), flat.view(50, 100)[:, ::3], flat.view(25, 200)[:, 1:30]]):
        want = exact_norm(tensors)
        assert abs(float(grad_norm(tensors)) - want) <= NORM * want
    mixed = [normal(1000, seed=i, dtype=t) for i, t in enumerate(DTYPES)]
    want = exact_norm(mixed)
    assert abs(float(grad_norm(mixed)) - want) <= NORM * want


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [1e-44, 1e-30, 1e-20, 1e-10, 1e10, 1e20, 1e30, 1e36])
def test_norm_of_far_magnitudes(size, dtype):
    tensors = [(normal(999).double() * size).to(dtype), (normal(10, seed=1).double() * size).to(dtype)]
    want = exact_norm(tensors)
    assert abs(float(grad_norm(tensors)) - want) <= NORM * want + 2.0**-149
    tensors.append(torch.ones(3, device="cuda", dtype=dtype))  # beside ordinary ones
    want = exact_norm(tensors)
    assert abs(float(grad_norm(tensors)) - want) <= NORM * want


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_norm_of_infinities_and_nan(bad):
    t = normal(5000)
    t[4321] = bad
    got = float(grad_norm([normal(3), t]))
    assert math.isnan(got) if math.isnan(bad) else got == math.inf
    assert float(grad_norm([torch.zeros(9, device="cuda")])) == 0 and float(grad_norm([torch.zeros(0, device="cuda")])) == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("max_norm", [0.0, 0.7, 1e9, math.inf])
def test_clip(dtype, max_norm):
    params = [torch.zeros(n, device="cuda", dtype=dtype, requires_grad=True) for n in (1, 4097, 333)] + [torch.zeros(3, device="cuda", requires_grad=True)]
    matrix = torch.zeros(40, 30, device="cuda", dtype=dtype, requires_grad=True)
    for i, p in enumerate(params[:3]):
        p.grad = normal(p.numel() + 1, seed=i, dtype=dtype)[1:]  # off 16 bytes
    matrix.grad = normal(30, 40, seed=7, dtype=dtype).t()
    params += [matrix, params[0]]
    live = [p for p in params[:5] if p.grad is not None]
    before = [p.grad.clone() for p in live]
    versions = [p.grad._version for p in live]
    want = exact_norm(before)
    norm = clip_grad_norm_(params, max_norm)
    assert abs(float(norm) - want) <= NORM * want
    factor = factor_of(norm, max_norm)
    for p, g, v in zip(live, before, versions):
        assert torch.equal(p.grad, (g.float() * factor).to(dtype)) and p.grad._version > v
    if max_norm < want:
        after = exact_norm([p.grad for p in live])
        # every element was rounded to its type once (float16 down to 2^-24, half of a step of its smallest)
        tiny = 2.0**-25 * math.sqrt(sum(g.numel() for g in before)) if dtype == torch.float16 else 0.0
        assert after <= max_norm * (1 + torch.finfo(dtype).eps) + tiny


def test_python_and_native_paths_agree():
    make = lambda: [torch.nn.Parameter(torch.zeros(n, device="cuda", dtype=t)) for n, t in ((1000, torch.float32), (33, torch.bfloat16), (4097, torch.float16))]  # noqa: E731
    ours, theirs = make(), make()
    for group in (ours, theirs):
        for i, p in enumerate(group):
            p.grad = normal(p.numel(), seed=i, dtype=p.dtype)
    first = clip_grad_norm_(ours, 0.5)
    with _lib.KernelTimer():  # leaves the call to Python
        second = clip_grad_norm_(theirs, 0.5)
    assert torch.equal(first, second) and all(torch.equal(p.grad, q.grad) for p, q in zip(ours, theirs))


def test_clip_of_nothing_and_of_norms_that_are_not_finite():
    p = torch.zeros(5, device="cuda", requires_grad=True)
    assert float(clip_grad_norm_([p], 1.0)) == 0
    p.grad = torch.tensor([1.0, float("inf"), 2.0, 0.0, -3.0], device="cuda")
    assert float(clip_grad_norm_(p, 1.0)) == math.inf
    assert p.grad.tolist()[0] == 0 and math.isnan(p.grad.tolist()[1])
    p.grad = torch.tensor([1.0, float("nan"), 2.0, 0.0, -3.0], device="cuda")
    assert math.isnan(float(clip_grad_norm_(p, 1.0))) and bool(p.grad.isnan().all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes", [[1], [4097, 3, 64], [1000] * 300, [50_001, 7]])
@pytest.mark.parametrize("max_norm", [0.3, 1e9])
def test_clipped_update_is_the_update_of_scaled_gradients(sizes, dtype, max_norm):
    make = lambda seed, **kw: [normal(n, seed=seed + i, **kw) for i, n in enumerate(sizes)]  # noqa: E731
    params, grads, m, v = make(0, dtype=dtype), make(1000, dtype=dtype), make(2000, scale=0.1), [t.abs() for t in make(3000, scale=0.01)]
    scales, zero = [1.0 + i % 2 for i in range(len(sizes))], [i % 3 == 0 for i in range(len(sizes))]
    mine = [[t.clone() for t in x] for x in (params, grads, m, v)]
    skipped = torch.zeros(1, dtype=torch.int32, device="cuda")
    norm = clipped_adam_updates(*mine, max_norm, 3, 1e-2, (0.9, 0.99), 1e-8, scales, zero, skipped)
    want = exact_norm(grads, scales)
    assert abs(float(norm) - want) <= NORM * want and int(skipped) == 0
    factor = torch.tensor(factor_of(norm, max_norm), dtype=torch.float32)
    for p, g, a, b, s, z in zip(params, grads, m, v, scales, zero):
        adam_update(p, g, a, b, 3, 1e-2, (0.9, 0.99), 1e-8, float(factor * s), z)
    for got, expected in zip(mine, (params, grads, m, v)):
        assert all(torch.equal(a, b) for a, b in zip(got, expected))


@pytest.mark.parametrize("dtype", DTYPES)
def test_clipped_update_of_views_off_their_packets(dtype):
    base = [normal(400, seed=i, dtype=dtype) for i in range(2)] + [normal(400, seed=2, scale=0.1), normal(400, seed=3, scale=0.01).abs()]
    aligned = [t[16:316].clone() for t in base]
    shifted = [t[3:303].copy_(a) for t, a in zip(base, aligned)]
    norm = clipped_adam_updates(*[[t] for t in shifted], 0.5, 2, 1e-2, (0.9, 0.99), 1e-8)
    want = exact_norm([aligned[1]])
    assert abs(float(norm) - want) <= NORM * want
    # squares are grouped by 16-byte packets, so the norm's last bit may be another than that of tensors on 16 bytes: the factor is its own
    adam_update(*aligned, 2, 1e-2, (0.9, 0.99), 1e-8, factor_of(norm, 0.5))
    assert all(torch.equal(a, b) for a, b in zip(aligned, shifted))


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_a_norm_that_is_not_finite_passes_over_the_step(bad):
    params = [torch.nn.Parameter(normal(50, seed=i)) for i in range(2)]
    before = [p.detach().clone() for p in params]
    opt = FusedAdam(params, lr=0.1)
    for p in params:
        p.grad = normal(50, seed=9)
    params[0].grad[7] = bad
    norm = opt.step(max_norm=1.0, zero_grad=True)
    assert not math.isfinite(float(norm)) and opt.skipped_elements() == 100
    assert all(torch.equal(p, b) for p, b in zip(params, before)) and all(bool((p.grad == 0).all()) for p in params)
    assert all(bool((opt.state[p]["exp_avg"] == 0).all()) for p in params)


def test_optimizer_step_clips_over_all_groups_and_types():
    make = lambda: [torch.nn.Parameter(normal(100 + i, seed=i, dtype=t)) for i, t in enumerate((torch.float32, torch.bfloat16, torch.float32))]  # noqa: E731
    ours, theirs = make(), make()
    opts = [FusedAdam([{"params": ps[:2]}, {"params": ps[2:], "lr": 0.05}], lr=0.01) for ps in (ours, theirs)]
    for step in range(3):
        for p, q in zip(ours, theirs):
            p.grad = normal(*p.shape, seed=50 + step, dtype=p.dtype)
            q.grad = p.grad.clone()
        want = exact_norm([p.grad for p in ours]) * 0.25
        norm = opts[0].step(grad_scale=0.25, max_norm=0.5)
        assert abs(float(norm) - want) <= NORM * want
        opts[1].step(grad_scale=float(torch.tensor(0.25) * torch.tensor(factor_of(norm, 0.5), dtype=torch.float32)))
        assert all(torch.equal(p, q) for p, q in zip(ours, theirs))
    assert opts[0].step() is None


def test_clipping_in_a_captured_graph():
    params = [torch.nn.Parameter(normal(n, seed=n)) for n in (1000, 33)]
    for p in params:
        p.grad = normal(*p.shape, seed=3)
    clip_grad_norm_(params, 1.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip_grad_norm_(params, 1.0)
    for p in params:
        p.grad.copy_(normal(*p.shape, seed=4))
    want = exact_norm([p.grad for p in params])
    graph.replay()
    assert abs(float(norm) - want) <= NORM * want
    after = exact_norm([p.grad for p in params])
    assert abs(after - 1.0) <= 2.0**-20


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("watched", [False, True])
def test_trainer_clips(dtype, watched):
    def make(max_grad_norm):
        torch.manual_seed(0)
        encoding = HashEncoding(2**10, 4, 2, 2, 4, 64).cuda().to(dtype)
        mlp = FullyFusedMLP(8, 16, 8, 2).cuda().to(dtype)
        return NeuralFieldTrainer(encoding, mlp, lr=1e-2, eps=1e-8, max_grad_norm=max_grad_norm)

    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.rand(512, 2, device="cuda", generator=g) * 2 - 1
    target = torch.randn(512, 8, device="cuda", generator=g, dtype=dtype)
    free, loose, tight = make(None), make(1e6), make(1e-4)
    if watched:
        for t in (free, loose, tight):
            if t.optimizer is not None:
                t.optimizer.register_step_post_hook(lambda *_: None)
    def moments(t):
        if t.optimizer is not None:
            return [t.optimizer.state[p]["exp_avg"] for p in t.parameters()]
        return [t._state.table_m, t._state.mlp_m]

    losses = [t.step(x, target) for t in (free, loose, tight)]
    # a bound that is not reached changes nothing (the table's gradient is summed in any order, in its own type)
    for a, b in zip(moments(free), moments(loose)):
        assert float((a - b).abs().max()) <= 64 * torch.finfo(dtype).eps * float(a.abs().max())
    # after one step the first moment is a tenth of the clipped gradient (1e-6 is added to the norm)
    assert abs(exact_norm(moments(tight)) / 1e-5 - 1) < 1e-3
    assert abs(exact_norm(moments(loose)) / float(loose.last_grad_norm) / 0.1 - 1) < 1e-5
    for _ in range(2):
        losses += [t.step(x, target) for t in (free, loose, tight)]
    assert free.last_grad_norm is None and 1e-2 < float(tight.last_grad_norm) < 1e3
    assert all(math.isfinite(float(v)) for v in losses) and tight.skipped_elements() == 0


def test_a_network_of_wide_layers_trains_step_by_step():
    class Network(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.norm = RMSNorm(128)
            self.up = Float8TrainingLinear(128, 256)
            self.experts = ExpertLinear(4, 256, 128)

        def forward(self, x, ends):
            return x + self.experts(torch.relu(self.up(self.norm(x))), ends)

    torch.manual_seed(0)
    net = Network().cuda().bfloat16()
    opt = FusedAdam(net.parameters(), lr=1e-3)
    x, target = normal(200, 128, dtype=torch.bfloat16), normal(200, 128, seed=1, dtype=torch.bfloat16)
    ends = torch.tensor([50, 50, 120, 190], device="cuda", dtype=torch.int32)
    for _ in range(3):
        out = net(x, ends)
        assert torch.equal(out[190:], x[190:])
        (out - target).float().square().mean().backward()
        grads = [p.grad for p in net.parameters()]
        assert all(g is not None and g.isfinite().all() for g in grads)
        want = exact_norm(grads)
        norm = opt.step(max_norm=0.1, zero_grad=True)
        assert abs(float(norm) - want) <= NORM * want
    assert opt.skipped_elements() == 0 and all(p.isfinite().all() for p in net.parameters()) and _lib.lib().th_linear_tc_status() == 0
