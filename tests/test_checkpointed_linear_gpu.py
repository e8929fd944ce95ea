r"""The linear layer that keeps its input in 8 bits, against float64."""
import copy

import pytest
import torch

from triton_helpers_b200 import _lib
from triton_helpers_b200.layers.checkpointed_linear import CheckpointedLinear, checkpointed_linear
from triton_helpers_b200.layers.int8_linear import dequantize_rows, quantize_rows
from triton_helpers_b200.layers.rms_norm import RMSNorm

pytestmark = pytest.mark.gpu

STEP = 2.0**-23  # a float32 addition in the tensor core, truncated at worst


def normal(*shape, seed=0, dtype=torch.float32, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)


def near(got, want, reach, terms, operands=0.0):
    r"""Sums of ``terms`` products of magnitudes adding up to ``reach``; ``operands``: what rounding an operand adds; and the result's half step."""
    bound = ((terms + 2) * STEP + operands) * reach + 1.01 * torch.finfo(got.dtype).eps / 2 * want.abs() + 2.0**-24
    return got.isfinite().all() and bool(((got.double() - want).abs() <= bound).all())


def assert_pass(x, w, b, gy, y, grads):
    rows, d_in, d_out = x.numel() // x.shape[-1], w.shape[1], w.shape[0]
    x8 = dequantize_rows(quantize_rows(x), torch.float32).double().reshape(-1, d_in)
    half = torch.finfo(x.dtype).eps / 2
    x, w, gy = x.double().reshape(-1, d_in), w.double(), gy.double().reshape(-1, d_out)
    bias = 0.0 if b is None else b.double()
    assert near(y.reshape(-1, d_out), x @ w.t() + bias, x.abs() @ w.abs().t() + (0.0 if b is None else b.double().abs()), d_in)
    assert near(grads[0].reshape(-1, d_in), gy @ w, gy.abs() @ w.abs(), d_out)
    assert near(grads[1], gy.t() @ x8, gy.abs().t() @ x8.abs(), rows, 1.01 * half)  # q * scale is rounded to 16 bits
    if b is not None:
        assert near(grads[2], gy.sum(0), gy.abs().sum(0), rows)


# from one row to many tiles; widths that are no multiple of anything; products of one CTA, split and of two CTAs
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize(
    "rows,d_in,d_out",
    [(1, 16, 16), (1, 1, 1), (2, 8, 24), (7, 33, 65), (128, 128, 128), (130, 64, 200), (300, 256, 512), (64, 1000, 40), (5000, 48, 72), (3001, 100, 77),
     (1, 4096, 300), (2048, 256, 2048), (2300, 2050, 1100), (4097, 2049, 130), (2500, 1100, 2049)],
)  # fmt: skip
def test_forward_and_gradients(rows, d_in, d_out, dtype):
    x, w = normal(rows, d_in, dtype=dtype).requires_grad_(True), normal(d_out, d_in, seed=1, dtype=dtype, scale=d_in**-0.5).requires_grad_(True)
    b = normal(d_out, seed=2, dtype=dtype).requires_grad_(True) if rows % 2 == 0 else None
    gy = normal(rows, d_out, seed=3, dtype=dtype, scale=0.1)
    y = checkpointed_linear(x, w, b)
    grads = torch.autograd.grad(y, [t for t in (x, w, b) if t is not None], gy)
    assert y.dtype == dtype and [g.dtype for g in grads] == [dtype] * len(grads) and [g.shape for g in grads] == [t.shape for t in (x, w, b) if t is not None]
    assert_pass(x.detach(), w.detach(), None if b is None else b.detach(), gy, y.detach(), grads)


def test_gradients_against_differences():
    # the loss is linear in w, x and b each, so differences of the float64 definition are exact; the weight's see the 8-bit rows
    x, w, b = normal(20, 48, dtype=torch.float16).requires_grad_(True), normal(24, 48, seed=1, dtype=torch.float16).requires_grad_(True), normal(24, seed=2, dtype=torch.float16).requires_grad_(True)
    gy = normal(20, 24, seed=3, dtype=torch.float16)
    grads = torch.autograd.grad(checkpointed_linear(x, w, b), [x, w, b], gy)
    x8 = dequantize_rows(quantize_rows(x.detach())).double()
    loss = lambda a, m, c: ((a @ m.t() + c) * gy.double()).sum()  # noqa: E731
    for k, (g, first) in enumerate(zip(grads, (x.detach().double(), x8, x8))):
        at = [first, w.detach().double(), b.detach().double()]
        direction = normal(*g.shape, seed=9 + k).double()
        moved = [t + direction if j == k else t for j, t in enumerate(at)]
        slope = float(loss(*moved) - loss(*at))
        # half a step of float16 on every entry of the gradient, and as much again on the entries of the 8-bit rows
        reach = [gy.double().abs() @ w.detach().double().abs(), gy.double().abs().t() @ x8.abs(), gy.double().abs().sum(0)][k]
        assert abs(float((g.double() * direction).sum()) - slope) <= 2.0**-10 * float((reach * direction.abs()).sum()) + 1e-6


def test_only_what_is_wanted_is_kept_and_computed():
    x, w, b, gy = normal(40, 64, dtype=torch.float16), normal(32, 64, seed=1, dtype=torch.float16), normal(32, seed=2, dtype=torch.float16), normal(40, 32, seed=3, dtype=torch.float16)
    full = [t.clone().requires_grad_(True) for t in (x, w, b)]
    want = torch.autograd.grad(checkpointed_linear(*full), full, gy)
    for k in range(3):
        args = [x, w, b]
        args[k] = args[k].clone().requires_grad_(True)
        (got,) = torch.autograd.grad(checkpointed_linear(*args), [args[k]], gy)
        assert torch.equal(got, want[k])
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
        checkpointed_linear(*full)
    assert sorted(str(t.dtype) for t in kept if t.numel()) == ["torch.float16", "torch.float32", "torch.int8"]  # the weight, scales, rows
    with torch.no_grad():
        assert torch.equal(checkpointed_linear(*full), checkpointed_linear(x, w, b))


def test_layouts():
    base, w = normal(6, 5, 64, dtype=torch.float16), normal(40, 64, seed=1, dtype=torch.float16)
    b, wide = normal(40, seed=2, dtype=torch.float16), normal(6, 5, 80, seed=3, dtype=torch.float16)
    for x in (base, base.transpose(0, 1), base[:, 1:], base[:, :1].expand(6, 3, 64), base[0, 0], base[:0]):
        for weight in (w, w.t().contiguous().t(), torch.cat([w, w], 1)[:, :64], torch.cat([w[:, :1], w], 1)[:, 1:]):
            leaf, wl, bl = x.detach().clone().requires_grad_(True), weight.detach().requires_grad_(True), b.clone().requires_grad_(True)
            y = checkpointed_linear(leaf if x.is_contiguous() else x, wl, bl)
            assert y.shape == (*x.shape[:-1], 40) and y.is_contiguous()
            gy = normal(*y.shape, seed=5, dtype=torch.float16)
            grads = torch.autograd.grad(y, [leaf, wl, bl] if x.is_contiguous() else [wl, bl], gy)
            if x.is_contiguous():
                assert_pass(x.detach(), weight, b, gy, y.detach(), grads)
    x = base.clone().requires_grad_(True)
    wl = w.clone().requires_grad_(True)
    for gy in (wide[..., :40], wide[..., 1:41], wide[..., ::2], wide[:, :1, :40].expand(6, 5, 40)):
        y = checkpointed_linear(x, wl)
        assert_pass(base, w, None, gy, y.detach(), torch.autograd.grad(y, [x, wl], gy))


def test_bad_rows_stay_alone():
    x, w = normal(200, 64, dtype=torch.float16), normal(48, 64, seed=1, dtype=torch.float16)
    x[3, 5], x[150, 0] = float("inf"), float("nan")
    y = checkpointed_linear(x, w)
    good = torch.ones(200, dtype=torch.bool, device="cuda")
    good[3] = good[150] = False
    assert bool(y[good].isfinite().all()) and not bool(y[~good].isfinite().any())
    leaf, weight = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    gy = torch.ones(200, 48, device="cuda", dtype=torch.float16)
    gy[7, 2] = float("inf")
    dx, dw = torch.autograd.grad(checkpointed_linear(leaf, weight), [leaf, weight], gy)
    rest = torch.ones(200, dtype=torch.bool, device="cuda")
    rest[7] = False
    assert bool(dx[rest].isfinite().all()) and not bool(dx[7].isfinite().any())
    assert bool(dw.isnan().all())  # every weight meets the two rows


def test_results_repeat():
    x, w, b = normal(3001, 1000, dtype=torch.bfloat16).requires_grad_(True), normal(777, 1000, seed=1, dtype=torch.bfloat16).requires_grad_(True), normal(777, seed=2, dtype=torch.bfloat16).requires_grad_(True)
    gy = normal(3001, 777, seed=3, dtype=torch.bfloat16)
    once = lambda: [y := checkpointed_linear(x, w, b), *torch.autograd.grad(y, [x, w, b], gy)]  # noqa: E731
    first = once()
    for _ in range(4):
        assert all(torch.equal(p, q) for p, q in zip(first, once()))


def test_module_autocast_and_state():
    plain = torch.nn.Linear(96, 56).cuda()
    layer = CheckpointedLinear(96, 56).cuda()
    layer.load_state_dict(plain.state_dict())
    x = normal(30, 96).requires_grad_(True)
    with torch.autocast("cuda", torch.float16):
        y = layer(x)
    assert y.dtype == torch.float16
    y.float().square().sum().backward()
    assert layer.weight.grad.dtype == torch.float32 and x.grad.dtype == torch.float32
    half = copy.deepcopy(layer).half()
    with torch.no_grad():
        assert torch.equal(half(x.half()), y)


def test_captured_step_beside_an_eager_graph():
    x, w = normal(256, 128, dtype=torch.float16).requires_grad_(True), normal(64, 128, seed=1, dtype=torch.float16).requires_grad_(True)
    gy = normal(256, 64, seed=3, dtype=torch.float16)
    step = lambda: [y := checkpointed_linear(x, w), *torch.autograd.grad(y, [x, w], gy)]  # noqa: E731
    step()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(step())
    with torch.no_grad():
        x.copy_(normal(256, 128, seed=8, dtype=torch.float16))
    want = step()
    for graph in graphs:
        graph.replay()
    for out in outs:
        assert all(torch.equal(p.detach(), q.detach()) for p, q in zip(out, want))


class Block(torch.nn.Module):
    def __init__(self, d):
        super().__init__()
        self.norm, self.up, self.down = RMSNorm(d), CheckpointedLinear(d, 2 * d), CheckpointedLinear(2 * d, d)

    def forward(self, x, residual):
        y, s = self.norm(x, residual)
        return self.down(torch.relu(self.up(y))), s


def test_together_as_they_are_trained():
    torch.manual_seed(0)
    blocks = torch.nn.ModuleList(Block(64) for _ in range(2)).cuda().bfloat16()
    x = normal(100, 64, dtype=torch.bfloat16).requires_grad_(True)

    def run(parts, x, norm, linear):
        h, s = x, torch.zeros_like(x)
        for blk in parts:
            y, s = norm(blk, h, s)
            h = linear(blk.down, torch.relu(linear(blk.up, y)))
        return h + s

    out = run(blocks, x, lambda blk, h, s: blk.norm(h, s), lambda layer, v: layer(v))
    gy = normal(100, 64, seed=5, dtype=torch.bfloat16)
    got = torch.autograd.grad(out, [x, *blocks.parameters()], gy)
    exact = copy.deepcopy(blocks).double()
    xd = x.detach().double().requires_grad_(True)

    def norm64(blk, h, s):
        s = h + s
        return s * (s.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * blk.norm.weight, s

    want = torch.autograd.grad(run(exact, xd, norm64, lambda layer, v: torch.nn.functional.linear(v, layer.weight, layer.bias)), [xd, *exact.parameters()], gy.double())
    for a, b in zip(got, want):
        # some ten bfloat16 roundings on the way (2^-8 each at most), 8-bit rows (half a step of 1 / 127 of the row's largest, which is about
        # three times its root mean square: 3 / 254), and ReLUs whose argument is within a rounding of zero
        assert float((a.double() - b).norm() / b.norm()) <= 10 * 2.0**-8 + 3 / 254


def test_refusals():
    x, w = normal(4, 32, dtype=torch.float16), normal(8, 32, dtype=torch.float16)
    with pytest.raises(AssertionError, match="Input dimension"):
        checkpointed_linear(x[:, :31], w)
    with pytest.raises(AssertionError, match="Bias"):
        checkpointed_linear(x, w, w[0])
    with pytest.raises(TypeError):
        checkpointed_linear(x.float(), w.float())
    with pytest.raises(TypeError):
        checkpointed_linear(x, w.bfloat16())
    with pytest.raises(AssertionError, match="same device"):
        checkpointed_linear(x, w.cpu())
    leaf = x.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(checkpointed_linear(leaf, w).sum(), [leaf], create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()  # not differentiable twice
    assert _lib.lib().th_linear_tc_status() == 0


def test_memory_around_operands_is_left():
    # padding beside the operands holds NaN: it meets neither a product nor a sum
    wide, weights = normal(70, 48, dtype=torch.float16), normal(40, 40, seed=1, dtype=torch.float16)
    wide[:, 33:], weights[:, 33:] = float("nan"), float("nan")
    x, w, b = wide[:, :33], weights[:, :33], normal(40, seed=2, dtype=torch.float16)
    leaf, wl, bl = wide.clone().requires_grad_(True), weights.clone().requires_grad_(True), b.clone().requires_grad_(True)
    gwide = normal(70, 48, seed=3, dtype=torch.float16)
    gwide[:, 40:] = float("nan")
    gy = gwide[:, :40]
    y = checkpointed_linear(leaf[:, :33], wl[:, :33], bl)
    dx, dw, db = torch.autograd.grad(y, [leaf, wl, bl], gy)
    assert_pass(x, w, b, gy, y.detach(), [dx[:, :33], dw[:, :33], db])
    assert bool((dx[:, 33:] == 0).all()) and bool((dw[:, 33:] == 0).all())


@pytest.mark.parametrize("rows", [511, 512, 513, 4099])
def test_bias_gradient_of_few_and_many_rows(rows):
    x, w, b = normal(rows, 16, dtype=torch.bfloat16), normal(300, 16, seed=1, dtype=torch.bfloat16), normal(300, seed=2, dtype=torch.bfloat16).requires_grad_(True)
    gy = normal(rows, 300, seed=3, dtype=torch.bfloat16)
    (alone,) = torch.autograd.grad(checkpointed_linear(x, w, b), [b], gy)
    assert near(alone, gy.double().sum(0), gy.double().abs().sum(0), rows)
    weight = w.clone().requires_grad_(True)
    both = torch.autograd.grad(checkpointed_linear(x, weight, b), [b, weight], gy)
    assert torch.equal(both[0], alone)


def test_offsets_past_32_bits():
    x = normal(1, 64, dtype=torch.float16).expand(1_000_000, 64).contiguous()
    x[-1] = normal(64, seed=5, dtype=torch.float16)
    w = normal(2304, 64, seed=1, dtype=torch.float16).requires_grad_(True)
    y = checkpointed_linear(x, w)  # 2.3e9 outputs
    assert torch.equal(y[-1], checkpointed_linear(x[-1:], w)[0]) and torch.equal(y[-2], y[0])
    gy = torch.zeros_like(y)
    gy[-1] = 1
    (dw,) = torch.autograd.grad(y, [w], gy)
    want = dequantize_rows(quantize_rows(x[-1])).double().expand(2304, 64)
    assert near(dw, want, want.abs(), 1, 1.01 * torch.finfo(torch.float16).eps / 2)


@pytest.mark.parametrize("rows,d_in,d_out", [(930, 40, 14272), (130, 16, 16000), (3000, 70, 9000)])
def test_tiles_that_lie_outside_in_part(rows, d_in, d_out):
    # many short tiles a CTA, some of whose rows are all outside: what is stored ahead of them stays
    x, w = normal(rows, d_in, dtype=torch.bfloat16), normal(d_out, d_in, seed=1, dtype=torch.bfloat16)
    first = checkpointed_linear(x, w)
    assert near(first, x.double() @ w.double().t(), x.double().abs() @ w.double().abs().t(), d_in)
    for _ in range(20):
        assert torch.equal(checkpointed_linear(x, w), first)
