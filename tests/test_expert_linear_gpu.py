r"""Linear layers of several experts against a float64 loop over them."""
import pytest
import torch

from triton_helpers_b200 import _lib
from triton_helpers_b200.layers.expert_linear import ExpertLinear, expert_linear

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]


def normal(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def ends_of(counts, dtype=torch.int32):
    return torch.tensor(counts, device="cuda").cumsum(0).to(dtype)


def spans(ends, rows):
    r"""(first, end) of each expert as the kernels read the ends."""
    start, out = 0, []
    for end in ends.tolist():
        end = max(start, min(end, rows))
        out.append((start, end))
        start = end
    return out


def exact(x, w, ends, gy):
    x, w, gy = x.detach().double(), w.detach().double(), gy.double()
    y, dx, dw = x.new_zeros(x.shape[0], w.shape[1]), torch.zeros_like(x), torch.zeros_like(w)
    reach = [torch.zeros_like(t) for t in (y, dx, dw)]
    for e, (a, b) in enumerate(spans(ends, x.shape[0])):
        for out, far, p, q in ((y, reach[0], x[a:b], w[e].t()), (dx, reach[1], gy[a:b], w[e])):
            out[a:b], far[a:b] = p @ q, p.abs() @ q.abs()
        dw[e], reach[2][e] = gy[a:b].t() @ x[a:b], gy[a:b].abs().t() @ x[a:b].abs()
    return (y, dx, dw), reach


def assert_near(got, want, reach, terms):
    # float32 sums of exact products in an unknown order, each addition off by at most a step of 2^-23, then one rounding; float16 may be below its
    # normal values
    half = torch.finfo(got.dtype).eps / 2
    allowed = 1.01 * ((terms + 1) * 2.0**-23 * reach + half * want.abs()) + (2.0**-25 if got.dtype == torch.float16 else 2.0**-134)
    assert got.isfinite().all()
    off = ((got.double() - want).abs() / allowed).max() if got.numel() else torch.zeros(())
    assert float(off) <= 1, f"{float(off)} of what is allowed"


def check(x, w, ends, gy):
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    y = expert_linear(x, w, ends)
    grads = torch.autograd.grad(y, (x, w), gy, retain_graph=True)
    want, reach = exact(x, w, ends, gy)
    most = max([b - a for a, b in spans(ends, x.shape[0])])
    for got, value, far, terms in zip((y.detach(), *grads), want, reach, (w.shape[2], w.shape[1], most)):
        assert_near(got, value, far, terms)
    again = torch.autograd.grad(y, (x, w), gy)
    assert all(torch.equal(a, b) for a, b in zip(again, grads)) and torch.equal(expert_linear(x, w, ends), y)
    assert _lib.lib().th_linear_tc_status() == 0
    return y.detach(), *grads


COUNTS = [
    [1], [5], [0], [300], [0, 0, 7], [1, 1, 1, 1], [128, 128], [127, 129, 1], [0, 257, 0, 3, 0], [64, 0, 65, 63, 200], [700, 2, 2, 2],
    [3] * 40, [0] * 30 + [9] + [0] * 30, [16] * 8, [33] * 5, [1000, 24],
]  # fmt: skip


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,n", [(64, 128), (520, 333), (1, 1), (8, 300), (257, 64)])
@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: "-".join(map(str, c)) if len(c) < 8 else f"{len(c)}x{max(c)}")
def test_forward_and_gradients(counts, d, n, dtype):
    rows = sum(counts) + 5  # some behind the last
    x, w = normal(rows, d, dtype=dtype), (normal(len(counts), n, d, seed=1) * d**-0.5).to(dtype)
    y, dx, dw = check(x, w, ends_of(counts), normal(rows, n, seed=2, dtype=dtype))
    assert bool((y[sum(counts) :] == 0).all()) and bool((dx[sum(counts) :] == 0).all())
    for e, count in enumerate(counts):
        assert count or bool((dw[e] == 0).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("counts,d,n", [([2000, 1500, 0, 600], 1024, 768), ([300] * 16, 512, 1024), ([4096], 256, 2048), ([2] * 64, 2048, 1024), ([40, 0, 90, 20], 4096, 256)])
def test_larger_sizes(counts, d, n, dtype):
    rows = sum(counts)
    x, w = normal(rows, d, dtype=dtype), (normal(len(counts), n, d, seed=1) * d**-0.5).to(dtype)
    check(x, w, ends_of(counts), (0.1 * normal(rows, n, seed=2)).to(dtype))


@pytest.mark.parametrize("experts,rows", [(1024, 3000), (1000, 300), (999, 60_000), (33, 1)])
def test_many_experts(experts, rows):
    g = torch.Generator().manual_seed(0)
    counts = torch.bincount(torch.randint(0, experts, (rows,), generator=g) // 3 * 2 % experts, minlength=experts).tolist()
    x, w = normal(rows, 64, dtype=torch.bfloat16), (normal(experts, 40, 64, seed=1) * 0.125).to(torch.bfloat16)
    check(x, w, ends_of(counts), normal(rows, 40, seed=2, dtype=torch.bfloat16))


@pytest.mark.parametrize("ends", [[5, 3, 9], [-4, 2, 100], [100, 100, 100], [0, 0, 0], [20, 0, 7], [-1, -2, -3]])
def test_ends_out_of_order_or_range(ends):
    x, w = normal(20, 40, dtype=torch.float16), normal(3, 24, 40, seed=1, dtype=torch.float16)
    for dtype in (torch.int32, torch.int64):
        check(x, w, torch.tensor(ends, device="cuda", dtype=dtype), normal(20, 24, seed=2, dtype=torch.float16))


@pytest.mark.parametrize("counts", [[30, 0, 50], [3, 4, 0], [200, 100, 20]])
def test_what_rows_behind_the_last_hold_reaches_nothing(counts):
    rows = sum(counts)
    x, w, gy = normal(rows + 70, 72, dtype=torch.bfloat16), normal(3, 136, 72, seed=1, dtype=torch.bfloat16), normal(rows + 70, 136, seed=2, dtype=torch.bfloat16)
    clean = check(x[:rows], w, ends_of(counts), gy[:rows])
    x[rows:], gy[rows:] = float("nan"), float("inf")
    x, w = x.requires_grad_(), w.requires_grad_()
    y = expert_linear(x, w, ends_of(counts))
    got = y.detach(), *torch.autograd.grad(y, (x, w), gy)
    for a, b in zip(got[:2], clean[:2]):
        assert torch.equal(a[:rows], b) and bool((a[rows:] == 0).all())
    assert torch.equal(got[2], clean[2])


@pytest.mark.parametrize("counts", [[30, 9, 50], [1, 2, 1], [200, 100, 20]])
@pytest.mark.parametrize("d,n", [(72, 136), (70, 131)])
def test_a_nan_stays_with_its_expert(counts, d, n):
    rows = sum(counts)
    x, w, gy = normal(rows, d, dtype=torch.float16), normal(3, n, d, seed=1, dtype=torch.float16), normal(rows, n, seed=2, dtype=torch.float16)
    clean = check(x, w, ends_of(counts), gy)
    mine = slice(counts[0], counts[0] + counts[1])
    x[mine], w[1], gy[mine] = float("nan"), float("inf"), float("nan")
    x, w = x.requires_grad_(), w.requires_grad_()
    y = expert_linear(x, w, ends_of(counts))
    got = y.detach(), *torch.autograd.grad(y, (x, w), gy)
    keep = torch.ones(rows, dtype=torch.bool, device="cuda")
    keep[mine] = False
    assert torch.equal(got[0][keep], clean[0][keep]) and torch.equal(got[1][keep], clean[1][keep])
    assert torch.equal(got[2][0], clean[2][0]) and torch.equal(got[2][2], clean[2][2])
    assert bool(got[0][mine].isnan().all()) and bool(got[1][mine].isnan().all()) and bool(got[2][1].isnan().all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_operands(dtype):
    counts = [30, 0, 55]
    ends, gy = ends_of(counts), normal(85, 48, seed=2, dtype=dtype)
    big, weights = normal(85, 200, dtype=dtype), normal(6, 100, 64, seed=1, dtype=dtype)
    check(big[:, 8:72], weights[::2, :48], ends, gy)
    check(big[:, 5:69], weights[:3, 3:51], ends, gy)
    check(big.t()[:64].t(), weights[:3].transpose(1, 2)[:, :48, :64], ends, gy)
    check(big[:, :50], weights[3:, :48, 7:57], ends, gy)
    x, w = big[:, :64].detach().requires_grad_(), weights[:3, :48].detach().requires_grad_()
    expert_linear(x, w, ends).sum().backward()  # an expanded gradient
    want = exact(x, w, ends, torch.ones(85, 48, device="cuda"))
    for got, value, far, terms in zip((x.grad, w.grad), want[0][1:], want[1][1:], (48, 55)):
        assert_near(got, value, far, terms)


def test_gradients_against_differences():
    # whole numbers: every sum is exact in float32 and every result in float16, so that differences of the layer, which is linear in each
    # input, are the gradients exactly
    g = torch.Generator(device="cuda").manual_seed(0)
    whole = lambda *shape: torch.randint(-2, 3, shape, device="cuda", generator=g).to(torch.float16)  # noqa: E731
    x, w, gy, ends = whole(40, 24), whole(3, 16, 24), whole(40, 16), ends_of([17, 0, 20])
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    dx, dw = torch.autograd.grad(expert_linear(xg, wg, ends), (xg, wg), gy)
    loss = lambda x, w: float((expert_linear(x, w, ends).double() * gy.double()).sum())  # noqa: E731
    for got, h, difference in (
        (dx, hx := whole(40, 24), loss(x + hx, w) - loss(x - hx, w)),
        (dw, hw := whole(3, 16, 24), loss(x, w + hw) - loss(x, w - hw)),
    ):
        assert float((got.double() * h.double()).sum()) == difference / 2


def test_frozen_parts_empty_rows_autocast_and_module():
    layer = ExpertLinear(3, 40, 24, device="cuda", dtype=torch.bfloat16)
    x, ends = normal(30, 40, dtype=torch.bfloat16).requires_grad_(), ends_of([10, 15, 5], torch.int64)
    y = layer(x, ends)
    dx, dw = torch.autograd.grad(y, (x, layer.weight), torch.ones_like(y))
    (alone,) = torch.autograd.grad(expert_linear(x, layer.weight.detach(), ends), x, torch.ones_like(y))
    assert torch.equal(alone, dx)
    (alone,) = torch.autograd.grad(layer(x.detach(), ends), layer.weight, torch.ones_like(y))
    assert torch.equal(alone, dw)
    none = x.detach()[:0].requires_grad_()
    out = layer(none, ends)
    out.sum().backward()
    assert out.shape == (0, 24) and none.grad.shape == (0, 40) and bool((layer.weight.grad == 0).all())
    wide = ExpertLinear(3, 40, 24, device="cuda")
    with torch.autocast("cuda", torch.bfloat16):
        z = wide(x.float(), ends)
    assert z.dtype == torch.bfloat16 and torch.equal(z, expert_linear(x, wide.weight.bfloat16(), ends))


def test_python_and_native_paths_agree():
    x, w = normal(90, 200, dtype=torch.float16).requires_grad_(), normal(4, 61, 200, seed=1, dtype=torch.float16).requires_grad_()
    gy, ends = normal(90, 61, seed=3, dtype=torch.float16), ends_of([20, 30, 0, 35])
    run = lambda: [y := expert_linear(x, w, ends), *torch.autograd.grad(y, (x, w), gy)]  # noqa: E731,F841
    first = run()
    with _lib.KernelTimer():  # leaves the calls to Python
        second = run()
    assert all(torch.equal(p, q) for p, q in zip(first, second))


def test_a_captured_graph_follows_new_ends():
    x, w = normal(64, 72, dtype=torch.float16), normal(4, 48, 72, seed=1, dtype=torch.float16)
    ends = ends_of([16, 16, 16, 16])
    expert_linear(x, w, ends)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = expert_linear(x, w, ends)
    for counts in ([64, 0, 0, 0], [0, 3, 40, 5], [1, 2, 3, 4]):
        ends.copy_(ends_of(counts))
        graph.replay()
        assert torch.equal(y, expert_linear(x, w, ends))
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        z = expert_linear(x, w, ends)
    torch.cuda.current_stream().wait_stream(other)
    assert torch.equal(z, y)


def test_second_derivatives_raise():
    x, w = normal(6, 40, dtype=torch.float16).requires_grad_(), normal(2, 8, 40, seed=1, dtype=torch.float16).requires_grad_()
    (dx,) = torch.autograd.grad(expert_linear(x, w, ends_of([2, 4])).float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="not differentiable twice"):
        dx.float().sum().backward()
