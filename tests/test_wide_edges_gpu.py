r"""Layers for wide networks where a definition has to hold at its edges: roundings, layouts, scales, threads, modes."""
import threading

import pytest
import torch

from triton_helpers_b200 import _lib
from triton_helpers_b200.layers.checkpointed_linear import checkpointed_linear
from triton_helpers_b200.layers.int8_linear import Int8Rows, dequantize_rows, int8_linear, quantize_rows
from triton_helpers_b200.layers.rms_norm import rms_norm, rms_norm_int8

pytestmark = pytest.mark.gpu


def normal(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,d_in,d_out", [(300, 256, 512), (3001, 100, 77), (2048, 512, 640)])
def test_weight_gradient_is_that_of_the_rows_back_in_16_bits(rows, d_in, d_out, dtype):
    # the operand's one rounding to 16 bits is all that is lost: float32 sums of the rounded rows, and the result's half step
    x, w = normal(rows, d_in, dtype=dtype), normal(d_out, d_in, seed=1, dtype=dtype).requires_grad_(True)
    gy = normal(rows, d_out, seed=2, dtype=dtype)
    (got,) = torch.autograd.grad(checkpointed_linear(x, w), [w], gy)
    x16 = dequantize_rows(quantize_rows(x), dtype).double()
    want, reach = gy.double().t() @ x16, gy.double().abs().t() @ x16.abs()
    assert bool(((got.double() - want).abs() <= (rows + 2) * 2.0**-23 * reach + 1.01 * torch.finfo(dtype).eps / 2 * want.abs() + 2.0**-24).all())


@pytest.mark.parametrize("lead", [(4, 3), (3, 4), (2, 4, 3), (4, 2, 3), (4, 1, 3)])
def test_expanded_8_bit_rows(lead):
    # rows that share memory along any leading dimension: what they hold is what counts, and nothing past them is read
    rows, weight = quantize_rows(normal(4, 40)), quantize_rows(normal(24, 40, seed=1))
    shape = [4 if n == 4 else 1 for n in lead]
    q, scale = rows.q.view(*shape, 40).expand(*lead, 40), rows.scale.view(shape).expand(lead).contiguous()
    want = int8_linear(Int8Rows(q.contiguous(), scale), weight, dtype=torch.float32)
    assert torch.equal(int8_linear(Int8Rows(q, scale), weight, dtype=torch.float32), want)
    assert torch.equal(want, int8_linear(rows, weight, dtype=torch.float32).view(*shape, 24).expand(*lead, 24))
    assert torch.equal(dequantize_rows(Int8Rows(q, scale)), q.float() * scale[..., None])


def test_expanded_8_bit_weights():
    rows, one = quantize_rows(normal(5, 48)), quantize_rows(normal(1, 48, seed=1))
    weight = Int8Rows(one.q.expand(7, 48), one.scale.expand(7).contiguous())
    assert torch.equal(int8_linear(rows, weight, dtype=torch.float32), int8_linear(rows, one, dtype=torch.float32).expand(5, 7))


def test_norm_backward_from_several_threads():
    # two widths of one kernel with different amounts of shared memory, each from a host thread and a stream of its own
    lib, failed = _lib.lib(), []
    torch.cuda.synchronize()

    def work(d, seed):
        with torch.cuda.stream(torch.cuda.Stream()):
            s, gy, gs, gain = (normal(*shape, seed=seed + k, dtype=torch.float16) for k, shape in enumerate([(8, d), (8, d), (8, d), (d,)]))
            rstd = torch.ones(8, device="cuda")
            size = lib.th_rms_norm_bwd_workspace_bytes(8, d, 1)
            dx, dw, scratch = torch.empty_like(s), torch.empty_like(gain), torch.empty(size, dtype=torch.uint8, device="cuda")
            stream = _lib.stream_ptr(s.device)
            for _ in range(3000):
                rc = lib.th_rms_norm_bwd(
                    s.data_ptr(), d, gain.data_ptr(), 1, rstd.data_ptr(), gy.data_ptr(), d, gs.data_ptr(), d, dx.data_ptr(), dw.data_ptr(),
                    scratch.data_ptr(), size, 8, d, 1, stream,
                )  # fmt: skip
                if rc:
                    failed.append((d, rc, lib.th_last_error_string()))
                    return
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(d, 10 * k)) for k, d in enumerate([4096, 2320, 4096, 2320])]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed


# few tokens, a tile per token group, split and whole products
@pytest.mark.parametrize("tokens,d_in,d_out", [(1, 64, 40), (3, 4096, 200), (100, 512, 130), (300, 200, 77), (300, 4096, 64), (2100, 640, 1930)])
@pytest.mark.parametrize("x_size,w_size", [(1e-30, 1e-6), (1e-20, 1e-17), (1e30, 1e-6), (1e18, 1e17), (1e-26, 1e30)])
def test_scales_far_from_one(tokens, d_in, d_out, x_size, w_size):
    # the scales' product, or a sum times one scale, is outside of what float32 holds well; the result is inside
    rows = quantize_rows(normal(tokens, d_in) * x_size)
    weight = quantize_rows(normal(d_out, d_in, seed=1) * w_size)
    bias = normal(d_out, seed=2) * (x_size * w_size)
    acc = rows.q.double() @ weight.q.double().t()
    scaled = acc * rows.scale.double()[:, None] * weight.scale.double()
    assert bool((scaled.abs() < 2.0**127).all())
    for b in (None, bias):
        y = int8_linear(rows, weight, b, dtype=torch.float32)
        want = scaled if b is None else scaled + b.double()
        # four roundings (conversion, product of the scales, product, bias), and half of float32's smallest step
        assert bool(((y.double() - want).abs() <= 4.01 * 2.0**-24 * (scaled.abs() + (0 if b is None else b.double().abs())) + 2.0**-150).all())
    if x_size * w_size > 2.0**-126:
        y = int8_linear(rows, weight, dtype=torch.bfloat16)
        assert bool(((y.double() - scaled).abs() <= (2.0**-8 + 4 * 2.0**-24) * scaled.abs() + 2.0**-134).all())


@pytest.mark.parametrize("tokens", [1, 40, 300])
def test_sums_of_nothing_under_the_largest_scales(tokens):
    # x and w are orthogonal as integers: 0, and not 0 times an infinite product of the scales
    x = torch.full((tokens, 64), torch.finfo(torch.float32).max, device="cuda")
    w = torch.full((24, 64), 1e30, device="cuda")
    w[:, ::2] *= -1
    y = int8_linear(quantize_rows(x), quantize_rows(w), dtype=torch.float32)
    assert bool((y == 0).all())
    w[0] = 1e30  # one output is past float32
    y = int8_linear(quantize_rows(x), quantize_rows(w), dtype=torch.float32)
    assert bool((y[:, 0] == float("inf")).all()) and bool((y[:, 1:] == 0).all())


@pytest.fixture(params=["native", "python"])
def path(request):
    _lib.native().defer(request.param == "python")
    yield request.param
    _lib.native().defer(False)


@pytest.mark.parametrize("leaf", [True, False])
def test_a_second_derivative_is_refused_and_not_dropped(path, leaf):
    def inputs(dtype):
        x = normal(6, 32, dtype=dtype).requires_grad_(True)
        return x, (lambda: x if leaf else x * 1), normal(32, seed=1, dtype=dtype).requires_grad_(True), normal(24, 32, seed=2, dtype=dtype).requires_grad_(True)

    layers = {
        "norm": (torch.float32, lambda h, gain, w: rms_norm(h, gain)),
        "norm of a sum": (torch.float32, lambda h, gain, w: sum(rms_norm(h, gain, h))),
        "linear": (torch.float16, lambda h, gain, w: checkpointed_linear(h, w)),
    }
    for dtype, layer in layers.values():
        x, h, gain, w = inputs(dtype)
        parameter = w if dtype == torch.float16 else gain
        plain = torch.autograd.grad(layer(h(), gain, w).sum(), [x, parameter])
        for k in range(2):
            y = layer(h(), gain, w)
            g = torch.autograd.grad(y.sum(), [x, parameter], create_graph=True)
            assert all(torch.equal(a, b) for a, b in zip(g, plain))
            loss = g[k].float().square().sum() + y.float().sum() + x.float().sum() + parameter.float().sum()
            for call in (lambda: loss.backward(retain_graph=True), *(lambda t=t: torch.autograd.grad(loss, [t], retain_graph=True) for t in (x, parameter))):
                with pytest.raises(RuntimeError, match="not differentiable twice"):
                    call()
        y = layer(h(), gain, w)  # an incoming gradient with a history of its own
        scale = torch.ones((), device="cuda", dtype=y.dtype, requires_grad=True)
        (g,) = torch.autograd.grad((y * scale).sum(), [x], create_graph=True)
        with pytest.raises(RuntimeError, match="not differentiable twice"):
            torch.autograd.grad(g.sum() + scale, [scale])
    # the sum beside the norm is a sum: its derivatives of any order are
    x = normal(6, 32).requires_grad_(True)
    s = rms_norm(x, torch.ones(32, device="cuda"), x.detach())[1]
    (g,) = torch.autograd.grad(s.square().sum(), [x], create_graph=True)
    (second,) = torch.autograd.grad(g.sum(), [x])
    assert torch.equal(second, torch.full_like(x, 2.0))


def test_functions_without_a_gradient_refuse_one(path):
    x, gain, w = normal(6, 32), normal(32, seed=1), quantize_rows(normal(24, 32, seed=2))
    rows, bias = quantize_rows(x), normal(24, seed=3)
    calls = {  # by the tensor that would need the gradient
        "quantize_rows": (x, lambda t: quantize_rows(t)),
        "dequantize_rows": (rows.scale, lambda t: dequantize_rows(Int8Rows(rows.q, t))),
        "rms_norm_int8": (gain, lambda t: rms_norm_int8(x, t)),
        "rms_norm_int8 ": (x, lambda t: rms_norm_int8(x, gain, t)),
        "int8_linear": (x, lambda t: int8_linear(t, w)),
        "int8_linear ": (bias, lambda t: int8_linear(x, w, t)),
        "int8_linear  ": (w.scale, lambda t: int8_linear(x, Int8Rows(w.q, t))),
        "int8_linear   ": (rows.scale, lambda t: int8_linear(Int8Rows(rows.q, t), w, dtype=torch.float32)),
    }
    for t, call in calls.values():
        leaf = t.clone().requires_grad_(True)
        with pytest.raises(RuntimeError, match="no gradient"):
            call(leaf)
        with torch.no_grad():
            want, got = call(t), call(leaf)
        assert all(torch.equal(a, b) for a, b in zip(*(v if isinstance(v, tuple) else (v,) for v in (want, got))) if torch.is_tensor(a))
        with torch.autograd.forward_ad.dual_level():
            dual = torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises(RuntimeError, match="no gradient"):
                    call(dual)
            call(t)  # without a tangent: as elsewhere


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("given", [torch.float16, torch.bfloat16, torch.float32])
def test_autocast_takes_the_type_that_it_is_given(given, dtype):
    # 1e5 is past float16: it is finite in and out under bfloat16
    size = 1e5 if dtype == torch.bfloat16 and given != torch.float16 else 1.0
    x = (normal(30, 96) * size).to(given).requires_grad_(True)
    w, b = normal(56, 96, seed=1, dtype=given).requires_grad_(True), normal(56, seed=2, dtype=given).requires_grad_(True)
    gy = (normal(30, 56, seed=3) * size).to(dtype)
    with torch.autocast("cuda", dtype):
        y = checkpointed_linear(x, w, b)
    grads = torch.autograd.grad(y, [x, w, b], gy)
    cast = [t.detach().to(dtype).requires_grad_(True) for t in (x, w, b)]
    want = checkpointed_linear(*cast)
    assert y.dtype == dtype and bool(y.isfinite().all()) and torch.equal(y, want)
    for got, leaf, exact in zip(grads, (x, w, b), torch.autograd.grad(want, cast, gy)):
        assert got.dtype == leaf.dtype and torch.equal(got, exact.to(given))
    with torch.autocast("cuda", dtype), torch.no_grad():
        assert torch.equal(checkpointed_linear(x, w, b), y)


# both sides of every width at which another number of threads or of 16-byte packets a thread takes over
PACKETS = [1, 2, 6, 7, 8, 9, 14, 16, 17, 30, 32, 33, 60, 64, 124, 128, 129, 256, 257, 496, 512, 513, 1000, 1024, 1025, 1984, 2048, 2049, 3968, 4096, 4097, 7936, 8192, 8193]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("packets", PACKETS)
def test_widths_where_the_kernel_changes(packets, dtype):
    per = 16 // dtype.itemsize
    for d in {packets * per, max(1, packets * per - 3), packets * per + 1}:
        x, r, gain = normal(2, d, dtype=dtype), normal(2, d, seed=1, dtype=dtype), (1 + 0.3 * normal(d, seed=2)).to(dtype)
        gy, gs = normal(2, d, seed=3, dtype=dtype), normal(2, d, seed=4, dtype=dtype)
        for residual in (None, r):
            leaves = [t.clone().requires_grad_(True) for t in (x, gain)]
            out = rms_norm(*leaves, residual, 1e-5)
            y, s = out if residual is not None else (out, leaves[0])
            grads = torch.autograd.grad(out, leaves, (gy, gs) if residual is not None else gy)
            v, g, dy = s.detach().double(), gain.double(), gy.double()
            rstd = (v.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
            h = v * rstd
            c = (dy * g * h).mean(-1, keepdim=True)
            dx = rstd * (dy * g - h * c) + (gs.double() if residual is not None else 0)
            reach = rstd * ((dy * g).abs() + h.abs() * (dy * g * h).abs().mean(-1, keepdim=True)) + (gs.double().abs() if residual is not None else 0)
            # a row's sum: up to 70 additions of a thread and 10 over the team, and some twenty roundings beside it; then the result's own half step
            half, step = 1.01 * torch.finfo(dtype).eps / 2, 100 * 2.0**-24
            for got, want, size in ((y, h * g, (h * g).abs()), (grads[0], dx, reach), (grads[1], (dy * h).sum(0), (dy * h).abs().sum(0))):
                assert bool(((got.detach().double() - want).abs() <= step * size + half * want.abs() + 2.0**-25).all())
            rows = rms_norm_int8(x, gain, residual, 1e-5)
            rows = rows[0] if residual is not None else rows
            top = (h * g).abs().amax(-1, keepdim=True)
            assert bool(((rows.q.double() - h * g * 127 / top).abs() <= 0.5 + 127 * 3 * step).all())
        rows, top = quantize_rows(x), x.float().abs().amax(-1, keepdim=True).clamp_min(2.0**-100)
        assert torch.equal(rows.q, torch.round(x.float() * (torch.full_like(top, 127.0) / top)).to(torch.int8))


def test_threads_with_a_stream_each():
    # pairs of CTAs, single ones and rows of several streams start beside one another, with deep queues: the bits of a pass alone
    def passes(r, d, n, dtype):
        x, res, g, w, b = normal(r, d, dtype=dtype), normal(r, d, seed=1, dtype=dtype), normal(d, seed=2, dtype=dtype), normal(n, d, seed=3, dtype=dtype) * 0.05, normal(n, seed=4, dtype=dtype)
        gz, gs, w8 = normal(r, n, seed=5, dtype=dtype), normal(r, d, seed=6, dtype=dtype), quantize_rows(w)
        leaves = [t.requires_grad_(True) for t in (x, res, g, w, b)]

        def one():
            y, s = rms_norm(x, g, res)
            z = checkpointed_linear(y, w, b)
            grads = torch.autograd.grad([z, s], leaves, [gz, gs])
            with torch.no_grad():
                rows, added = rms_norm_int8(x, g, res)
                return [z.detach(), *grads, added, int8_linear(rows, w8, dtype=dtype), int8_linear(y.detach(), w8, b)]

        return one

    shapes = [(2100, 4100, 4096, torch.bfloat16), (2100, 4100, 77, torch.float16), (3, 100, 4096, torch.float16), (700, 100, 4096, torch.bfloat16)]
    calls = [passes(*s) for s in shapes]
    want = [call() for call in calls]
    torch.cuda.synchronize()
    got = [None] * 4

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(60):
                got[k] = calls[k]()
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(a, b) for out, alone in zip(got, want) for a, b in zip(out, alone))
    assert _lib.lib().th_linear_tc_status() == 0
