r"""8-bit floating-point blocks and the linear layers on them against a float64 statement of their definition."""
from contextlib import nullcontext

import pytest
import torch

from triton_helpers_b200 import _lib
from triton_helpers_b200.layers.float8_linear import (
    Float8Blocks,
    Float8Linear,
    Float8TrainingLinear,
    dequantize_float8,
    float8_linear,
    float8_training_linear,
    quantize_float8_rows,
    quantize_float8_weight,
)

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32]
SIXTEEN = DTYPES[:2]


def normal(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def blocks_by_definition(x, tall):
    r"""The definition in elementary float32 operations (tensors on both sides of a division: a true one)."""
    m, k = x.shape
    held = torch.zeros(-(-m // tall) * tall, -(-k // 128) * 128, device=x.device)
    held[:m, :k] = x.float()
    held = held.view(held.shape[0] // tall, tall, -1, 128)
    a = held.abs().amax((1, 3), keepdim=True).clamp_min(2.0**-60)
    top = torch.full_like(a, 448.0)
    q = (held * (top / a)).to(torch.float8_e4m3fn)
    return q.view(held.shape[0] * tall, -1)[:m, :k], (a / top)[:, 0, :, 0]


def stands_for(q, scale, tall):
    r"""What blocks stand for, float64."""
    wide = scale.double().repeat_interleave(tall, 0)[: q.shape[0]].repeat_interleave(128, 1)[:, : q.shape[1]]
    return q.float().double() * wide


def same_values(a, b):
    return torch.equal(a.float(), b.float())


def bound(x, w, exact, dtype, bias=None):
    r"""Products of two e4m3 values are exact in float32. A block's 128 of them are added in an unknown order, each addition off by at most
    a whole step (2^-23) of a partial sum; three roundings for the scales; then the blocks' sums, the bias and the result's rounding (half a step, or half of the type's smallest)."""
    reach = x.abs() @ w.abs().t() + (0 if bias is None else bias.double().abs())
    adds = 128 * 2.0**-23 + (-(-x.shape[1] // 128) + 4) * 2.0**-24
    return 1.01 * adds * reach + 1.01 * torch.finfo(dtype).eps / 2 * exact.abs() + (2.0**-25 if dtype == torch.float16 else 2.0**-134)


def assert_linear(y, x, w, bias=None):
    x, w = x.reshape(-1, x.shape[-1]), w
    exact = x @ w.t() + (0 if bias is None else bias.double())
    assert y.isfinite().all()
    off = (y.double().reshape(exact.shape) - exact).abs() / bound(x, w, exact, y.dtype, bias)
    assert float(off.max()) <= 1, f"{float(off.max())} of what is allowed"


# ---- blocks -------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 16), (17, 127), (5, 128), (2, 3, 129), (33, 1000), (16, 512), (4, 1028), (1, 16384), (300, 640)])
def test_rows_are_the_definition_bit_for_bit(shape, dtype):
    x = (normal(*shape) * torch.exp(2 * normal(*shape[:-1], 1, seed=1))).to(dtype)
    q, scale = quantize_float8_rows(x)
    want_q, want_scale = blocks_by_definition(x.reshape(-1, shape[-1]), 1)
    assert q.shape == x.shape and q.dtype == torch.float8_e4m3fn and scale.shape == (*shape[:-1], -(-shape[-1] // 128)) and scale.dtype == torch.float32
    assert same_values(q.reshape(-1, shape[-1]), want_q) and torch.equal(scale.reshape(want_scale.shape), want_scale)
    assert q.data_ptr() % 16 == 0 and (q.dim() < 2 or q.shape[-2] == 1 or q.stride(-2) % 16 == 0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (128, 128), (129, 127), (3, 1000), (300, 50), (777, 640)])
def test_weights_are_the_definition_bit_for_bit(shape, dtype):
    w = (normal(*shape) * torch.exp(normal(shape[0], 1, seed=1))).to(dtype)
    q, scale = quantize_float8_weight(w)
    want_q, want_scale = blocks_by_definition(w, 128)
    assert same_values(q, want_q) and torch.equal(scale, want_scale)


@pytest.mark.parametrize("dtype", DTYPES)
def test_blocks_of_strided_shifted_and_expanded_rows(dtype):
    big = normal(40, 700, dtype=dtype)
    for x in (big[:, 3:300], big[::2, 8:264], big.t(), big[:, ::3], big[5:6].expand(9, -1)):
        want_q, want_scale = blocks_by_definition(x, 1)
        q, scale = quantize_float8_rows(x)
        assert same_values(q, want_q) and torch.equal(scale, want_scale)
        want_q, want_scale = blocks_by_definition(x, 128)
        q, scale = quantize_float8_weight(x)
        assert same_values(q, want_q) and torch.equal(scale, want_scale)


@pytest.mark.parametrize("dtype", DTYPES)
def test_blocks_back(dtype):
    for shape, make, tall in (((37, 300), quantize_float8_rows, 1), ((200, 333), quantize_float8_weight, 128)):
        blocks = make(normal(*shape))
        want = stands_for(*blocks, tall).float().to(dtype)
        assert torch.equal(dequantize_float8(blocks, dtype), want)
    x = normal(2, 3, 5, 40)
    assert dequantize_float8(quantize_float8_rows(x), dtype).shape == x.shape
    rows = quantize_float8_rows(normal(9, 256))
    strided = Float8Blocks(rows.q[::2], rows.scale[::2])  # every other row, scales two apart
    assert torch.equal(dequantize_float8(strided, dtype), dequantize_float8(rows, dtype)[::2])


def test_blocks_of_zeros_tiny_and_largest_values():
    x = torch.zeros(6, 300, device="cuda")
    x[1, 3] = 1e-40
    x[2] = torch.finfo(torch.float32).max
    x[3, 0] = -torch.finfo(torch.float32).max
    x[4, 5] = 2.0**-59
    x[5, 130] = 2.0**-61  # under the floor: half of the top value
    q, scale = quantize_float8_rows(x)
    want_q, want_scale = blocks_by_definition(x, 1)
    assert same_values(q, want_q) and torch.equal(scale, want_scale)
    assert bool((q[0].float() == 0).all()) and bool((q[2].float() == 448).all()) and float(q[5, 130]) == 224


@pytest.mark.parametrize("make", [quantize_float8_rows, quantize_float8_weight])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_a_block_with_an_infinity_or_nan_reads_back_as_nan(bad, make):
    x = normal(130, 300)
    x[1, 140] = bad
    blocks = make(x)
    back = dequantize_float8(blocks)
    tall = 1 if make is quantize_float8_rows else 128
    hit = torch.zeros_like(back, dtype=torch.bool)
    hit[(slice(1, 2) if tall == 1 else slice(0, 128)), 128:256] = True
    assert bool(back[hit].isnan().all()) and bool(back[~hit].isfinite().all()) and bool((blocks.q[hit].float() == 0).all())


# ---- the layer for serving ----------------------------------------------------------------------------------


def served(rows, d, n, dtype, seed=0):
    x = (normal(rows, d, seed=seed) * torch.exp(normal(rows, 1, seed=seed + 1))).to(dtype)
    return x, quantize_float8_weight(normal(n, d, seed=seed + 2) * d**-0.5 * torch.exp(normal(n, 1, seed=seed + 3)))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(
    "rows,d,n",
    [(1, 1, 1), (1, 128, 128), (1, 4096, 4096), (1, 1000, 777), (2, 129, 3), (7, 300, 640), (16, 2048, 256), (17, 520, 1111), (33, 4096, 130),
     (64, 256, 512), (65, 4097, 257), (100, 1280, 1000), (128, 16, 16), (129, 640, 384), (300, 256, 512), (1023, 2500, 1111), (1000, 127, 4000),
     (520, 8192, 260), (2048, 1024, 1024), (1, 16384, 300), (130, 100, 16384)],
)  # fmt: skip
def test_linear(rows, d, n, dtype):
    x, w = served(rows, d, n, dtype)
    bias = normal(n, seed=9, dtype=dtype)
    xs, ws = stands_for(*blocks_by_definition(x, 1), 1), stands_for(*w, 128)
    assert_linear(float8_linear(x, w), xs, ws)
    y = float8_linear(x, w, bias)
    assert_linear(y, xs, ws, bias)
    # the same through blocks made before, and bit for bit again
    assert torch.equal(float8_linear(quantize_float8_rows(x), w, bias, dtype=dtype), y)
    assert torch.equal(float8_linear(x, w, bias), y)
    assert _lib.lib().th_linear_tc_status() == 0


@pytest.mark.parametrize("rows", [1, 5, 40, 300])
def test_scales_of_any_layout_and_size(rows):
    d, n = 700, 300
    x, w = served(rows, d, n, torch.float32)
    held = quantize_float8_rows(x)
    # rows' scales lying row by row, a weight's transposed, and scales far from one that meet
    moved = Float8Blocks(held.q, held.scale.contiguous() * 2.0**70)
    turned = Float8Blocks(w.q, (w.scale * 2.0**-70).t().contiguous().t())
    want = float8_linear(held, w, dtype=torch.float32)
    assert torch.equal(float8_linear(moved, turned, dtype=torch.float32), want)
    # the product of these scales is no float32; the results are
    vast, small = Float8Blocks(held.q, held.scale * 2.0**100), Float8Blocks(w.q, w.scale * 2.0**60)
    q = vast._replace(q=(held.q.float() * 0).to(torch.float8_e4m3fn))
    assert bool((float8_linear(q, small, dtype=torch.float32) == 0).all())
    tiny = Float8Blocks(held.q, held.scale * 2.0**-80), Float8Blocks(w.q, w.scale * 2.0**-56)
    got = float8_linear(*tiny, dtype=torch.float32).double() * 2.0**136
    reach = stands_for(*held, 1).abs() @ stands_for(*w, 128).abs().t()
    # near the smallest float32 (a step of 2^-149, 2^-13 here) each of the six blocks' sums is rounded three times at most, by half a step
    assert bool(((got - want.double()).abs() <= 2.0**-15 * reach + 18 * 2.0**-14).all())


@pytest.mark.parametrize("rows", [1, 3, 200])
def test_a_nan_reaches_its_row_only(rows):
    x, w = served(rows, 300, 140, torch.bfloat16)
    clean = float8_linear(x, w)
    x[rows // 2, 131] = float("inf")
    y = float8_linear(x, w)
    keep = torch.arange(rows, device="cuda") != rows // 2
    assert bool(y[rows // 2].isnan().all()) and torch.equal(y[keep], clean[keep])


def test_strided_inputs_leading_dimensions_and_types():
    x, w = served(12, 200, 96, torch.float16)
    y = float8_linear(x, w)
    assert torch.equal(float8_linear(x.view(3, 4, 200), w), y.view(3, 4, 96))
    assert torch.equal(float8_linear(x[3], w), y[3])
    big = normal(12, 411, dtype=torch.float16)
    assert torch.equal(float8_linear(big[:, 5:205], w), float8_linear(big[:, 5:205].contiguous(), w))
    assert torch.equal(float8_linear(big.t()[:200].t(), w), float8_linear(big[:, :200].contiguous(), w))
    assert torch.equal(float8_linear(x[:1].expand(12, -1), w), y[:1].expand(12, -1))
    assert float8_linear(x, w, dtype=torch.float32).dtype == torch.float32
    assert float8_linear(x[:0], w).shape == (0, 96)
    shifted = torch.empty(96 * 208 + 1, device="cuda").to(torch.float8_e4m3fn)[1:].view(96, 208)[:, :200].copy_(w.q)  # rows off 16 bytes
    assert torch.equal(float8_linear(x, Float8Blocks(shifted, w.scale)), y)


def test_outputs_end_where_they_should():
    x, w = served(150, 260, 333, torch.float16)
    held = quantize_float8_rows(x)
    for dtype in DTYPES:
        out = torch.full((160, 400), 7.0, device="cuda", dtype=dtype)
        lib, code = _lib.lib(), _lib.DTYPE_CODE[dtype]
        _lib.check(
            lib.th_float8_linear(
                held.q.data_ptr(), held.q.stride(0), held.scale.data_ptr(), *held.scale.stride(), w.q.data_ptr(), w.q.stride(0), w.scale.data_ptr(),
                *w.scale.stride(), None, out.data_ptr(), 400, 150, 260, 333, code, _lib.stream_ptr(out.device),
            ),
            "th_float8_linear",
        )  # fmt: skip
        assert torch.equal(out[:150, :333], float8_linear(held, w, dtype=dtype))
        assert bool((out[150:] == 7).all()) and bool((out[:, 333:] == 7).all())


def test_another_stream_and_a_captured_graph():
    x, w = served(5, 512, 256, torch.bfloat16)
    want = float8_linear(x, w)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        got = float8_linear(x, w)
    torch.cuda.current_stream().wait_stream(other)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = float8_linear(x, w)
    x.copy_(normal(5, 512, seed=4, dtype=torch.bfloat16))
    graph.replay()
    assert torch.equal(y, float8_linear(x, w))


def test_module():
    linear = torch.nn.Linear(300, 70, device="cuda", dtype=torch.bfloat16)
    layer = Float8Linear.from_linear(linear)
    x = normal(4, 300, dtype=torch.bfloat16)
    y = layer(x)
    assert torch.equal(y, float8_linear(x, quantize_float8_weight(linear.weight.detach()), linear.bias.detach()))
    other = Float8Linear.from_linear(torch.nn.Linear(300, 70, device="cuda", dtype=torch.bfloat16))
    other.load_state_dict(layer.state_dict())
    assert torch.equal(other(x), y)
    layer.half()
    assert layer.q.dtype == torch.float8_e4m3fn and layer.scale.dtype == torch.float32 and layer.bias.dtype == torch.float16
    assert torch.equal(layer.cpu().cuda()(x.half()), layer(x.half()))


# ---- training -----------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", SIXTEEN)
@pytest.mark.parametrize(
    "rows,d,n", [(1, 1, 1), (8, 16, 24), (100, 128, 128), (129, 130, 131), (300, 256, 512), (777, 1000, 333), (64, 2048, 40), (2000, 520, 1030)]
)
@pytest.mark.parametrize("with_bias", [False, True])
def test_training_layer_and_its_gradients(rows, d, n, dtype, with_bias):
    x = (normal(rows, d) * torch.exp(normal(rows, 1, seed=1))).to(dtype).requires_grad_()
    w = (normal(n, d, seed=2) * d**-0.5).to(dtype).requires_grad_()
    bias = normal(n, seed=3, dtype=dtype).requires_grad_() if with_bias else None
    gy = (normal(rows, n, seed=4) * torch.exp(normal(rows, 1, seed=5))).to(dtype)
    wanted = [t for t in (x, w, bias) if t is not None]
    y = float8_training_linear(x, w, bias)
    grads = torch.autograd.grad(y, wanted, gy, retain_graph=True)
    xs, ws = stands_for(*blocks_by_definition(x.detach(), 1), 1), stands_for(*blocks_by_definition(w.detach(), 128), 128)
    gs = stands_for(*blocks_by_definition(gy, 1), 1)
    assert_linear(y.detach(), xs, ws, None if bias is None else bias.detach())
    assert_linear(grads[0], gs, ws.t().contiguous())
    # dw: 16-bit operands, Q(x) rounded once to their type; float32 sums over the rows, in pieces of 16 at least
    g64 = gy.double()
    exact, reach = g64.t() @ xs, g64.abs().t() @ xs.abs()
    half = torch.finfo(dtype).eps / 2
    tiny = 2.0**-25 if dtype == torch.float16 else 0.0  # a float16 operand or result may be below the normal ones
    allowed = 1.01 * (half + (rows + 2) * 2.0**-23) * reach + 1.01 * half * exact.abs() + tiny * (1 + g64.abs().sum(0)[:, None])
    assert bool(((grads[1].double() - exact).abs() <= allowed).all())
    if with_bias:
        total = g64.sum(0)
        allowed = 1.01 * ((rows + 2) * 2.0**-24 * g64.abs().sum(0) + half * total.abs()) + tiny
        assert bool(((grads[2].double() - total).abs() <= allowed).all())
    again = torch.autograd.grad(y, wanted, gy)
    assert all(torch.equal(a, b) for a, b in zip(again, grads))
    assert _lib.lib().th_linear_tc_status() == 0


@pytest.mark.parametrize("dtype", SIXTEEN)
def test_gradients_against_differences(dtype):
    # values that 8-bit blocks hold as they are (multiples of 2^-4 up to 14 of them, the largest in every block), so that the layer is linear
    # in each of its inputs; results are whole multiples of 2^-8 of which float32 and, here, the sums of float64 lose nothing
    rows, d, n = 32, 256, 128

    def grid(*shape, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        t = torch.randint(-6, 7, shape, device="cuda", generator=g).float()
        t[:, ::128] = 14.0
        return t / 16

    def step(like, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        t = torch.randint(-1, 2, like.shape, device="cuda", generator=g).float()
        t[:, ::128] = 0
        return t / 16

    x, w, gy = grid(rows, d, seed=0), grid(n, d, seed=1), grid(rows, n, seed=2)
    xg, wg = x.to(dtype).requires_grad_(), w.to(dtype).requires_grad_()
    dx, dw = torch.autograd.grad(float8_training_linear(xg, wg), (xg, wg), gy.to(dtype))

    def loss(x, w):
        with torch.no_grad():
            y = float8_linear(quantize_float8_rows(x), quantize_float8_weight(w), dtype=torch.float32)
            return float((y.double() * gy.double()).sum())

    half = torch.finfo(dtype).eps / 2
    hx, hw = step(x, 3), step(w, 4)
    for got, difference, h in ((dx, loss(x + hx, w) - loss(x - hx, w), hx), (dw, loss(x, w + hw) - loss(x, w - hw), hw)):
        along = float((got.double() * h.double()).sum())
        # each gradient was rounded to its 16-bit type
        assert abs(along - difference / 2) <= 1.01 * half * float((got.double() * h.double()).abs().sum()) + 1e-9


def test_training_layer_frozen_parts_autocast_and_module():
    layer = Float8TrainingLinear(130, 70, device="cuda", dtype=torch.bfloat16)
    x = normal(3, 50, 130, dtype=torch.bfloat16).requires_grad_()
    y = layer(x)
    y.sum().backward()  # an expanded gradient
    assert y.shape == (3, 50, 70) and x.grad.shape == x.shape and layer.weight.grad.shape == layer.weight.shape and layer.bias.grad.shape == (70,)
    full = x.grad, layer.weight.grad
    frozen = layer.weight.detach()
    (dx,) = torch.autograd.grad(float8_training_linear(x, frozen, None).sum(), x)
    assert torch.equal(dx, full[0])
    (dw,) = torch.autograd.grad(float8_training_linear(x.detach(), layer.weight, None).sum(), layer.weight)
    assert torch.equal(dw, full[1])
    wide = Float8TrainingLinear(130, 70, device="cuda")
    with torch.autocast("cuda", torch.bfloat16):
        z = wide(x.float())
    assert z.dtype == torch.bfloat16
    z.sum().backward()
    assert wide.weight.grad.dtype == torch.float32
    assert torch.equal(z, float8_training_linear(x, wide.weight.bfloat16(), wide.bias.bfloat16()))
    empty = x.detach()[:0].requires_grad_()
    out = layer(empty)
    assert out.shape == (0, 50, 70)
    layer.zero_grad()
    out.sum().backward()
    assert bool((layer.weight.grad == 0).all()) and empty.grad.shape == empty.shape


def test_python_and_native_paths_agree():
    x, w, b = normal(90, 200, dtype=torch.float16).requires_grad_(), normal(60, 200, seed=1, dtype=torch.float16).requires_grad_(), normal(60, seed=2, dtype=torch.float16).requires_grad_()
    gy = normal(90, 60, seed=3, dtype=torch.float16)
    run = lambda: [y := float8_training_linear(x, w, b), *torch.autograd.grad(y, (x, w, b), gy)]  # noqa: E731,F841
    first = run()
    with _lib.KernelTimer():  # leaves the calls to Python
        second = run()
    assert all(torch.equal(p, q) for p, q in zip(first, second))
    blocks = quantize_float8_weight(w.detach())
    with torch.no_grad():
        one = float8_linear(x, blocks, b)
        with _lib.KernelTimer():
            assert torch.equal(float8_linear(x, blocks, b), one)


def test_second_derivatives_raise():
    x = normal(4, 130, dtype=torch.float16).requires_grad_()
    w = normal(9, 130, seed=1, dtype=torch.float16).requires_grad_()
    (dx,) = torch.autograd.grad(float8_training_linear(x, w).float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="not differentiable twice"):
        dx.float().sum().backward()


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("rows, n", [(33, 130), (1, 77), (40, 128), (150, 1)])
def test_output_gradients_of_any_layout(rows, n, native):
    # rows that start off 16 bytes, that are strided or shared: blocks and the 16-bit rows of the weight's product come out as those of a plain tensor
    dtype = torch.bfloat16
    x = normal(rows, 200, dtype=dtype, seed=3).requires_grad_()
    w = normal(n, 200, dtype=dtype, seed=4).requires_grad_()
    b = normal(n, dtype=dtype, seed=5).requires_grad_()
    big = normal(2 * rows, n + 8, dtype=dtype, seed=6)
    with nullcontext() if native else _lib.KernelTimer():
        for gy in (big[:rows, 3 : 3 + n], big[::2, 8:], big[:rows, :n], big[1:2, :n].expand(rows, -1), big[:rows, 1 : 1 + n].contiguous()):
            plain = torch.zeros(rows, -(-n // 8) * 8, dtype=dtype, device="cuda")
            plain[:, :n] = gy
            out = [torch.autograd.grad(float8_training_linear(x, w, b), (x, w, b), g) for g in (gy, plain[:, :n])]
            assert all(torch.equal(got, want) for got, want in zip(*out))
            (dw,) = torch.autograd.grad(float8_training_linear(x.detach(), w, None), w, gy)
            assert torch.equal(dw, out[0][1])
