r"""8-bit rows and the 8-bit linear layer against a float64 statement of their definition."""
import pytest
import torch

from triton_helpers_b200 import _lib
from triton_helpers_b200.layers.int8_linear import Int8Linear, Int8Rows, dequantize_rows, int8_linear, quantize_rows

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def normal(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def rows_by_definition(x):
    r"""The definition in elementary float32 operations (tensors on both sides of a division: a true one)."""
    x = x.float()
    a = x.abs().amax(-1, keepdim=True).clamp_min(2.0**-100)
    top = torch.full_like(a, 127.0)
    return torch.round(x * (top / a)).to(torch.int8), (a / top).squeeze(-1)


def some_weight(n, k, seed=1):
    return quantize_rows(normal(n, k, seed=seed) * k**-0.5)


def assert_linear(y, rows, weight, bias):
    acc = rows.q.double().reshape(-1, rows.q.shape[-1]) @ weight.q.double().t()
    scaled = acc * rows.scale.double().reshape(-1, 1) * weight.scale.double()
    exact = scaled if bias is None else scaled + bias.double()
    reach = scaled.abs() if bias is None else scaled.abs() + bias.double().abs()
    # four float32 roundings (conversion, product of the scales, product, bias), then the result's own; 2^-25 is float16's smallest half step
    bound = 4.01 * 2.0**-24 * reach + 1.01 * torch.finfo(y.dtype).eps / 2 * exact.abs() + 2.0**-25
    assert y.isfinite().all() and bool(((y.double().reshape(exact.shape) - exact).abs() <= bound).all())


# ---- 8-bit rows ---------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 16), (5, 17), (2, 3, 40), (7, 1000), (4, 1028), (3, 4097), (2, 8192), (1, 70000), (2, 33333)])
def test_rows_are_the_definition_bit_for_bit(shape, dtype):
    x = (normal(*shape) * torch.exp(normal(*shape[:-1], 1, seed=1))).to(dtype)
    q, scale = quantize_rows(x)
    want_q, want_scale = rows_by_definition(x)
    assert q.shape == x.shape and q.dtype == torch.int8 and scale.shape == x.shape[:-1] and scale.dtype == torch.float32
    assert torch.equal(q, want_q) and torch.equal(scale, want_scale)
    assert q.data_ptr() % 16 == 0 and (q.dim() < 2 or q.shape[-2] == 1 or q.stride(-2) % 16 == 0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_back(dtype):
    rows = quantize_rows(normal(37, 123))
    want = (rows.q.float() * rows.scale[:, None]).to(dtype)
    assert torch.equal(dequantize_rows(rows, dtype), want)
    assert torch.equal(dequantize_rows(Int8Rows(rows.q[:, ::2], rows.scale), dtype), want[:, ::2])  # strided columns are copied


def test_rows_of_zeros_tiny_and_largest_values():
    x = torch.zeros(5, 48, device="cuda")
    x[1, 3] = 1e-40  # below the floor: rounds to zero, with a finite factor
    x[2] = torch.finfo(torch.float32).max
    x[3, 0] = -torch.finfo(torch.float32).max
    x[4, 5] = 2.0**-99
    q, scale = quantize_rows(x)
    want_q, want_scale = rows_by_definition(x)
    assert torch.equal(q, want_q) and torch.equal(scale, want_scale)
    assert bool((q[0] == 0).all()) and bool((q[2] == 127).all()) and int(q[3, 0]) == -127 and int(q[4, 5]) == 127


@pytest.mark.parametrize("d", [1, 40, 4097])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_a_row_with_an_infinity_or_nan_reads_back_as_nan(bad, d):
    x = normal(3, d)
    x[1, d // 2] = bad
    rows = quantize_rows(x)
    assert bool((rows.q[1] == 0).all()) and bool(rows.scale[1].isnan())
    back = dequantize_rows(rows)
    assert bool(back[1].isnan().all()) and bool(back[[0, 2]].isfinite().all())


def test_rows_of_other_layouts():
    base = normal(6, 5, 64, dtype=torch.float16)
    for x in (base.transpose(0, 1), base[..., ::2], base[..., 1:], base.permute(2, 0, 1), base[:, :1].expand(6, 3, 64), base[:0]):
        q, scale = quantize_rows(x)
        want_q, want_scale = rows_by_definition(x)
        assert torch.equal(q, want_q) and torch.equal(scale, want_scale)


# ---- linear layer ---------------------------------------------------------------------------------------------


@pytest.mark.parametrize("tokens", [1, 2, 15, 16, 17, 33, 64, 100, 128, 129, 300])
@pytest.mark.parametrize("d_in,d_out", [(16, 16), (128, 128), (100, 77), (1, 1), (1000, 257), (2048, 130)])
def test_linear(tokens, d_in, d_out):
    dtype = DTYPES[(tokens + d_in) % 3]
    x, weight = normal(tokens, d_in, dtype=dtype), some_weight(d_out, d_in)
    bias = normal(d_out, seed=3, dtype=dtype) if tokens % 2 else None
    y = int8_linear(x, weight, bias)
    assert y.dtype == dtype and y.shape == (tokens, d_out)
    assert_linear(y, Int8Rows(*rows_by_definition(x)), weight, bias)


# tiles of two CTAs, partial tiles on every side, many tiles a CTA
@pytest.mark.parametrize("tokens,d_in,d_out", [(2048, 512, 2048), (2100, 640, 1930), (4000, 129, 3000), (2049, 4096, 2049), (8192, 256, 4096)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_of_many_tokens(tokens, d_in, d_out, dtype):
    x, weight, bias = normal(tokens, d_in, dtype=dtype), some_weight(d_out, d_in), normal(d_out, seed=3, dtype=dtype)
    assert_linear(int8_linear(x, weight, bias), Int8Rows(*rows_by_definition(x)), weight, bias)


@pytest.mark.parametrize("tokens,d_in,d_out", [(1, 16384, 64), (3, 20000, 200), (140, 30000, 130), (1, 131071, 16)])
def test_long_sums_are_exact(tokens, d_in, d_out):
    x = torch.full((tokens, d_in), 3.0, device="cuda")  # every integer is 127: sums up to 2^31 - 2^24
    weight = quantize_rows(torch.where(torch.arange(d_out, device="cuda")[:, None] % 2 == 0, 1.0, -1.0).expand(d_out, d_in))
    assert_linear(int8_linear(x, weight), Int8Rows(*rows_by_definition(x)), weight, None)


def test_the_lowest_integer_on_both_sides():
    q = torch.full((2, 131071 // 16 * 16), -128, dtype=torch.int8, device="cuda")
    one = torch.ones(2, device="cuda")
    y = int8_linear(Int8Rows(q, one), Int8Rows(q.clone(), one.clone()), dtype=torch.float32)
    assert bool((y == float(128 * 128 * q.shape[1])).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_as_input_and_leading_dimensions(dtype):
    x, weight = normal(2, 3, 5, 72), some_weight(40, 72)
    rows = quantize_rows(x)
    y = int8_linear(rows, weight, dtype=dtype)
    assert y.shape == (2, 3, 5, 40) and y.dtype == dtype and y.is_contiguous()
    assert_linear(y, rows, weight, None)
    assert torch.equal(int8_linear(x, weight, dtype=dtype), y)
    assert int8_linear(normal(72), weight).shape == (40,)
    assert int8_linear(x[:0], weight).shape == (0, 3, 5, 40)


def test_rows_of_any_layout():
    x, weight = normal(9, 90), some_weight(50, 90)
    rows, want = quantize_rows(x), int8_linear(x, weight)
    packed = Int8Rows(rows.q.contiguous(), rows.scale)  # rows of 90 bytes: copied
    odd = torch.empty(9 * 90 + 1, dtype=torch.int8, device="cuda")[1:].view(9, 90).copy_(rows.q)
    for q in (packed.q, odd, rows.q.t().contiguous().t()):
        assert torch.equal(int8_linear(Int8Rows(q, rows.scale), weight, dtype=torch.float32), want)
    assert torch.equal(int8_linear(x, Int8Rows(weight.q.contiguous(), weight.scale)), want)
    every_other = Int8Rows(weight.q[::2], weight.scale[::2])
    assert torch.equal(int8_linear(x, every_other), want[:, ::2])


def test_a_bad_token_stays_alone():
    x, weight = normal(40, 64), some_weight(48, 64)
    x[7, 1], x[21, 5] = float("nan"), float("inf")
    y = int8_linear(x, weight)
    bad = torch.zeros(40, dtype=torch.bool, device="cuda")
    bad[7] = bad[21] = True
    assert bool(y[bad].isnan().all()) and bool(y[~bad].isfinite().all())


def test_results_repeat_and_memory_behind_is_left():
    x, weight = normal(150, 3000), some_weight(70, 3000)
    first = int8_linear(x, weight)
    assert all(torch.equal(first, int8_linear(x, weight)) for _ in range(5))
    lib, rows = _lib.lib(), quantize_rows(x[:20])
    held = torch.full((22, 80), 7.0, device="cuda")  # rows and columns behind the result stay as they are
    _lib.check(lib.th_int8_linear(rows.q.data_ptr(), rows.q.stride(0), rows.scale.data_ptr(), weight.q.data_ptr(), weight.q.stride(0), weight.scale.data_ptr(),
                                  None, held.data_ptr(), 80, 20, 3000, 70, 0, _lib.stream_ptr(x.device)), "th_int8_linear")  # fmt: skip
    assert bool((held[20:] == 7).all()) and bool((held[:, 70:] == 7).all())
    assert_linear(held[:20, :70], rows, weight, None)


def test_captured_calls_and_another_stream():
    x, weight = normal(5, 2048, dtype=torch.float16), some_weight(512, 2048)
    want = int8_linear(x, weight)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = int8_linear(x, weight)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(on_side, want)
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(int8_linear(x, weight))
    x.copy_(normal(5, 2048, seed=9, dtype=torch.float16))
    want = int8_linear(x, weight)
    for graph in graphs:
        graph.replay()
    assert all(torch.equal(out, want) for out in outs)


def test_module_follows_linear():
    linear = torch.nn.Linear(200, 90).cuda().half()
    layer = Int8Linear.from_linear(linear)
    x = normal(11, 200, dtype=torch.float16)
    y, want = layer(x), torch.nn.functional.linear(x.double(), linear.weight.double(), linear.bias.double()).detach()
    # a half step of 1 / 254 of the row's largest on either side: at most (|x|max |w|sum + |w|max |x|sum + ...) / 254
    wide = x.double().abs().amax(1, keepdim=True) * linear.weight.double().abs().sum(1) + x.double().abs().sum(1, keepdim=True) * linear.weight.double().abs().amax(1)
    assert bool(((y.double() - want).abs() <= 1.01 * wide / 254 + 2.0**-10 * want.abs() + 1e-3).all())
    other = Int8Linear(quantize_rows(torch.zeros(90, 200, device="cuda")), torch.zeros(90, device="cuda").half())
    other.load_state_dict(layer.state_dict())
    assert torch.equal(other(x), y)
    layer.bfloat16()
    assert layer.scale.dtype == torch.float32 and layer.q.dtype == torch.int8 and layer(x.bfloat16()).dtype == torch.bfloat16


def test_refusals():
    x, weight = normal(4, 32), some_weight(8, 32)
    with pytest.raises(AssertionError, match="Input dimension"):
        int8_linear(normal(4, 31), weight)
    with pytest.raises(AssertionError, match="Bias"):
        int8_linear(x, weight, normal(9))
    with pytest.raises(TypeError, match="bias"):
        int8_linear(x, weight, normal(8, dtype=torch.float16))
    with pytest.raises(TypeError, match="dtype"):
        int8_linear(quantize_rows(x), weight)
    with pytest.raises(RuntimeError, match="no gradient"):
        int8_linear(x.clone().requires_grad_(True), weight)
    with pytest.raises(AssertionError, match="same device"):
        int8_linear(x, Int8Rows(weight.q.cpu(), weight.scale.cpu()))
    with pytest.raises(AssertionError, match="32-bit sums"):
        int8_linear(normal(1, 131072), some_weight(1, 131072))
    with pytest.raises(TypeError):
        quantize_rows(x.double())


def test_two_streams_at_once():
    x, weight = [normal(n, 3000, seed=n) for n in (1, 90, 700)], some_weight(500, 3000)
    want = [int8_linear(t, weight) for t in x]
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in x], [[] for _ in x]
    for _ in range(10):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[k].append(int8_linear(x[k], weight))
    torch.cuda.synchronize()
    assert all(torch.equal(y, w) for ys, w in zip(outs, want) for y in ys)


def test_weights_quantised_right_before_their_use():
    # the product may fetch weights while its input is quantised, but not before whatever wrote them has finished
    x = normal(1, 8192, dtype=torch.float16)
    weights = [normal(8192, 8192, seed=k, dtype=torch.float16) for k in range(2)]
    want = [int8_linear(x, quantize_rows(w)) for w in weights]
    torch.cuda.synchronize()
    held = quantize_rows(weights[0])
    for k in (1, 0, 1, 0, 1):
        fresh = quantize_rows(weights[k])
        held.q.copy_(fresh.q)
        held.scale.copy_(fresh.scale)
        assert torch.equal(int8_linear(x, held), want[k])
        assert torch.equal(int8_linear(x, quantize_rows(weights[k])), want[k])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (9, 33), (4, 3001), (2, 70001)])
def test_rows_back_at_odd_widths(shape, dtype):
    rows = quantize_rows(normal(*shape))
    assert torch.equal(dequantize_rows(rows, dtype), (rows.q.float() * rows.scale[:, None]).to(dtype))


def test_offsets_past_32_bits():
    x = normal(1, 64, dtype=torch.float16).expand(1_000_000, 64).contiguous()
    x[-1] = normal(64, seed=5, dtype=torch.float16)
    weight = some_weight(2304, 64)
    y = int8_linear(x, weight)  # 2.3e9 outputs
    assert torch.equal(y[-1], int8_linear(x[-1:], weight)[0]) and torch.equal(y[-2], y[0])


@pytest.mark.parametrize("tokens,d_in,d_out", [(930, 40, 14272), (140, 16, 16000), (3000, 200, 9000)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_tiles_that_lie_outside_in_part(tokens, d_in, d_out, dtype):
    x, weight = normal(tokens, d_in, dtype=dtype), some_weight(d_out, d_in)
    first = int8_linear(x, weight)
    assert_linear(first, Int8Rows(*rows_by_definition(x)), weight, None)
    for _ in range(20):
        assert torch.equal(int8_linear(x, weight), first)
