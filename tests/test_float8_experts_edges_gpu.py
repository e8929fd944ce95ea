r"""8-bit floating-point layers and layers of experts where calls meet: parts of larger matrices, streams, threads, graphs, offsets beyond 32 bits."""
import threading

import pytest
import torch

from triton_helpers_b200 import _lib
from triton_helpers_b200.layers.expert_linear import expert_linear
from triton_helpers_b200.layers.float8_linear import (
    Float8Blocks,
    dequantize_float8,
    float8_linear,
    float8_training_linear,
    quantize_float8_rows,
    quantize_float8_weight,
)
from triton_helpers_b200.optim import FusedAdam, clip_grad_norm_, grad_norm

pytestmark = pytest.mark.gpu


def normal(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def whole(*shape, seed=0, dtype=torch.float16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-2, 3, shape, device="cuda", generator=g).to(dtype)


@pytest.mark.parametrize("n", [333, 330, 328, 136, 5])
@pytest.mark.parametrize("counts", [[40, 0, 90, 15], [3, 0, 9, 2], [300, 20, 0, 1]])
@pytest.mark.parametrize("offset", [0, 1, 8])
def test_experts_into_a_part_of_a_matrix(n, counts, offset):
    d, behind, experts, lib = 72, 7, len(counts), _lib.lib()
    rows, pad = sum(counts) + behind, (n + 7) // 8 * 8
    x, w, gy = whole(rows, d), whole(experts, n, d, seed=1), torch.zeros(rows, pad, device="cuda", dtype=torch.float16)
    gy[:, :n] = whole(rows, n, seed=2)
    ends = torch.tensor(counts, device="cuda").cumsum(0).to(torch.int32)
    stream = _lib.stream_ptr(x.device)
    out = torch.full((rows + 3, 400), 7.0, device="cuda", dtype=torch.float16)
    back = torch.full((rows + 3, 400), 7.0, device="cuda", dtype=torch.float16)
    at = lambda t: t.data_ptr() + 2 * offset  # noqa: E731
    _lib.check(lib.th_expert_linear_fwd(x.data_ptr(), d, w.data_ptr(), d, n * d, ends.data_ptr(), at(out), 400, rows, experts, d, n, 1, stream), "fwd")
    _lib.check(lib.th_expert_linear_bwd_input(gy.data_ptr(), pad, w.data_ptr(), d, n * d, ends.data_ptr(), at(back), 400, rows, experts, d, n, 1, stream), "bwd")
    want, dx = torch.zeros(rows, n, device="cuda", dtype=torch.float64), torch.zeros(rows, d, device="cuda", dtype=torch.float64)
    first = 0
    for e, end in enumerate(ends.tolist()):
        want[first:end] = x[first:end].double() @ w[e].double().t()
        dx[first:end] = gy[first:end, :n].double() @ w[e].double()
        first = end
    for t, value in ((out, want), (back, dx)):
        width = value.shape[1]
        assert torch.equal(t[:rows, offset : offset + width], value.half())  # whole numbers: exact
        assert bool((t[rows:] == 7).all()) and bool((t[:, :offset] == 7).all()) and bool((t[:, offset + width :] == 7).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("rows,n", [(3, 333), (150, 333), (150, 328), (150, 5), (700, 400)])
@pytest.mark.parametrize("offset", [0, 1, 4])
def test_float8_into_a_part_of_a_matrix(rows, n, dtype, offset):
    d, lib, code = 260, _lib.lib(), _lib.DTYPE_CODE[dtype]
    x, w = quantize_float8_rows(normal(rows, d)), quantize_float8_weight(normal(n, d, seed=1))
    out = torch.full((rows + 3, n + 75), 7.0, device="cuda", dtype=dtype)
    _lib.check(
        lib.th_float8_linear(
            x.q.data_ptr(), x.q.stride(0) if rows > 1 else 272, x.scale.data_ptr(), *x.scale.stride(), w.q.data_ptr(), w.q.stride(0), w.scale.data_ptr(),
            *w.scale.stride(), None, out.data_ptr() + offset * out.element_size(), n + 75, rows, d, n, code, _lib.stream_ptr(out.device),
        ),
        "th_float8_linear",
    )  # fmt: skip
    assert torch.equal(out[:rows, offset : offset + n], float8_linear(x, w, dtype=dtype))
    assert bool((out[rows:] == 7).all()) and bool((out[:, :offset] == 7).all()) and bool((out[:, offset + n :] == 7).all())


def test_rows_beside_the_operands_hold_nan():
    # what lies between rows of an operand, or behind them, meets no product
    d, n, counts = 70, 131, [30, 0, 41]
    ends = torch.tensor(counts, device="cuda").cumsum(0).to(torch.int32)
    held = torch.full((80, 80), float("nan"), device="cuda", dtype=torch.float16)
    x = held[:71, :d].copy_(whole(71, d))
    weights = torch.full((3, 140, 72), float("nan"), device="cuda", dtype=torch.float16)
    w = weights[:, :n, :d].copy_(whole(3, n, d, seed=1))
    x, w, gy = x.requires_grad_(), w.requires_grad_(), torch.full((71, 136), float("nan"), device="cuda", dtype=torch.float16)[:, :n].copy_(whole(71, n, seed=2))
    y = expert_linear(x, w, ends)
    dx, dw = torch.autograd.grad(y, (x, w), gy)
    plain = x.detach().clone().requires_grad_(), w.detach().clone().requires_grad_()
    z = expert_linear(*plain, ends)
    assert torch.equal(y, z) and all(torch.equal(a, b) for a, b in zip((dx, dw), torch.autograd.grad(z, plain, gy.clone())))
    assert y.isfinite().all() and dx.isfinite().all() and dw.isfinite().all()
    big = torch.full((40, 400), float("inf"), device="cuda")
    part = big[:33, 40:340].copy_(normal(33, 300))
    blocks = quantize_float8_rows(part)
    want = quantize_float8_rows(part.clone())
    assert torch.equal(blocks.q.float(), want.q.float()) and torch.equal(blocks.scale, want.scale)


def test_streams_side_by_side():
    # pairs of CTAs, single ones and few rows of several streams start beside one another, with deep queues: the bits of a pass alone
    calls = []
    for i, (rows, d, n) in enumerate([(2100, 1024, 1100), (300, 4096, 512), (5, 2048, 2048), (100, 512, 3000)]):
        x, w = normal(rows, d, seed=i, dtype=torch.bfloat16), quantize_float8_weight(normal(n, d, seed=9 + i))
        calls.append(lambda x=x, w=w: float8_linear(x, w))
    for i, (counts, d, n) in enumerate([([700, 0, 1300], 1024, 512), ([3] * 20, 2048, 256), ([90, 100], 512, 2048), ([1, 0, 2], 4096, 4096)]):
        x, w = normal(sum(counts), d, seed=20 + i, dtype=torch.float16), normal(len(counts), n, d, seed=30 + i, dtype=torch.float16)
        ends = torch.tensor(counts, device="cuda").cumsum(0).to(torch.int32)
        calls.append(lambda x=x, w=w, ends=ends: expert_linear(x, w, ends))
    grads = [normal(n, seed=40 + i) for i, n in enumerate((100_000, 33, 4097))]
    calls.append(lambda: grad_norm(grads))
    alone = [call() for call in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for turn in range(40):
        for i, call in enumerate(calls):
            with torch.cuda.stream(streams[(i + turn) % 4]):
                got.append((i, call()))
    torch.cuda.synchronize()
    assert all(torch.equal(t, alone[i]) for i, t in got) and _lib.lib().th_linear_tc_status() == 0


def test_threads_side_by_side():
    x, w = normal(200, 300, dtype=torch.float16).requires_grad_(), normal(130, 300, seed=1, dtype=torch.float16).requires_grad_()
    weights, ends = normal(3, 64, 300, seed=2, dtype=torch.float16).requires_grad_(), torch.tensor([50, 50, 180], device="cuda", dtype=torch.int32)
    gy, ge = normal(200, 130, seed=3, dtype=torch.float16), normal(200, 64, seed=4, dtype=torch.float16)

    def work():
        y, z = float8_training_linear(x, w), expert_linear(x, weights, ends)
        return [y, z, *torch.autograd.grad((y, z), (x, w, weights), (gy, ge))]

    want, found = work(), []

    def loop():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                out = work()
            torch.cuda.current_stream().synchronize()
            found.append(all(torch.equal(a, b) for a, b in zip(out, want)))

    torch.cuda.synchronize()
    threads = [threading.Thread(target=loop) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert found == [True] * 4


def test_two_graphs_of_a_training_step():
    # two captured steps of the same layers, replayed in turn: each has its own scratch, and the second's gradients are not the first's
    w = normal(200, 136, dtype=torch.bfloat16).requires_grad_()
    weights = normal(3, 72, 200, seed=1, dtype=torch.bfloat16).requires_grad_()
    ends = [torch.tensor(e, device="cuda", dtype=torch.int32) for e in ([10, 60, 100], [90, 90, 110])]
    inputs = [normal(120, 136, seed=2 + i, dtype=torch.bfloat16) for i in range(2)]
    gy = normal(120, 72, seed=5, dtype=torch.bfloat16)

    def step(i):
        y = expert_linear(float8_training_linear(inputs[i], w), weights, ends[i])
        grads = torch.autograd.grad(y, (w, weights), gy)
        return [y.detach(), *grads, grad_norm([g.contiguous() for g in grads])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [[t.clone() for t in step(i)] for i in range(2)]
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append(step(i))
        graphs.append(graph)
    for turn in (0, 1, 1, 0, 1):
        graphs[turn].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs[turn], want[turn]))


def test_clipping_on_another_stream_than_the_current_device_default():
    params = [torch.nn.Parameter(normal(1000 + i, seed=i)) for i in range(3)]
    opt = FusedAdam(params, lr=1e-2)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for p in params:
            p.grad = torch.ones_like(p)
        norm = clip_grad_norm_(params, 1.0)
        second = opt.step(max_norm=10.0)
    torch.cuda.current_stream().wait_stream(stream)
    want = (sum(p.numel() for p in params)) ** 0.5
    assert abs(float(norm) / want - 1) < 1e-6 and abs(float(second) - 1) < 1e-5


def test_offsets_beyond_32_bits():
    rows, d, n = 280_000, 8192, 40  # 2.3e9 values in, 4.6 GB of bfloat16
    x = torch.zeros(rows, d, device="cuda", dtype=torch.bfloat16)
    some = torch.tensor([0, 1, 131_071, 262_143, 262_144, rows - 1], device="cuda")
    x[some] = normal(6, d, dtype=torch.bfloat16)
    w = quantize_float8_weight(normal(n, d, seed=1))
    y = float8_linear(x, w)
    assert torch.equal(y[some], float8_linear(x[some].repeat(40, 1), w)[:6])  # 240 rows: tiles of the same kind
    blocks = quantize_float8_rows(x)
    assert torch.equal(blocks.scale[some], quantize_float8_rows(x[some]).scale)
    del blocks
    back = dequantize_float8(Float8Blocks(*quantize_float8_rows(x)), torch.bfloat16)
    assert torch.equal(back[some], dequantize_float8(quantize_float8_rows(x[some]), torch.bfloat16))
    del back
    ends = torch.tensor([131_072, 262_144, rows - 3], device="cuda", dtype=torch.int32)
    weights = normal(3, 16, d, seed=2, dtype=torch.bfloat16)
    z = expert_linear(x, weights, ends)
    for i, e in enumerate((0, 0, 0, 1, 2)):
        want = x[some[i]].double() @ weights[e].double().t()
        assert float((z[some[i]].double() - want).abs().max()) <= 2.0**-7 * float(want.abs().max())
    assert bool((z[rows - 3 :] == 0).all())
    del x, y, z
    # an expert's weights, and their gradients, beyond 2^31 elements
    big = torch.zeros(36, 8192, 8192, device="cuda", dtype=torch.bfloat16)
    big[35] = normal(8192, 8192, seed=3, dtype=torch.bfloat16)
    few, last = normal(5, 8192, seed=4, dtype=torch.bfloat16).requires_grad_(), torch.zeros(36, device="cuda", dtype=torch.int32)
    last[35] = 5
    big.requires_grad_()
    out = expert_linear(few, big, last)
    want = few.detach().double() @ big[35].detach().double().t()
    assert float((out.double() - want).abs().max()) <= 2.0**-7 * float(want.abs().max())
    dx, dw = torch.autograd.grad(out, (few, big), torch.ones_like(out))
    total = few.detach().double().sum(0)
    assert float((dw[35, 8191].double() - total).abs().max()) <= 2.0**-7 * float(total.abs().max()) and not bool(dw[34].any()) and not bool(dw[0].any())


def test_command_lines_run(tmp_path):
    from triton_helpers_b200.benchmark import CLI
    from triton_helpers_b200.layers.expert_linear.__main__ import Baseline, Experts
    from triton_helpers_b200.layers.float8_linear.__main__ import Serving, Training

    flags = ["benchmark", "-m", "fwd", "fwd-bwd", "-w", "2", "-r", "5", "-o", str(tmp_path)]
    charts = CLI.entrypoint("Float8 Linear", [Training("training")], {"L": ((16, 300), "values"), "D": (256, "values"), "N": (128, "values")}, flags)
    assert len(charts) == 2 and all(v > 0 for c in charts for row in c.rows for v in row)
    charts = CLI.entrypoint("Float8 Linear", [Serving("serving")], {"L": ((16, 300), "values"), "D": (256, "values"), "N": (128, "values")},
                            ["benchmark", "-m", "fwd", "-w", "2", "-r", "5"])  # fmt: skip
    assert charts[0].rows[0][0] > 0
    charts = CLI.entrypoint("Expert Linear", [Baseline("baseline"), Experts("experts")],
                            {"L": ((64, 1000), "values"), "E": (4, "values"), "D": (256, "values"), "N": (128, "values")}, flags)  # fmt: skip
    assert len(charts) == 2 and all(v > 0 for c in charts for row in c.rows for v in row)
