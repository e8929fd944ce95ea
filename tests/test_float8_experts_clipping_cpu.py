r"""8-bit floating-point layers, layers of experts and clipping where no GPU is needed: argument errors of the C entry points and of the
Python functions."""
import ctypes

import pytest
import torch

from triton_helpers_b200 import _lib, build
from triton_helpers_b200.layers.expert_linear import ExpertLinear, expert_linear
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
from triton_helpers_b200.optim import FusedAdam, clip_grad_norm_, clipped_adam_updates, grad_norm

AT = 1 << 20  # an aligned address that no call here gets to read


@pytest.fixture(scope="module")
def library():
    if not _lib.LIB_PATH.exists():
        build.build()
    return _lib.lib()


def said(library, text):
    return text in library.th_last_error_string()


def test_block_entry_points_refuse(library):
    rows = library.th_float8_rows
    assert rows(AT, 8, AT, 16, AT, 4, -1, 8, 0, None) == -1
    assert rows(AT, 8, AT, 16, AT, 4, 4, 0, 0, None) == -1
    assert rows(AT, 8, AT, 16, AT, 4, 4, 8, 3, None) == -2 and said(library, b"dtype")
    assert rows(None, 8, AT, 16, AT, 4, 4, 8, 0, None) == -1 and said(library, b"null")
    assert rows(AT, 8, AT + 8, 16, AT, 4, 4, 8, 0, None) == -3 and said(library, b"16 bytes")
    assert rows(AT, 40, AT, 32, AT, 4, 4, 40, 0, None) == -3
    assert rows(AT + 1, 8, AT, 16, AT, 4, 4, 8, 1, None) == -3
    assert rows(AT, 8, AT, 16, AT + 2, 4, 4, 8, 1, None) == -3
    assert rows(AT, 8, AT, 16, AT, 3, 4, 8, 1, None) == -1 and said(library, b"scales")
    assert rows(AT, 8, AT, 1 << 25, AT, 4, 4, (1 << 24) + 1, 0, None) == -2
    assert rows(None, 8, None, 16, None, 0, 0, 8, 0, None) == 0
    copied = lambda copy=AT, stride=8, dtype=1: library.th_float8_rows_copied(AT, 8, AT, 16, AT, 4, copy, stride, 4, 8, dtype, None)  # noqa: E731
    assert copied(dtype=0) == -2 and copied(copy=None) == -1 and copied(stride=7) == -1 and copied(stride=12) == -3 and copied(copy=AT + 2) == -3
    weight = library.th_float8_weight
    assert weight(AT, 8, AT, 24, AT, 4, 8, 0, None) == -3
    assert weight(AT, 8, AT, 16, AT, 65535 * 128 + 1, 8, 0, None) == -2
    values = library.th_float8_values
    assert values(AT, 16, AT, 1, 4, 64, AT, 8, 4, 8, 0, None) == -1 and said(library, b"64 rows")
    assert values(AT, 16, AT, 1, 4, 1, AT, 7, 4, 8, 0, None) == -1
    assert values(AT, 16, AT, -1, 4, 1, AT, 8, 4, 8, 0, None) == -1


def test_float8_products_refuse(library):
    def linear(q=AT, qs=16, s=AT, w=AT, ws=16, w_s=AT, bias=None, y=AT, ys=8, rows=4, d=16, n=8, dtype=0, s_row=1, ws_row=1):
        return library.th_float8_linear(q, qs, s, s_row, 4, w, ws, w_s, ws_row, 1, bias, y, ys, rows, d, n, dtype, None)

    assert linear(rows=-1) == -1 and linear(d=0) == -1 and linear(n=0) == -1
    assert linear(dtype=5) == -2 and linear(rows=(1 << 30) + 1) == -2
    assert linear(q=None) == -1 and linear(s=None) == -1 and linear(w=None) == -1 and linear(w_s=None) == -1 and linear(y=None) == -1
    assert linear(s_row=-1) == -1 and linear(ws_row=-2) == -1
    assert linear(qs=24) == -3 and linear(q=AT + 4) == -3 and linear(ws=8) == -3 and linear(w=AT + 1) == -3
    assert linear(ys=7) == -1 and linear(y=AT + 2) == -3 and linear(bias=AT + 1) == -3 and linear(s=AT + 1) == -3
    assert linear(rows=0, q=None) == 0
    size = library.th_float8_quantized_linear_workspace_bytes
    assert size(0, 8) == 0 and size(3, 130) >= 3 * (144 + 8)
    quantized = lambda ws, n: library.th_float8_quantized_linear(AT, 16, 0, AT, 16, AT, 1, 1, None, AT, 8, ws, n, 4, 16, 8, 0, None)  # noqa: E731
    assert quantized(None, 1 << 20) == -4 and quantized(AT, 16) == -4 and quantized(AT + 8, 1 << 20) == -4
    back = lambda gs=16, ws=16, xs=16: library.th_float8_bwd_input(AT, gs, AT, 1, 4, AT, ws, AT, 1, 1, AT, xs, 4, 16, 8, 1, None)  # noqa: E731
    assert back(gs=0) == -3 and back(ws=8) == -3 and back(xs=15) == -1


def test_expert_entry_points_refuse(library):
    def fwd(x=AT, xs=16, w=AT, ws=16, we=128, ends=AT, y=AT, ys=8, rows=4, experts=2, d=16, n=8, dtype=1):
        return library.th_expert_linear_fwd(x, xs, w, ws, we, ends, y, ys, rows, experts, d, n, dtype, None)

    assert fwd(rows=-1) == -1 and fwd(experts=0) == -1 and fwd(d=0) == -1
    assert fwd(experts=1025) == -2 and fwd(dtype=0) == -2 and said(library, b"float16") and fwd(rows=(1 << 30) + 1) == -2
    assert fwd(x=None) == -1 and fwd(w=None) == -1 and fwd(ends=None) == -1 and fwd(y=None) == -1
    assert fwd(xs=15) == -1 and fwd(xs=20) == -3 and fwd(x=AT + 8) == -3 and fwd(ws=17) == -3 and fwd(we=132) == -3
    assert fwd(we=64) == -1 and said(library, b"overlap") and fwd(ys=7) == -1 and fwd(y=AT + 1) == -3 and fwd(ends=AT + 2) == -3
    assert fwd(rows=0, x=None, w=None) == 0
    back = lambda gs=8, xs=16: library.th_expert_linear_bwd_input(AT, gs, AT, 16, 128, AT, AT, xs, 4, 2, 16, 8, 1, None)  # noqa: E731
    assert back(gs=7) == -1 and back(xs=15) == -1
    weight = lambda g=AT, x=AT, dw=AT, xs=16: library.th_expert_linear_bwd_weight(g, 8, x, xs, AT, dw, 4, 2, 16, 8, 1, None)  # noqa: E731
    assert weight(g=None) == -1 and weight(x=AT + 4) == -3 and weight(dw=None) == -1 and weight(xs=9) == -1


def test_norm_entry_points_refuse(library):
    pointers = lambda *p: (ctypes.c_void_p * len(p))(*p)  # noqa: E731
    sizes, codes, ones = _lib.i64_array([8, 0]), (ctypes.c_int * 2)(0, 1), (ctypes.c_float * 2)(1, 1)
    size = library.th_grad_norm_workspace_bytes
    assert size(0, None) == 0 and size(2, sizes) == 8 and size(1, _lib.i64_array([2**30])) < 2**16
    norm = lambda p, c=codes, pair=AT, ws=AT, n=64: library.th_grad_norm(2, p, sizes, c, None, 1.0, pair, ws, n, None)  # noqa: E731
    assert norm(pointers(None, None)) == -1 and norm(pointers(AT + 2, None)) == -3 and norm(pointers(AT, None), pair=None) == -1
    assert norm(pointers(AT, None), (ctypes.c_int * 2)(0, 7)) == -2
    assert norm(pointers(AT, None), ws=None) == -4 and norm(pointers(AT, None), n=7) == -4 and norm(pointers(AT, None), ws=AT + 4) == -4
    assert library.th_grad_norm(-1, None, None, None, None, 1.0, AT, None, 0, None) == -1
    assert library.th_scale_tensors(2, pointers(AT, None), sizes, codes, None, None) == -1
    assert library.th_scale_tensors(2, pointers(None, None), sizes, codes, AT, None) == -1
    flags = (ctypes.c_int * 2)(0, 0)
    adam = lambda p=AT, m=AT, step=1, dtype=0, pair=AT: library.th_adam_clipped(  # noqa: E731
        2, pointers(p, None), pointers(AT, None), pointers(m, None), pointers(AT, None), sizes, ones, flags, pair, 1e-3, 0.9, 0.99, 1e-8, step, dtype, None, None
    )
    assert adam(p=None) == -1 and adam(step=0) == -1 and adam(dtype=3) == -2 and adam(pair=None) == -1 and adam(m=AT + 2) == -3


def blocks(n, k, tall=1):
    return Float8Blocks(torch.zeros(n, k).to(torch.float8_e4m3fn), torch.ones(-(-n // tall), -(-k // 128)))


def test_float8_functions_refuse():
    x, w = torch.zeros(4, 300), blocks(200, 300, 128)
    with pytest.raises(AssertionError, match="same device"):
        float8_linear(x, w)
    with pytest.raises(AssertionError, match="dimension"):
        float8_linear(x[:, :200], w)
    with pytest.raises(AssertionError, match="128 x 128"):
        float8_linear(x, blocks(200, 300))
    with pytest.raises(AssertionError, match="each 128 columns"):
        float8_linear(w, w, dtype=torch.float16)
    with pytest.raises(AssertionError, match="Bias"):
        float8_linear(x, w, torch.zeros(300))
    with pytest.raises(TypeError, match="result's type"):
        float8_linear(x, w, torch.zeros(200).half())
    with pytest.raises(TypeError, match="pass dtype"):
        float8_linear(blocks(4, 300), w)
    with pytest.raises(TypeError, match="x must be"):
        float8_linear(x.double(), w)
    with pytest.raises(TypeError, match="the result"):
        float8_linear(x, w, dtype=torch.float64)
    with pytest.raises(TypeError, match="float8_e4m3fn"):
        float8_linear(x, w._replace(q=w.q.to(torch.float8_e5m2)))
    with pytest.raises(TypeError, match="float32 scales"):
        float8_linear(x, w._replace(scale=w.scale.half()))
    with pytest.raises(RuntimeError, match="no gradient"):
        float8_linear(x.requires_grad_(), w)
    for make in (quantize_float8_rows, quantize_float8_weight):
        with pytest.raises(RuntimeError, match="no gradient"):
            make(torch.zeros(3, 4, requires_grad=True))
        with pytest.raises(TypeError, match="float16"):
            make(torch.zeros(3, 4).double())
        with pytest.raises(AssertionError):
            make(torch.zeros(3, 0))
        with pytest.raises(AssertionError, match="same device"):
            make(torch.zeros(3, 4))
    with pytest.raises(AssertionError, match="matrix"):
        quantize_float8_weight(torch.zeros(3, 4, 5))
    with pytest.raises(AssertionError):
        dequantize_float8(Float8Blocks(w.q, w.scale[:1]))
    with pytest.raises(AssertionError):
        Float8Linear(w, torch.zeros(3))


def test_float8_training_refuses():
    x, w = torch.zeros(4, 300).half(), torch.zeros(200, 300).half()
    with pytest.raises(AssertionError, match="same device"):
        float8_training_linear(x, w)
    with pytest.raises(TypeError, match="one dtype"):
        float8_training_linear(x, w.bfloat16())
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        float8_training_linear(x.float(), w.float())
    with pytest.raises(AssertionError, match="dimension"):
        float8_training_linear(x[:, 1:], w)
    with pytest.raises(AssertionError, match="Bias"):
        float8_training_linear(x, w, x[0])
    layer = Float8TrainingLinear(7, 9)
    assert set(layer.state_dict()) == {"weight", "bias"}


def test_expert_functions_refuse():
    x, w, ends = torch.zeros(6, 40).half(), torch.zeros(3, 24, 40).half(), torch.tensor([1, 2, 6])
    with pytest.raises(AssertionError, match="same device"):
        expert_linear(x, w, ends)
    with pytest.raises(AssertionError, match="one end"):
        expert_linear(x, w, ends[:2])
    with pytest.raises(TypeError, match="int32 or int64"):
        expert_linear(x, w, ends.float())
    with pytest.raises(TypeError, match="one dtype"):
        expert_linear(x, w.bfloat16(), ends)
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        expert_linear(x.float(), w.float(), ends)
    with pytest.raises(AssertionError, match="dimension"):
        expert_linear(x[:, 1:], w, ends)
    with pytest.raises(AssertionError, match="experts, out, in"):
        expert_linear(x, w[0], ends)
    with pytest.raises(AssertionError, match="at most"):
        expert_linear(x, w[:1, :1].expand(1025, 1, 40), torch.zeros(1025, dtype=torch.int32))
    with pytest.raises(AssertionError):
        ExpertLinear(0, 4, 4)
    layer = ExpertLinear(3, 16, 8)
    assert layer.weight.shape == (3, 8, 16) and float(layer.weight.detach().abs().max()) <= 0.25


def test_clipping_refuses():
    p = torch.zeros(4, requires_grad=True)
    p.grad = torch.ones(4)
    with pytest.raises(ValueError, match="negative"):
        clip_grad_norm_([p], -1.0)
    with pytest.raises(ValueError, match="negative"):
        clip_grad_norm_([p], float("nan"))
    with pytest.raises(AssertionError, match="same device"):
        clip_grad_norm_([p], 1.0)
    with pytest.raises(AssertionError, match="same device"):
        grad_norm([torch.ones(3)])
    with pytest.raises(ValueError, match="no tensors"):
        grad_norm([])
    with pytest.raises(ValueError, match="scales"):
        grad_norm([torch.ones(3)], [1.0, 2.0])
    with pytest.raises(TypeError, match="dtype"):
        grad_norm([torch.ones(3).double()])
    with pytest.raises(TypeError, match="dense"):
        grad_norm([torch.ones(3).to_sparse()])
    with pytest.raises(ValueError, match="as many"):
        clipped_adam_updates([p], [], [p], [p], 1.0, 1, 1e-3, (0.9, 0.99), 1e-8)
    with pytest.raises(ValueError, match="negative"):
        FusedAdam([p]).step(max_norm=-2.0)
    assert float(clip_grad_norm_([torch.zeros(3, requires_grad=True)], 1.0)) == 0
