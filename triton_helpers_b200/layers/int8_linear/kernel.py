r"""Linear layers on 8-bit integers, and the 8-bit rows they take, on hand-written sm_100a kernels.

There is no such operator in triton_helpers; this module follows the conventions of its fused MLP
(``triton_helpers/layers/fully_fused_mlp/kernel.py:640-686``): a functional entry point, assertions on shapes,
``TypeError`` for types, weights as ``(out, in)``.

8-bit rows hold a matrix as signed integers with one float32 scale per row::

    a = max(max_k |x_k|, 2^-100)      q_k = rint(x_k * (127 / a))      scale = a / 127        (float32)

A row that holds an infinity or a NaN has zeros and the scale NaN, so it reads back as NaN throughout.  With one scale per
token and one per output channel a linear layer is an integer product and a factor per output::

    y[t, n] = scale[t] * weight.scale[n] * sum_k q[t, k] * weight.q[n, k] + bias[n]

The sums are exact in 32 bits (up to 131071 inputs) and rounded once, to the type of the result.
"""
from functools import wraps
from typing import Callable, List, NamedTuple, Optional, Union

import torch
from torch import Tensor
from torch.autograd import Function, forward_ad

from ... import _lib

MAX_INPUTS = 131071  # 128 * 128 * 131071 < 2^31


class Int8Rows(NamedTuple):
    r"""``q``: int8 ``(..., K)``, laid out by ``quantize_rows`` with rows that start on 16 bytes; ``scale``: float32 ``(...)``."""

    q: Tensor
    scale: Tensor


def float_dtype(t: Tensor, what: str) -> torch.dtype:
    if t.dtype not in (torch.float16, torch.bfloat16, torch.float32):
        raise TypeError(f"{what} must be float16, bfloat16 or float32, got {t.dtype}")
    return t.dtype


def refuse_gradients(what: str, *tensors: Optional[Tensor]) -> None:
    given = [t for t in tensors if t is not None]
    if torch.is_grad_enabled() and any(t.requires_grad for t in given):
        raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad() or on detached tensors")
    # a tangent is carried without regard to no_grad
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in given):
        raise RuntimeError(f"{what} has no gradient: its inputs must not have tangents")


class _Once(Function):
    r"""A gradient as it is, with a history on the way to ``reach`` that raises."""

    @staticmethod
    def forward(ctx, what: str, grad: Tensor, *reach: Tensor) -> Tensor:
        ctx.what = what
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError(f"{ctx.what} is not differentiable twice")


def _leaves(ctx) -> List[Tensor]:
    r"""The leaves that a node's inputs come from."""
    nodes, seen, leaves = [ctx], set(), []
    while nodes:
        for node, _ in nodes.pop().next_functions:
            if node is None or node in seen:
                continue
            seen.add(node)
            if hasattr(node, "variable"):
                leaves.append(node.variable)
            else:
                nodes.append(node)
    return leaves


def first_order(what: str) -> Callable:
    r"""For a backward pass of kernels: gradients that are to be differentiated themselves (``create_graph``) raise where that happens,
    whatever the loss is made of besides.  ``once_differentiable`` lets them pass as constants where the incoming gradient is one."""

    def decorate(backward: Callable) -> Callable:
        @wraps(backward)
        def wrapper(ctx, *grads: Optional[Tensor]):
            with torch.no_grad():
                out = backward(ctx, *grads)
            if not torch.is_grad_enabled():
                return out
            reach = [t for t in (*grads, *ctx.saved_tensors) if t is not None and t.requires_grad] + _leaves(ctx)
            passed = lambda t: t is None or any(t is g for g in grads)  # noqa: E731  an incoming gradient handed on keeps its own history
            return tuple(t if passed(t) else _Once.apply(what, t.detach().requires_grad_(), *reach) for t in out)

        return wrapper

    return decorate


def rows2d(t: Tensor, width: int) -> Tensor:
    r"""``t`` as rows of ``width`` elements with unit stride inside a row; a copy only where the strides ask for it."""
    t = t.reshape(-1, width)
    return t if t.stride(1) == 1 or width == 1 else t.contiguous()


def row_stride(t: Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def empty_int8_rows(lead, width: int, device: torch.device) -> Int8Rows:
    pitch = -(-width // 16) * 16
    rows = 1
    for n in lead:
        rows *= n
    q = torch.empty((rows, pitch), dtype=torch.int8, device=device)
    return Int8Rows(q[:, :width].view(*lead, width), torch.empty(lead, dtype=torch.float32, device=device))


def int8_rows2d(rows: Int8Rows, what: str) -> Int8Rows:
    r"""Checks 8-bit rows and returns them as a matrix whose rows start on 16 bytes (copied where they do not)."""
    q, scale = rows
    if q.dtype != torch.int8 or scale.dtype != torch.float32:
        raise TypeError(f"{what}: 8-bit rows are int8 with float32 scales, got {q.dtype} and {scale.dtype}")
    assert q.dim() >= 1 and q.shape[-1] >= 1, f"{what}: 8-bit rows need at least one column"
    assert scale.shape == q.shape[:-1], f"{what}: one scale per row: {tuple(scale.shape)} for rows {tuple(q.shape)}"
    width = q.shape[-1]
    q, scale = q.reshape(-1, width), scale.reshape(-1).contiguous()
    if q.numel() and ((width > 1 and q.stride(1) != 1) or q.data_ptr() % 16 or (q.shape[0] > 1 and (q.stride(0) % 16 or q.stride(0) < width))):
        q = empty_int8_rows((q.shape[0],), width, q.device).q.copy_(q)
    return Int8Rows(q, scale)


def int8_stride(q: Tensor) -> int:
    return q.stride(0) if q.shape[0] > 1 else -(-q.shape[1] // 16) * 16


def quantize_rows(x: Tensor) -> Int8Rows:
    r"""8-bit rows of ``x`` (..., K), float16, bfloat16 or float32.  No gradient: an ``x`` that requires one is refused outside of
    ``torch.no_grad()``."""
    refuse_gradients("quantize_rows", x)
    with torch.no_grad():
        return _quantize_rows(x)


def _quantize_rows(x: Tensor) -> Int8Rows:
    assert x.dim() >= 1 and x.shape[-1] >= 1, "8-bit rows need at least one column"
    float_dtype(x, "x")
    device = _lib.require_cuda(x)
    width = x.shape[-1]
    x2d = rows2d(x, width)
    out = empty_int8_rows(x.shape[:-1], width, device)
    with torch.cuda.device(device):
        _lib.check(
            _lib.lib().th_quantize_rows(
                x2d.data_ptr(), row_stride(x2d), out.q.data_ptr(), -(-width // 16) * 16, out.scale.data_ptr(), x2d.shape[0], width,
                _lib.dtype_code(x), _lib.stream_ptr(device),
            ),
            "th_quantize_rows",
        )  # fmt: skip
    return out


def dequantize_rows(rows: Int8Rows, dtype: torch.dtype = torch.float32) -> Tensor:
    r"""``q * scale`` of 8-bit rows, rounded once to ``dtype`` (float16, bfloat16 or float32); contiguous.  No gradient: scales that
    require one are refused outside of ``torch.no_grad()``."""
    refuse_gradients("dequantize_rows", rows.scale)
    with torch.no_grad():
        return _dequantize_rows(rows, dtype)


def _dequantize_rows(rows: Int8Rows, dtype: torch.dtype) -> Tensor:
    lead, width = rows.q.shape[:-1], rows.q.shape[-1]
    q, scale = int8_rows2d(rows, "dequantize_rows")
    device = _lib.require_cuda(q, scale)
    out = torch.empty((*lead, width), dtype=dtype, device=device)
    float_dtype(out, "dtype")
    with torch.cuda.device(device):
        _lib.check(
            _lib.lib().th_dequantize_rows(
                q.data_ptr(), int8_stride(q), scale.data_ptr(), out.data_ptr(), width, q.shape[0], width, _lib.dtype_code(out),
                _lib.stream_ptr(device),
            ),
            "th_dequantize_rows",
        )  # fmt: skip
    return out


def int8_linear(
    x: Union[Tensor, Int8Rows], weight: Int8Rows, bias: Optional[Tensor] = None, dtype: Optional[torch.dtype] = None
) -> Tensor:
    r"""Linear layer with 8-bit weights; a float ``x`` is turned into 8-bit rows on the way.  No gradient.

    Args:
        x: float16, bfloat16 or float32 tensor, or 8-bit rows (of ``quantize_rows`` or ``rms_norm_int8``)
        weight: 8-bit rows of the ``(out, in)`` weight matrix
        bias: of the result's type, or ``None``
        dtype: type of the result; that of ``x`` by default, and required where ``x`` is 8-bit rows

    Shapes:
        - x: :math:`(..., D_{in})`, output: :math:`(..., D_{out})`, bias: :math:`(D_{out},)`
    """
    held = isinstance(x, Int8Rows)
    out = _lib.native().int8_linear(None if held else x, *(x if held else (None, None)), *weight, bias, dtype)
    if out is not NotImplemented:
        return out
    if held:
        if dtype is None:
            raise TypeError("8-bit rows do not say the type of the result: pass dtype")
        refuse_gradients("int8_linear", x.scale, weight.scale, bias)
        rows = x
    else:
        refuse_gradients("int8_linear", x, weight.scale, bias)
        dtype = float_dtype(x, "x") if dtype is None else dtype
        rows = None
    if dtype not in _lib.DTYPE_CODE:
        raise TypeError(f"the result must be float16, bfloat16 or float32, got {dtype}")
    with torch.no_grad():
        assert weight.q.dim() == 2, "the weight is a matrix of 8-bit rows"
        w, w_scale = int8_rows2d(weight, "weight")
        d_out, d_in = w.shape
        lead, width = (x.shape[:-1], x.shape[-1]) if rows is None else (rows.q.shape[:-1], rows.q.shape[-1])
        assert width == d_in, f"Input dimension mismatch: {width} and {d_in}"
        assert d_out >= 1, "the weight needs at least one row"
        assert d_in <= MAX_INPUTS, f"Input dimension {d_in} too large for 32-bit sums"
        assert bias is None or bias.shape == (d_out,), "Bias shape mismatch"
        if bias is not None and bias.dtype != dtype:
            raise TypeError(f"the bias must be of the result's type {dtype}, got {bias.dtype}")
        q, scale = (None, None) if rows is None else int8_rows2d(rows, "x")
        device = _lib.require_cuda(x if rows is None else q, scale, w, w_scale, bias)
        bias = None if bias is None else bias.contiguous()
        y = torch.empty((*lead, d_out), dtype=dtype, device=device)
        lib, code = _lib.lib(), _lib.DTYPE_CODE[dtype]
        with torch.cuda.device(device):
            stream = _lib.stream_ptr(device)
            if rows is None:
                x2d = rows2d(x, d_in)
                ws_bytes = lib.th_quantized_linear_workspace_bytes(x2d.shape[0], d_in)
                workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=device)
                _lib.check(
                    lib.th_quantized_linear(
                        x2d.data_ptr(), row_stride(x2d), _lib.dtype_code(x), w.data_ptr(), int8_stride(w), w_scale.data_ptr(), _lib.ptr(bias),
                        y.data_ptr(), d_out, workspace.data_ptr(), ws_bytes, x2d.shape[0], d_in, d_out, code, stream,
                    ),
                    "th_quantized_linear",
                )  # fmt: skip
            else:
                _lib.check(
                    lib.th_int8_linear(
                        q.data_ptr(), int8_stride(q), scale.data_ptr(), w.data_ptr(), int8_stride(w), w_scale.data_ptr(), _lib.ptr(bias),
                        y.data_ptr(), d_out, q.shape[0], d_in, d_out, code, stream,
                    ),
                    "th_int8_linear",
                )  # fmt: skip
    return y
