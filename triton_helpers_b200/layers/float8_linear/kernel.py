r"""Linear layers on 8-bit floating point with a scale for each block of 128, on hand-written sm_100a kernels.

There is no such operator in triton_helpers; this module follows the conventions of its fused MLP
(``triton_helpers/layers/fully_fused_mlp/kernel.py:640-686``): a functional entry point, assertions on shapes,
``TypeError`` for types, weights as ``(out, in)``.

A block is 128 neighbouring inputs of one row, or of 128 rows of a weight (the last ones may be smaller). It holds e4m3 values
with one float32 scale::

    a = max(max |x|, 2^-60)      q = e4m3(x * (448 / a)), to nearest even      scale = a / 448        (float32)

A block that holds an infinity or a NaN has zeros and the scale NaN, so it reads back as NaN throughout. The products of 8-bit values
are summed in float32 block by block, every block's sum times its two scales::

    y[t, n] = sum_b scale[t, b] * weight.scale[n // 128, b] * sum_{k in b} q[t, k] * weight.q[n, k]  + bias[n]

``float8_linear`` is for serving: weights are turned into blocks once, tokens on the way. ``float8_training_linear`` takes 16-bit
weights and has gradients::

    y = Q(x) Q(w)^T + b          dx = Q(dy) Q(w)          dw = dy^T Q(x)          db = sum over rows of dy

where ``Q`` is what blocks stand for; ``dy`` is cut along the outputs, and a weight's square blocks serve both products. The weight's
gradient is a product in 16 bits, with ``Q(x)`` rounded once more to the layer's type as its operand: its blocks would have to run along
the rows, and one more rounding of ``dy`` and of ``x`` each. Kept for the backward pass are ``Q(x)`` and ``Q(w)``, a little over a byte
a value.
"""
from functools import lru_cache
from typing import Callable, NamedTuple, Optional, Tuple, Union

import torch
from torch import Tensor
from torch.autograd import Function

from ... import _lib
from ..checkpointed_linear.kernel import _empty_operand, _operand, _stride
from ..int8_linear.kernel import first_order, float_dtype, refuse_gradients, row_stride, rows2d

BLOCK = 128


class Float8Blocks(NamedTuple):
    r"""``q``: float8_e4m3fn ``(..., K)``; ``scale``: float32, ``(..., ceil(K / 128))`` for rows and ``(ceil(N / 128), ceil(K / 128))`` for
    a weight ``(N, K)``."""

    q: Tensor
    scale: Tensor


def _count(n: int) -> int:
    return -(-n // BLOCK)


def _pitch(width: int) -> int:
    return -(-width // 16) * 16


def _empty_q(lead, width: int, device: torch.device) -> Tensor:
    rows = 1
    for n in lead:
        rows *= n
    return torch.empty((rows, _pitch(width)), dtype=torch.float8_e4m3fn, device=device)[:, :width].view(*lead, width)


def _check_types(blocks: Float8Blocks, what: str) -> None:
    q, scale = blocks
    if q.dtype != torch.float8_e4m3fn or scale.dtype != torch.float32:
        raise TypeError(f"{what}: 8-bit blocks are float8_e4m3fn with float32 scales, got {q.dtype} and {scale.dtype}")
    assert q.dim() >= 1 and q.shape[-1] >= 1, f"{what}: 8-bit blocks need at least one column"


def _aligned_q(q: Tensor) -> Tensor:
    r"""``q`` as a matrix whose rows start on 16 bytes; a copy only where they do not."""
    width = q.shape[-1]
    q = q.reshape(-1, width)
    if q.numel() and ((width > 1 and q.stride(1) != 1) or q.data_ptr() % 16 or (q.shape[0] > 1 and (q.stride(0) % 16 or q.stride(0) < width))):
        q = _empty_q((q.shape[0],), width, q.device).copy_(q)
    return q


def _q_stride(q: Tensor) -> int:
    return q.stride(0) if q.shape[0] > 1 else _pitch(q.shape[1])


def _rows2d(blocks: Float8Blocks, what: str) -> Float8Blocks:
    r"""Blocks of 1 x 128 as matrices."""
    _check_types(blocks, what)
    q, scale = blocks
    assert scale.shape == (*q.shape[:-1], _count(q.shape[-1])), (
        f"{what}: one scale for each 128 columns of a row: {tuple(scale.shape)} for rows {tuple(q.shape)}"
    )
    return Float8Blocks(_aligned_q(q), scale.reshape(-1, scale.shape[-1]))


def _weight2d(blocks: Float8Blocks, what: str) -> Float8Blocks:
    r"""Blocks of 128 x 128."""
    _check_types(blocks, what)
    q, scale = blocks
    assert q.dim() == 2 and q.shape[0] >= 1, f"{what}: a weight is a matrix (out, in)"
    assert scale.shape == (_count(q.shape[0]), _count(q.shape[1])), (
        f"{what}: one scale for each 128 x 128 block: {tuple(scale.shape)} for a weight {tuple(q.shape)}"
    )
    return Float8Blocks(_aligned_q(q), scale)


def _block_args(blocks: Float8Blocks) -> tuple:
    q, scale = blocks
    return q.data_ptr(), _q_stride(q), scale.data_ptr(), scale.stride(0), scale.stride(1)


def _empty_rows(lead, width: int, device: torch.device) -> Float8Blocks:
    rows = 1
    for n in lead:
        rows *= n
    scale = torch.empty((_count(width), rows), dtype=torch.float32, device=device).t()  # neighbouring rows lie side by side
    return Float8Blocks(_empty_q(lead, width, device), scale.as_strided((*lead, _count(width)), (*_contiguous_strides(lead), rows)))


def _contiguous_strides(lead) -> Tuple[int, ...]:
    strides, step = [], 1
    for n in reversed(tuple(lead)):
        strides.append(step)
        step *= max(n, 1)
    return tuple(reversed(strides))


def _make_rows(x2d: Tensor, out: Float8Blocks) -> None:
    rows, width = x2d.shape
    with torch.cuda.device(x2d.device):
        _lib.check(
            _lib.lib().th_float8_rows(
                x2d.data_ptr(), row_stride(x2d), out.q.data_ptr(), _pitch(width), out.scale.data_ptr(), rows, rows, width,
                _lib.dtype_code(x2d), _lib.stream_ptr(x2d.device),
            ),
            "th_float8_rows",
        )  # fmt: skip


def _make_weight(w: Tensor) -> Float8Blocks:
    rows, width = w.shape
    out = Float8Blocks(_empty_q((rows,), width, w.device), torch.empty((_count(rows), _count(width)), dtype=torch.float32, device=w.device))
    with torch.cuda.device(w.device):
        _lib.check(
            _lib.lib().th_float8_weight(
                w.data_ptr(), row_stride(w), out.q.data_ptr(), _pitch(width), out.scale.data_ptr(), rows, width, _lib.dtype_code(w),
                _lib.stream_ptr(w.device),
            ),
            "th_float8_weight",
        )  # fmt: skip
    return out


def quantize_float8_rows(x: Tensor) -> Float8Blocks:
    r"""``x`` (..., K), float16, bfloat16 or float32, in blocks of 128 columns. The scales of neighbouring rows lie side by side. No
    gradient: an ``x`` that requires one is refused outside of ``torch.no_grad()``."""
    refuse_gradients("quantize_float8_rows", x)
    with torch.no_grad():
        assert x.dim() >= 1 and x.shape[-1] >= 1, "8-bit blocks need at least one column"
        float_dtype(x, "x")
        device = _lib.require_cuda(x)
        out = _empty_rows(x.shape[:-1], x.shape[-1], device)
        _make_rows(rows2d(x, x.shape[-1]), out)
        return out


def quantize_float8_weight(weight: Tensor) -> Float8Blocks:
    r"""A weight (N, K), float16, bfloat16 or float32, in blocks of 128 x 128. No gradient: a weight that requires one is refused outside
    of ``torch.no_grad()``."""
    refuse_gradients("quantize_float8_weight", weight)
    with torch.no_grad():
        assert weight.dim() == 2 and min(weight.shape) >= 1, "a weight is a matrix (out, in)"
        float_dtype(weight, "weight")
        _lib.require_cuda(weight)
        return _make_weight(rows2d(weight, weight.shape[1]))


def dequantize_float8(blocks: Float8Blocks, dtype: torch.dtype = torch.float32) -> Tensor:
    r"""``q * scale``, rounded once to ``dtype`` (float16, bfloat16 or float32); contiguous. Blocks are a weight's where their scales have a
    weight's shape, ``(ceil(N / 128), ceil(K / 128))``, and rows' where they have rows'. No gradient: scales that require one are refused
    outside of ``torch.no_grad()``."""
    refuse_gradients("dequantize_float8", blocks.scale)
    with torch.no_grad():
        _check_types(blocks, "dequantize_float8")
        lead, width = blocks.q.shape[:-1], blocks.q.shape[-1]
        rows = blocks.scale.shape == (*lead, _count(width))
        held = (_rows2d if rows else _weight2d)(blocks, "dequantize_float8")
        device = _lib.require_cuda(*held)
        out = torch.empty((*lead, width), dtype=dtype, device=device)
        float_dtype(out, "dtype")
        _values(held, 1 if rows else BLOCK, out.view(-1, width), width)
        return out


def _values(blocks: Float8Blocks, block_rows: int, out: Tensor, out_stride: int) -> None:
    rows, width = blocks.q.shape
    with torch.cuda.device(out.device):
        _lib.check(
            _lib.lib().th_float8_values(
                *_block_args(blocks), block_rows, out.data_ptr(), out_stride, rows, width, _lib.dtype_code(out), _lib.stream_ptr(out.device)
            ),
            "th_float8_values",
        )


def float8_linear(
    x: Union[Tensor, Float8Blocks], weight: Float8Blocks, bias: Optional[Tensor] = None, dtype: Optional[torch.dtype] = None
) -> Tensor:
    r"""Linear layer on 8-bit floating-point weights; a float ``x`` is turned into 8-bit blocks on the way. No gradient.

    Args:
        x: float16, bfloat16 or float32 tensor, or 8-bit blocks of ``quantize_float8_rows``
        weight: 8-bit blocks of the ``(out, in)`` weight matrix; their scales may be any float32 values
        bias: of the result's type, or ``None``
        dtype: type of the result; that of ``x`` by default, and required where ``x`` is 8-bit blocks

    Shapes:
        - x: :math:`(..., D_{in})`, output: :math:`(..., D_{out})`, bias: :math:`(D_{out},)`
    """
    held = x if isinstance(x, Float8Blocks) else None
    out = NotImplemented if held else _lib.native().float8_linear(x, *weight, bias, dtype)
    if out is not NotImplemented:
        return out
    if held:
        if dtype is None:
            raise TypeError("8-bit blocks do not say the type of the result: pass dtype")
        refuse_gradients("float8_linear", x.scale, weight.scale, bias)
    else:
        refuse_gradients("float8_linear", x, weight.scale, bias)
        dtype = float_dtype(x, "x") if dtype is None else dtype
    if dtype not in _lib.DTYPE_CODE:
        raise TypeError(f"the result must be float16, bfloat16 or float32, got {dtype}")
    with torch.no_grad():
        w = _weight2d(weight, "weight")
        d_out, d_in = w.q.shape
        source = x if held is None else held.q
        assert source.dim() >= 1 and source.shape[-1] == d_in, f"Input dimension mismatch: {tuple(source.shape)} and {d_in}"
        assert bias is None or bias.shape == (d_out,), "Bias shape mismatch"
        if bias is not None and bias.dtype != dtype:
            raise TypeError(f"the bias must be of the result's type {dtype}, got {bias.dtype}")
        held = None if held is None else _rows2d(held, "x")
        device = _lib.require_cuda(*((x,) if held is None else held), *w, bias)
        bias = None if bias is None else bias.contiguous()
        y = torch.empty((*source.shape[:-1], d_out), dtype=dtype, device=device)
        lib, code = _lib.lib(), _lib.DTYPE_CODE[dtype]
        with torch.cuda.device(device):
            stream = _lib.stream_ptr(device)
            if held is None:
                x2d = rows2d(x, d_in)
                ws_bytes = lib.th_float8_quantized_linear_workspace_bytes(x2d.shape[0], d_in)
                workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=device)
                _lib.check(
                    lib.th_float8_quantized_linear(
                        x2d.data_ptr(), row_stride(x2d), _lib.dtype_code(x), *_block_args(w), _lib.ptr(bias), y.data_ptr(), d_out,
                        workspace.data_ptr(), ws_bytes, x2d.shape[0], d_in, d_out, code, stream,
                    ),
                    "th_float8_quantized_linear",
                )  # fmt: skip
            else:
                _lib.check(
                    lib.th_float8_linear(
                        *_block_args(held), *_block_args(w), _lib.ptr(bias), y.data_ptr(), d_out, held.q.shape[0], d_in, d_out, code, stream
                    ),
                    "th_float8_linear",
                )
    return y


# ---- training -----------------------------------------------------------------------------------------------


def _validate(x: Tensor, weight: Tensor, bias: Optional[Tensor]) -> Tuple[int, int]:
    assert weight.dim() == 2 and min(weight.shape) >= 1, "the weight is a matrix (out, in)"
    d_out, d_in = weight.shape
    assert x.dim() >= 1 and x.shape[-1] == d_in, f"Input dimension mismatch: {tuple(x.shape)} and {d_in}"
    assert bias is None or bias.shape == (d_out,), "Bias shape mismatch"
    dtypes = {t.dtype for t in (x, weight, bias) if t is not None}
    if len(dtypes) != 1 or next(iter(dtypes)) not in (torch.float16, torch.bfloat16):
        raise TypeError(f"8-bit training kernels take float16 or bfloat16 tensors of one dtype, got {dtypes}")
    return d_in, d_out


class _float8_training_linear(Function):

    @staticmethod
    def forward(ctx, x: Tensor, weight: Tensor, bias: Optional[Tensor]) -> Tensor:
        return _forward_in(torch.get_autocast_dtype("cuda"))(ctx, x, weight, bias)  # the type to cast to is known at the call

    @staticmethod
    def _forward(ctx, x: Tensor, weight: Tensor, bias: Optional[Tensor]) -> Tensor:
        d_in, d_out = _validate(x, weight, bias)
        device = _lib.require_cuda(x, weight, bias)
        x2d = rows2d(x, d_in)
        rows, code = x2d.shape[0], _lib.DTYPE_CODE[x.dtype]
        held = _empty_rows((rows,), d_in, device)
        _make_rows(x2d, held)
        w = _make_weight(rows2d(weight, d_in))
        b = None if bias is None else bias.contiguous()
        y = torch.empty((*x.shape[:-1], d_out), dtype=x.dtype, device=device)
        with torch.cuda.device(device):
            _lib.check(
                _lib.lib().th_float8_linear(
                    *_block_args(held), *_block_args(w), _lib.ptr(b), y.data_ptr(), d_out, rows, d_in, d_out, code, _lib.stream_ptr(device)
                ),
                "th_float8_linear",
            )
        ctx.save_for_backward(*(w if ctx.needs_input_grad[0] else (None, None)), *(held if ctx.needs_input_grad[1] else (None, None)))
        ctx.x_shape, ctx.d_out, ctx.dtype = x.shape, d_out, x.dtype
        return y

    @staticmethod
    @torch.amp.custom_bwd(device_type="cuda")
    @first_order("float8_training_linear")
    def backward(ctx, gy: Tensor):
        wq, w_scale, xq, x_scale = ctx.saved_tensors
        want_x, want_w, want_b = ctx.needs_input_grad
        d_in, d_out, dtype, device = ctx.x_shape[-1], ctx.d_out, ctx.dtype, gy.device
        gy2d = rows2d(gy.to(dtype), d_out)
        gy2d = gy2d if gy2d.shape[0] < 2 or gy2d.stride(0) >= d_out else gy2d.contiguous()
        # the weight's product wants rows that start on 16 bytes: where they do not, the kernel that makes blocks of them copies them
        copied = want_w and (gy2d.data_ptr() % 16 != 0 or row_stride(gy2d) % 8 != 0)
        if copied and not want_x:
            gy2d = _operand(gy2d, d_out)
        rows, code = gy2d.shape[0], _lib.DTYPE_CODE[dtype]
        dx = dw = db = None
        lib = _lib.lib()
        with torch.cuda.device(device):
            stream = _lib.stream_ptr(device)
            if want_x:
                g8 = _empty_rows((rows,), d_out, device)
                if copied:
                    rows16 = _empty_operand(rows, d_out, gy2d)
                    _lib.check(
                        lib.th_float8_rows_copied(
                            gy2d.data_ptr(), row_stride(gy2d), g8.q.data_ptr(), _pitch(d_out), g8.scale.data_ptr(), rows, rows16.data_ptr(),
                            _stride(rows16), rows, d_out, code, stream,
                        ),
                        "th_float8_rows_copied",
                    )  # fmt: skip
                    gy2d = rows16
                else:
                    _make_rows(gy2d, g8)
                w = _weight2d(Float8Blocks(wq, w_scale), "kept weight")
                dx = torch.empty(ctx.x_shape, dtype=dtype, device=device)
                _lib.check(
                    lib.th_float8_bwd_input(*_block_args(g8), *_block_args(w), dx.data_ptr(), d_in, rows, d_in, d_out, code, stream),
                    "th_float8_bwd_input",
                )
            if want_b:
                db = torch.empty(d_out, dtype=dtype, device=device)
                sum_bytes = lib.th_column_sum_workspace_bytes(rows, d_out)
                partial = torch.empty(sum_bytes, dtype=torch.uint8, device=device)
                _lib.check(
                    lib.th_column_sum(
                        gy2d.data_ptr(), _stride(gy2d), db.data_ptr(), partial.data_ptr(), sum_bytes, rows, d_out, code, stream
                    ),
                    "th_column_sum",
                )
            if want_w:
                x16 = _empty_operand(rows, d_in, gy2d)
                _values(_rows2d(Float8Blocks(xq, x_scale), "kept input"), 1, x16, _stride(x16))
                dw = torch.empty((d_out, d_in), dtype=dtype, device=device)
                _lib.check(
                    lib.th_linear_bwd_weight(
                        gy2d.data_ptr(), _stride(gy2d), x16.data_ptr(), _stride(x16), dw.data_ptr(), rows, d_in, d_out, code, stream
                    ),
                    "th_linear_bwd_weight",
                )
        return dx, dw, db


@lru_cache(maxsize=None)
def _forward_in(dtype: torch.dtype) -> Callable:
    return torch.amp.custom_fwd(_float8_training_linear._forward, device_type="cuda", cast_inputs=dtype)


def float8_training_linear(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None) -> Tensor:
    r"""Linear layer whose products run on 8-bit blocks of its input, weight and output gradient; see the module's text.

    Args:
        x: float16 or bfloat16; under autocast any float type but float64, cast to autocast's (float16 or bfloat16)
        weight, bias: of x's type; the bias may be ``None``

    Shapes:
        - x: :math:`(..., D_{in})`, output: :math:`(..., D_{out})`
        - weight: :math:`(D_{out}, D_{in})`, bias: :math:`(D_{out},)`
    """
    out = _lib.native().float8_training_linear(x, weight, bias)
    if out is not NotImplemented:
        return out
    return _float8_training_linear.apply(x, weight, bias)
