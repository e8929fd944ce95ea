r"""Linear layer of any width that keeps its input in 8 bits for the backward pass, on hand-written sm_100a kernels.

There is no such operator in triton_helpers, whose fused network ends at 64 columns
(``triton_helpers/layers/fully_fused_mlp/kernel.py:13-14``); this module follows its conventions: a
``torch.autograd.Function`` plus a functional wrapper, ``(out, in)`` weights.  Under autocast the layer runs in autocast's type.

    y = x w^T + b                     16-bit operands, float32 sums, rounded once
    kept: q, scale = 8-bit rows of x (``layers.int8_linear``): K + 4 bytes a row instead of 2 K
    dx = dy w          dw = dy^T (q * scale)          db = sum over rows of dy

Only the weight's gradient sees the 8-bit values: the output and the input's gradient are those of an ordinary layer, so the
rounding does not add up from layer to layer.  A row's rounding is at most half a step, 1/254 of its largest magnitude; as an
operand of the product ``q * scale`` is rounded once more, to the layer's 16-bit type.
"""
from ctypes import c_int, c_void_p
from functools import lru_cache
from typing import Callable, Optional, Tuple

import torch
from torch import Tensor
from torch.autograd import Function

from ... import _lib
from ..int8_linear.kernel import empty_int8_rows, first_order, int8_rows2d, int8_stride, Int8Rows


def _validate(x: Tensor, weight: Tensor, bias: Optional[Tensor]) -> Tuple[int, int]:
    assert weight.dim() == 2 and min(weight.shape) >= 1, "the weight is a matrix (out, in)"
    d_out, d_in = weight.shape
    assert x.dim() >= 1 and x.shape[-1] == d_in, f"Input dimension mismatch: {tuple(x.shape)} and {d_in}"
    assert bias is None or bias.shape == (d_out,), "Bias shape mismatch"
    dtypes = {t.dtype for t in (x, weight, bias) if t is not None}
    if len(dtypes) != 1 or next(iter(dtypes)) not in (torch.float16, torch.bfloat16):
        raise TypeError(f"checkpointed linear kernels take float16 or bfloat16 tensors of one dtype, got {dtypes}")
    return d_in, d_out


def _operand(t: Tensor, width: int) -> Tensor:
    r"""``t`` as rows that start on 16 bytes, which is what the products read; a copy only where they do not."""
    t = t.reshape(-1, width)
    if (width > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < width):
        t = t.contiguous()
    if t.data_ptr() % 16 or (t.shape[0] > 1 and t.stride(0) % 8):
        out = _empty_operand(t.shape[0], width, t)
        with torch.cuda.device(t.device):
            _lib.check(
                _lib.lib().th_copy_rows(
                    1, (c_void_p * 1)(t.data_ptr()), _lib.i64_array([t.stride(0) if t.shape[0] > 1 else width]), (c_void_p * 1)(out.data_ptr()),
                    _lib.i64_array([_stride(out)]), _lib.i64_array([t.shape[0]]), (c_int * 1)(width), _lib.stream_ptr(t.device),
                ),
                "th_copy_rows",
            )  # fmt: skip
        return out
    return t


def _empty_operand(rows: int, width: int, like: Tensor) -> Tensor:
    return torch.empty((rows, -(-width // 8) * 8), dtype=like.dtype, device=like.device)[:, :width]


def _stride(t: Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else -(-t.shape[1] // 8) * 8


class _checkpointed_linear(Function):

    @staticmethod
    def forward(ctx, x: Tensor, weight: Tensor, bias: Optional[Tensor]) -> Tensor:
        return _forward_in(torch.get_autocast_dtype("cuda"))(ctx, x, weight, bias)  # the type to cast to is known at the call

    @staticmethod
    def _forward(ctx, x: Tensor, weight: Tensor, bias: Optional[Tensor]) -> Tensor:
        d_in, d_out = _validate(x, weight, bias)
        device = _lib.require_cuda(x, weight, bias)
        x2d, w = _operand(x, d_in), _operand(weight, d_in)
        b = None if bias is None else bias.contiguous()
        rows, code = x2d.shape[0], _lib.DTYPE_CODE[x.dtype]
        y = torch.empty((*x.shape[:-1], d_out), dtype=x.dtype, device=device)
        lib = _lib.lib()
        rows8 = None
        with torch.cuda.device(device):
            _lib.check(
                lib.th_linear_fwd(
                    x2d.data_ptr(), _stride(x2d), w.data_ptr(), _stride(w), _lib.ptr(b), y.data_ptr(), d_out, rows, d_in,
                    d_out, code, _lib.stream_ptr(device),
                ),
                "th_linear_fwd",
            )  # fmt: skip
            if ctx.needs_input_grad[1]:
                rows8 = empty_int8_rows((rows,), d_in, device)
                _lib.check(
                    lib.th_quantize_rows(
                        x2d.data_ptr(), _stride(x2d), rows8.q.data_ptr(), int8_stride(rows8.q), rows8.scale.data_ptr(), rows, d_in, code,
                        _lib.stream_ptr(device),
                    ),
                    "th_quantize_rows",
                )  # fmt: skip
        ctx.save_for_backward(weight if ctx.needs_input_grad[0] else None, *(rows8 or (None, None)))
        ctx.x_shape, ctx.d_out, ctx.dtype = x.shape, d_out, x.dtype
        return y

    @staticmethod
    @torch.amp.custom_bwd(device_type="cuda")
    @first_order("checkpointed_linear")
    def backward(ctx, gy: Tensor):
        weight, q, scale = ctx.saved_tensors
        want_x, want_w, want_b = ctx.needs_input_grad
        d_in, d_out, dtype, device = ctx.x_shape[-1], ctx.d_out, ctx.dtype, gy.device
        gy2d = _operand(gy.to(dtype), d_out)
        rows, code = gy2d.shape[0], _lib.DTYPE_CODE[dtype]
        dx = dw = db = None
        lib = _lib.lib()
        with torch.cuda.device(device):
            stream = _lib.stream_ptr(device)
            if want_x:
                w = _operand(weight, d_in)
                dx = torch.empty(ctx.x_shape, dtype=dtype, device=device)
                _lib.check(
                    lib.th_linear_bwd_input(
                        gy2d.data_ptr(), _stride(gy2d), w.data_ptr(), _stride(w), dx.data_ptr(), d_in, rows, d_in,
                        d_out, code, stream,
                    ),
                    "th_linear_bwd_input",
                )  # fmt: skip
            if want_b:
                db = torch.empty(d_out, dtype=dtype, device=device)
                sum_bytes = lib.th_column_sum_workspace_bytes(rows, d_out)
                partial = torch.empty(sum_bytes, dtype=torch.uint8, device=device)
            if want_w:
                q, scale = int8_rows2d(Int8Rows(q, scale), "kept input")
                x8 = _empty_operand(rows, d_in, gy2d)
                if want_b:
                    _lib.check(
                        lib.th_checkpoint_rows(
                            q.data_ptr(), int8_stride(q), scale.data_ptr(), x8.data_ptr(), _stride(x8), d_in, gy2d.data_ptr(), _stride(gy2d),
                            db.data_ptr(), d_out, partial.data_ptr(), sum_bytes, rows, code, stream,
                        ),
                        "th_checkpoint_rows",
                    )  # fmt: skip
                else:
                    _lib.check(
                        lib.th_dequantize_rows(
                            q.data_ptr(), int8_stride(q), scale.data_ptr(), x8.data_ptr(), _stride(x8), rows, d_in, code, stream
                        ),
                        "th_dequantize_rows",
                    )
                dw = torch.empty((d_out, d_in), dtype=dtype, device=device)
                _lib.check(
                    lib.th_linear_bwd_weight(
                        gy2d.data_ptr(), _stride(gy2d), x8.data_ptr(), _stride(x8), dw.data_ptr(), rows, d_in, d_out, code,
                        stream,
                    ),
                    "th_linear_bwd_weight",
                )  # fmt: skip
            elif want_b:
                _lib.check(
                    lib.th_column_sum(
                        gy2d.data_ptr(), _stride(gy2d), db.data_ptr(), partial.data_ptr(), sum_bytes, rows, d_out, code, stream
                    ),
                    "th_column_sum",
                )
        return dx, dw, db


@lru_cache(maxsize=None)
def _forward_in(dtype: torch.dtype) -> Callable:
    return torch.amp.custom_fwd(_checkpointed_linear._forward, device_type="cuda", cast_inputs=dtype)


def checkpointed_linear(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None) -> Tensor:
    r"""Linear layer whose backward pass reads its input from 8-bit rows kept by the forward pass.

    Args:
        x: float16 or bfloat16; under autocast any float type but float64, cast to autocast's (float16 or bfloat16)
        weight, bias: of x's type; the bias may be ``None``

    Shapes:
        - x: :math:`(..., D_{in})`, output: :math:`(..., D_{out})`
        - weight: :math:`(D_{out}, D_{in})`, bias: :math:`(D_{out},)`
    """
    out = _lib.native().checkpointed_linear(x, weight, bias)
    if out is not NotImplemented:
        return out
    return _checkpointed_linear.apply(x, weight, bias)
