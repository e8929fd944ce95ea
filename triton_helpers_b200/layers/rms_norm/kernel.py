r"""Root-mean-square norm with the residual's addition, and with 8-bit rows as its output, on hand-written sm_100a kernels.

There is no such operator in triton_helpers; this module follows the conventions of its fused MLP
(``triton_helpers/layers/fully_fused_mlp/kernel.py:503-686``): a ``torch.autograd.Function`` plus functional wrappers.

    s = x + residual                            rounded to the rows' type; s = x without a residual
    y = s / sqrt(mean_k s_k^2 + eps) * weight   float32 arithmetic, rounded once

``rms_norm`` returns ``y``, or ``(y, s)`` with a residual: ``s`` is the stream the next block adds to.  Its backward pass reads ``s``
and one float32 per row.  ``rms_norm_int8`` returns ``y`` as the 8-bit rows of ``layers.int8_linear``, taken from the unrounded
float32 values, for the linear layer that follows; it has no gradient.
"""
from typing import Optional, Tuple, Union

import torch
from torch import Tensor
from torch.autograd import Function

from ... import _lib
from ..int8_linear.kernel import Int8Rows, empty_int8_rows, first_order, float_dtype, refuse_gradients, row_stride, rows2d


def _validate(x: Tensor, weight: Tensor, residual: Optional[Tensor]) -> int:
    assert x.dim() >= 1 and x.shape[-1] >= 1, "the norm needs at least one column"
    d = x.shape[-1]
    assert weight.shape == (d,), f"Weight shape mismatch: {tuple(weight.shape)} for rows of {d}"
    assert residual is None or residual.shape == x.shape, "Residual shape mismatch"
    dtype = float_dtype(x, "x")
    if residual is not None and residual.dtype != dtype:
        raise TypeError(f"x and residual must share one dtype, got {dtype} and {residual.dtype}")
    if weight.dtype not in (dtype, torch.float32):
        raise TypeError(f"the weight must be float32 or of x's dtype {dtype}, got {weight.dtype}")
    return d


class _rms_norm(Function):

    @staticmethod
    @torch.amp.custom_fwd(device_type="cuda")
    def forward(ctx, x: Tensor, weight: Tensor, residual: Optional[Tensor], eps: float):
        d = _validate(x, weight, residual)
        device = _lib.require_cuda(x, weight, residual)
        weight = weight.contiguous()
        x2d = rows2d(x, d)
        res2d = None if residual is None else rows2d(residual, d)
        rows = x2d.shape[0]
        y = torch.empty(x.shape, dtype=x.dtype, device=device)
        s = None if residual is None else torch.empty_like(y)
        rstd = torch.empty(rows, dtype=torch.float32, device=device)
        with torch.cuda.device(device):
            _lib.check(
                _lib.lib().th_rms_norm_fwd(
                    x2d.data_ptr(), row_stride(x2d), _lib.ptr(res2d), 0 if res2d is None else row_stride(res2d), weight.data_ptr(),
                    _lib.dtype_code(weight), _lib.ptr(s), y.data_ptr(), rstd.data_ptr(), rows, d, eps, _lib.dtype_code(x),
                    _lib.stream_ptr(device),
                ),
                "th_rms_norm_fwd",
            )  # fmt: skip
        ctx.save_for_backward(x if s is None else s, weight, rstd)
        ctx.set_materialize_grads(False)
        ctx.shape = x.shape
        return y if s is None else (y, s)

    @staticmethod
    @torch.amp.custom_bwd(device_type="cuda")
    @first_order("rms_norm")
    def backward(ctx, gy: Optional[Tensor], gs: Optional[Tensor] = None):
        s, weight, rstd = ctx.saved_tensors
        want_x, want_w, want_r, _ = ctx.needs_input_grad
        if gy is None:  # only the sum was used
            return gs if want_x else None, None, gs if want_r else None, None
        d, device, dtype = ctx.shape[-1], s.device, s.dtype
        s2d, gy2d = rows2d(s, d), rows2d(gy.to(dtype), d)
        gs2d = None if gs is None else rows2d(gs.to(dtype), d)
        rows = s2d.shape[0]
        dx = torch.empty(ctx.shape, dtype=dtype, device=device)
        dw = torch.empty_like(weight) if want_w else None
        lib = _lib.lib()
        with torch.cuda.device(device):
            ws_bytes = lib.th_rms_norm_bwd_workspace_bytes(rows, d, _lib.dtype_code(s)) if want_w else 0
            workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=device) if ws_bytes else None
            _lib.check(
                lib.th_rms_norm_bwd(
                    s2d.data_ptr(), row_stride(s2d), weight.data_ptr(), _lib.dtype_code(weight), rstd.data_ptr(), gy2d.data_ptr(),
                    row_stride(gy2d), _lib.ptr(gs2d), 0 if gs2d is None else row_stride(gs2d), dx.data_ptr(), _lib.ptr(dw),
                    _lib.ptr(workspace), ws_bytes, rows, d, _lib.dtype_code(s), _lib.stream_ptr(device),
                ),
                "th_rms_norm_bwd",
            )  # fmt: skip
        return dx if want_x else None, dw, dx if want_r else None, None


def rms_norm(x: Tensor, weight: Tensor, residual: Optional[Tensor] = None, eps: float = 1e-6) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    r"""Root-mean-square norm of ``x``, or of ``x + residual``.

    Args:
        x: float16, bfloat16 or float32
        weight: gain per column, float32 or of x's type
        residual: added to ``x`` first, same shape and type
        eps: added to the mean square

    Returns:
        ``y``, or ``(y, x + residual)`` where a residual is given

    Shapes:
        - x, residual, outputs: :math:`(..., D)`, weight: :math:`(D,)`
    """
    out = _lib.native().rms_norm(x, weight, residual, eps)
    if out is not NotImplemented:
        return out
    return _rms_norm.apply(x, weight, residual, float(eps))


def rms_norm_int8(
    x: Tensor, weight: Tensor, residual: Optional[Tensor] = None, eps: float = 1e-6
) -> Union[Int8Rows, Tuple[Int8Rows, Tensor]]:
    r"""``rms_norm`` with 8-bit rows as its output, for ``int8_linear``: ``rows``, or ``(rows, x + residual)``.  No gradient."""
    out = _lib.native().rms_norm_int8(x, weight, residual, eps)
    if out is not NotImplemented:
        return Int8Rows(*out) if residual is None else (Int8Rows(out[0], out[1]), out[2])
    refuse_gradients("rms_norm_int8", x, weight, residual)
    with torch.no_grad():
        d = _validate(x, weight, residual)
        device = _lib.require_cuda(x, weight, residual)
        weight = weight.contiguous()
        x2d = rows2d(x, d)
        res2d = None if residual is None else rows2d(residual, d)
        out = empty_int8_rows(x.shape[:-1], d, device)
        s = None if residual is None else torch.empty(x.shape, dtype=x.dtype, device=device)
        with torch.cuda.device(device):
            _lib.check(
                _lib.lib().th_rms_norm_int8(
                    x2d.data_ptr(), row_stride(x2d), _lib.ptr(res2d), 0 if res2d is None else row_stride(res2d), weight.data_ptr(),
                    _lib.dtype_code(weight), _lib.ptr(s), out.q.data_ptr(), -(-d // 16) * 16, out.scale.data_ptr(), x2d.shape[0], d,
                    float(eps), _lib.dtype_code(x), _lib.stream_ptr(device),
                ),
                "th_rms_norm_int8",
            )  # fmt: skip
    return out if s is None else (out, s)
