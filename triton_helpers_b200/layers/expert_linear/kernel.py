r"""Linear layers of several experts on rows sorted by expert, on hand-written sm_100a kernels.

There is no such operator in triton_helpers; this module follows the conventions of its fused MLP
(``triton_helpers/layers/fully_fused_mlp/kernel.py:640-686``): a ``torch.autograd.Function`` plus a functional wrapper, weights as
``(out, in)`` behind the experts. Under autocast the layer runs in autocast's type.

    rows ends[e - 1] .. ends[e] - 1 belong to expert e (ends[-1] = 0)

    y[r] = x[r] W_e^T          dx[r] = dy[r] W_e          dW_e = sum over its rows of dy[r]^T x[r]

Operands have 16 bits, sums float32, results are rounded once and repeat bit for bit. The ends stay on the device: nothing waits for
them, and a captured graph follows new ones. Any number of rows may go to an expert, none among them. Rows behind the last end belong to
no expert: their results and their input gradients are zero, and what they hold (a NaN, say) reaches nothing else. An end below the one before it counts as
that one, an end above the number of rows as that number.
"""
from functools import lru_cache
from typing import Callable, Tuple

import torch
from torch import Tensor
from torch.autograd import Function

from ... import _lib
from ..checkpointed_linear.kernel import _operand, _stride
from ..int8_linear.kernel import first_order

MAX_EXPERTS = 1024


def _validate(x: Tensor, weight: Tensor, ends: Tensor) -> Tuple[int, int, int]:
    assert weight.dim() == 3 and min(weight.shape) >= 1, "the weight is (experts, out, in)"
    experts, d_out, d_in = weight.shape
    assert experts <= MAX_EXPERTS, f"at most {MAX_EXPERTS} experts, got {experts}"
    assert x.dim() == 2 and x.shape[1] == d_in, f"Input dimension mismatch: {tuple(x.shape)} and {d_in}"
    assert ends.shape == (experts,), f"one end for each expert: {tuple(ends.shape)} for {experts}"
    if ends.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"ends must be int32 or int64, got {ends.dtype}")
    if x.dtype != weight.dtype or x.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"expert kernels take float16 or bfloat16 tensors of one dtype, got {x.dtype} and {weight.dtype}")
    return experts, d_in, d_out


def _weight_rows(weight: Tensor) -> Tuple[Tensor, int, int]:
    r"""A weight whose rows and experts start on 16 bytes, the stride of its rows and that of its experts; a copy only where they do not."""
    experts, d_out, d_in = weight.shape
    row = weight.stride(1) if d_out > 1 else -(-d_in // 8) * 8
    expert = weight.stride(0) if experts > 1 else -(-d_out * row // 8) * 8
    if (d_in == 1 or weight.stride(2) == 1) and weight.data_ptr() % 16 == 0 and row % 8 == 0 and expert % 8 == 0 and row >= d_in and expert >= d_out * row:
        return weight, row, expert
    held = _operand(weight.reshape(-1, d_in), d_in)
    return held, _stride(held), d_out * _stride(held)


class _expert_linear(Function):

    @staticmethod
    def forward(ctx, x: Tensor, weight: Tensor, ends: Tensor) -> Tensor:
        return _forward_in(torch.get_autocast_dtype("cuda"))(ctx, x, weight, ends)  # the type to cast to is known at the call

    @staticmethod
    def _forward(ctx, x: Tensor, weight: Tensor, ends: Tensor) -> Tensor:
        experts, d_in, d_out = _validate(x, weight, ends)
        device = _lib.require_cuda(x, weight, ends)
        rows = x.shape[0]
        if ends.dtype == torch.int64:
            ends = ends.clamp(0, rows).to(torch.int32)
        ends = ends.contiguous()
        x2d, (w, w_row, w_expert) = _operand(x, d_in), _weight_rows(weight)
        y = torch.empty((rows, d_out), dtype=x.dtype, device=device)
        with torch.cuda.device(device):
            _lib.check(
                _lib.lib().th_expert_linear_fwd(
                    x2d.data_ptr(), _stride(x2d), w.data_ptr(), w_row, w_expert, ends.data_ptr(), y.data_ptr(), d_out, rows, experts, d_in,
                    d_out, _lib.DTYPE_CODE[x.dtype], _lib.stream_ptr(device),
                ),
                "th_expert_linear_fwd",
            )  # fmt: skip
        ctx.save_for_backward(x if ctx.needs_input_grad[1] else None, weight if ctx.needs_input_grad[0] else None, ends)
        ctx.x_shape, ctx.w_shape, ctx.dtype = x.shape, weight.shape, x.dtype
        return y

    @staticmethod
    @torch.amp.custom_bwd(device_type="cuda")
    @first_order("expert_linear")
    def backward(ctx, gy: Tensor):
        x, weight, ends = ctx.saved_tensors
        want_x, want_w, _ = ctx.needs_input_grad
        (experts, d_out, d_in), dtype, device = ctx.w_shape, ctx.dtype, gy.device
        gy2d = _operand(gy.to(dtype), d_out)
        rows, code = gy2d.shape[0], _lib.DTYPE_CODE[dtype]
        dx = dw = None
        lib = _lib.lib()
        with torch.cuda.device(device):
            stream = _lib.stream_ptr(device)
            if want_x:
                w, w_row, w_expert = _weight_rows(weight)
                dx = torch.empty(ctx.x_shape, dtype=dtype, device=device)
                _lib.check(
                    lib.th_expert_linear_bwd_input(
                        gy2d.data_ptr(), _stride(gy2d), w.data_ptr(), w_row, w_expert, ends.data_ptr(), dx.data_ptr(), d_in, rows, experts,
                        d_in, d_out, code, stream,
                    ),
                    "th_expert_linear_bwd_input",
                )  # fmt: skip
            if want_w:
                x2d = _operand(x, d_in)
                dw = torch.empty(ctx.w_shape, dtype=dtype, device=device)
                _lib.check(
                    lib.th_expert_linear_bwd_weight(
                        gy2d.data_ptr(), _stride(gy2d), x2d.data_ptr(), _stride(x2d), ends.data_ptr(), dw.data_ptr(), rows, experts, d_in,
                        d_out, code, stream,
                    ),
                    "th_expert_linear_bwd_weight",
                )  # fmt: skip
        return dx, dw, None


@lru_cache(maxsize=None)
def _forward_in(dtype: torch.dtype) -> Callable:
    return torch.amp.custom_fwd(_expert_linear._forward, device_type="cuda", cast_inputs=dtype)


def expert_linear(x: Tensor, weight: Tensor, ends: Tensor) -> Tensor:
    r"""Linear layers of several experts, each on its own rows of ``x``.

    Args:
        x: float16 or bfloat16 rows sorted by expert; under autocast any float type but float64, cast to autocast's (float16 or bfloat16)
        weight: one matrix for each expert, of x's type
        ends: int32 or int64 on the device: the first row behind each expert's, the cumulative sum of the experts' numbers of rows
            (``torch.cumsum(counts, 0, dtype=torch.int32)``). int32 is what the kernels read; int64, which ``cumsum`` gives by itself, is
            converted by two more kernels, and such calls take the longer way through Python.

    Shapes:
        - x: :math:`(R, D_{in})`, output: :math:`(R, D_{out})`
        - weight: :math:`(E, D_{out}, D_{in})`, ends: :math:`(E,)`
    """
    out = _lib.native().expert_linear(x, weight, ends)
    if out is not NotImplemented:
        return out
    return _expert_linear.apply(x, weight, ends)
