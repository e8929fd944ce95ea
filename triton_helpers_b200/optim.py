r"""Adam for 16-bit parameters with fp32 moments, all tensors of a dtype in one CUDA kernel.

``torch.optim.Adam`` keeps its moments in the parameter dtype; with float16 hash tables the
second moment underflows (``g*g < 6e-8`` for ``|g| < 2.4e-4``) and the update divides by
``eps``.  ``FusedAdam`` follows the same update rule (no weight decay, no amsgrad) but stores
``exp_avg`` / ``exp_avg_sq`` in float32, scales the stored gradient by ``grad_scale`` on the fly
(inverse loss scale and world size) and can clear the gradient buffer in the same pass, which
replaces the separate zero-fill the hash-encoding backward needs before every step.

Elements whose gradient is not finite (an overflowed 16-bit sum, a NaN from upstream) are left
untouched - parameter and moments - and counted; ``FusedAdam.skipped_elements()`` reads the count
(on each device at most 2^31 - 1, where it stays).

Gradients may be clipped to a global norm on the way: all of them as one vector, its norm and the factor
stay on the device, and the update multiplies by the factor as it reads::

    norm = sqrt(sum_k scale_k^2 sum_i g_k[i]^2)        factor = min(1, max_norm / (norm + 1e-6))

Squares are added in float32 over 16 bytes of gradients and in float64 from there, in a fixed order (results repeat bit
for bit); 16 bytes whose largest element is outside of 2^-50 .. 2^50 are added in float64 throughout, so that neither large nor small
squares are lost. A norm that is not finite passes over the whole step: every element counts as skipped.
"""
import math
from ctypes import c_float, c_int, c_void_p
from typing import Dict, Iterable, List, Optional, Sequence, Tuple, Union

import torch
from torch import Tensor
from torch.optim.optimizer import _global_optimizer_post_hooks, _global_optimizer_pre_hooks

from . import _lib


@torch.no_grad()
def adam_update(
    param: Tensor,
    grad: Tensor,
    exp_avg: Tensor,
    exp_avg_sq: Tensor,
    step: int,
    lr: float,
    betas: Tuple[float, float],
    eps: float,
    grad_scale: float = 1.0,
    zero_grad: bool = False,
    skipped: Optional[Tensor] = None,
) -> None:
    r"""One ``th_adam_step`` launch: ``param`` (float32 / float16 / bfloat16, contiguous) is updated in
    place from ``grad`` (same dtype and element count) times ``grad_scale``; ``exp_avg`` / ``exp_avg_sq``
    are float32.  ``skipped`` is an int32 device counter of elements passed over because their gradient
    was not finite; it stays at 2^31 - 1."""
    if grad.dtype != param.dtype or not param.is_contiguous() or not grad.is_contiguous():
        raise RuntimeError("adam_update needs contiguous parameters and same-dtype contiguous gradients")
    device = _lib.require_cuda(param, grad, exp_avg, exp_avg_sq, skipped)
    with torch.cuda.device(device):
        _lib.check(
            _lib.lib().th_adam_step(
                param.data_ptr(), grad.data_ptr(), exp_avg.data_ptr(), exp_avg_sq.data_ptr(), param.numel(), lr,
                betas[0], betas[1], eps, step, grad_scale, int(zero_grad), _lib.dtype_code(param), _lib.ptr(skipped),
                _lib.stream_ptr(device),
            ),
            "th_adam_step",
        )  # fmt: skip


def adam_updates(params, grads, exp_avgs, exp_avg_sqs, grad_scales, zero_grads, step, lr, betas, eps, skipped) -> None:
    r"""``adam_update`` of several tensors of one dtype and device: one launch where the native path takes them."""
    done = _lib.native().adam_steps(params, grads, exp_avgs, exp_avg_sqs, tuple(grad_scales), tuple(zero_grads), lr, betas[0], betas[1], eps, step, skipped)
    if done is NotImplemented:
        for p, g, m, v, scale, zero in zip(params, grads, exp_avgs, exp_avg_sqs, grad_scales, zero_grads):
            adam_update(p, g, m, v, step, lr, betas, eps, scale, zero, skipped)


# ---- the global norm ----------------------------------------------------------------------------------------


def _flat(tensors: Sequence[Tensor], what: str) -> Tuple[List[Tensor], torch.device]:
    r"""Checks a list of gradients and returns them contiguous (copied where they are not)."""
    for t in tensors:
        if t.layout != torch.strided:
            raise TypeError(f"{what}: gradients must be dense, got {t.layout}")
        _lib.dtype_code(t)
    device = _lib.require_cuda(*tensors)
    return [t.detach().contiguous() for t in tensors], device


def _lists(tensors: Sequence[Tensor]) -> tuple:
    n = len(tensors)
    return (
        (c_void_p * n)(*(t.data_ptr() for t in tensors)),
        _lib.i64_array([t.numel() for t in tensors]),
        (c_int * n)(*(_lib.DTYPE_CODE[t.dtype] for t in tensors)),
    )


def _check_norm(max_norm: float) -> float:
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError(f"max_norm must not be negative, got {max_norm}")
    return max_norm


def _norm_factor(tensors: Sequence[Tensor], scales: Optional[Sequence[float]], max_norm: float) -> Tensor:
    r"""(norm, factor) of a list of gradients, a float32 pair on their device."""
    pair = _lib.native().grad_norm(tensors, None if scales is None else tuple(scales), max_norm)
    if pair is not NotImplemented:
        return pair
    _lib.refuse_trace("the global norm")
    flat, device = _flat(tensors, "the global norm")
    pointers, sizes, codes = _lists(flat)
    lib = _lib.lib()
    pair = torch.empty(2, dtype=torch.float32, device=device)
    ws_bytes = lib.th_grad_norm_workspace_bytes(len(flat), sizes)
    workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=device)
    with torch.cuda.device(device):
        _lib.check(
            lib.th_grad_norm(
                len(flat), pointers, sizes, codes, None if scales is None else (c_float * len(flat))(*scales), max_norm, pair.data_ptr(),
                workspace.data_ptr(), ws_bytes, _lib.stream_ptr(device),
            ),
            "th_grad_norm",
        )  # fmt: skip
    return pair


@torch.no_grad()
def grad_norm(tensors: Sequence[Tensor], grad_scales: Optional[Sequence[float]] = None) -> Tensor:
    r"""2-norm of all given tensors (float32, float16 or bfloat16, on one CUDA device) as one vector, each times its scale: a float32
    scalar on their device, not synchronised. A tensor that is listed twice counts twice."""
    tensors = list(tensors)
    if not tensors:
        raise ValueError("the norm of no tensors has no device")
    if grad_scales is not None and len(grad_scales) != len(tensors):
        raise ValueError(f"{len(grad_scales)} scales for {len(tensors)} tensors")
    return _norm_factor(tensors, grad_scales, math.inf)[0]


@torch.no_grad()
def clip_grad_norm_(parameters: Union[Tensor, Iterable[Tensor]], max_norm: float) -> Tensor:
    r"""Scales the gradients of ``parameters`` in place so that their global 2-norm is at most ``max_norm``, and returns the norm that they
    had (a float32 scalar on their device, not synchronised). As ``torch.nn.utils.clip_grad_norm_``: parameters without a gradient are passed
    over, gradients whose norm is below ``max_norm`` stay as they are (and are not written), those of an infinite or NaN norm become zeros and
    NaN. A parameter that is listed twice is taken once. A gradient that several parameters hold counts for each of them in the norm and is scaled
    once; gradients that overlap otherwise must not be given."""
    max_norm = _check_norm(max_norm)
    parameters = [parameters] if isinstance(parameters, Tensor) else list(parameters)
    grads = list({id(p): p.grad for p in parameters if p.grad is not None}.values())
    if not grads:
        return torch.tensor(0.0)
    pair = _lib.native().clip_grads(grads, max_norm)
    if pair is not NotImplemented:
        return pair[0]
    pair = _norm_factor(grads, None, max_norm)
    grads = list({(g.data_ptr(), g.shape, g.stride(), g.dtype): g for g in grads}.values())  # a gradient that several parameters hold is scaled once
    flat, device = _flat(grads, "clip_grad_norm_")
    pointers, sizes, codes = _lists(flat)
    with torch.cuda.device(device):
        _lib.check(
            _lib.lib().th_scale_tensors(len(flat), pointers, sizes, codes, pair.data_ptr(), _lib.stream_ptr(device)), "th_scale_tensors"
        )
    for g, held in zip(grads, flat):
        if held.data_ptr() != g.data_ptr():
            g.copy_(held)  # a gradient that is not contiguous was scaled in a copy
        else:
            torch.autograd.graph.increment_version(g)
    return pair[0]


def _adam_clipped(params, grads, exp_avgs, exp_avg_sqs, grad_scales, zero_grads, pair, max_norm, step, lr, betas, eps, skipped) -> Tensor:
    r"""The update of parameters of one dtype and device, gradients times their scale times the pair's factor; without a pair that of these
    gradients and ``max_norm``. Returns the pair."""
    done = _lib.native().adam_clipped(
        params, grads, exp_avgs, exp_avg_sqs, None if grad_scales is None else tuple(grad_scales), None if zero_grads is None else tuple(zero_grads), pair,
        max_norm, lr, betas[0], betas[1], eps, step, skipped,
    )  # fmt: skip
    if done is not NotImplemented:
        return done
    n = len(params)
    for p, g, m, v in zip(params, grads, exp_avgs, exp_avg_sqs):
        if g.dtype != p.dtype or p.dtype != params[0].dtype or m.dtype != torch.float32 or v.dtype != torch.float32:
            raise RuntimeError("a clipped update needs parameters and gradients of one dtype and float32 moments")
        if not all(t.is_contiguous() and t.numel() == p.numel() for t in (p, g, m, v)):
            raise RuntimeError("a clipped update needs contiguous parameters, gradients and moments of one size")
    if len({p.data_ptr() for p in params if p.numel()}) != sum(p.numel() > 0 for p in params):
        raise ValueError("a clipped update takes a parameter once")
    device = _lib.require_cuda(*params, *grads, *exp_avgs, *exp_avg_sqs, pair, skipped)
    if pair is None:
        pair = _norm_factor(grads, grad_scales, max_norm)
    pointers = lambda tensors: (c_void_p * n)(*(t.data_ptr() for t in tensors))  # noqa: E731
    with torch.cuda.device(device):
        _lib.check(
            _lib.lib().th_adam_clipped(
                n, pointers(params), pointers(grads), pointers(exp_avgs), pointers(exp_avg_sqs), _lib.i64_array([p.numel() for p in params]),
                (c_float * n)(*([1.0] * n if grad_scales is None else grad_scales)), (c_int * n)(*map(int, zero_grads or [0] * n)), pair.data_ptr(),
                lr, betas[0], betas[1], eps, step, _lib.dtype_code(params[0]), _lib.ptr(skipped), _lib.stream_ptr(device),
            ),
            "th_adam_clipped",
        )  # fmt: skip
    for p in params:
        torch.autograd.graph.increment_version(p)
    return pair


@torch.no_grad()
def clipped_adam_updates(
    params: Sequence[Tensor],
    grads: Sequence[Tensor],
    exp_avgs: Sequence[Tensor],
    exp_avg_sqs: Sequence[Tensor],
    max_norm: float,
    step: int,
    lr: float,
    betas: Tuple[float, float],
    eps: float,
    grad_scales: Optional[Sequence[float]] = None,
    zero_grads: Optional[Sequence[bool]] = None,
    skipped: Optional[Tensor] = None,
) -> Tensor:
    r"""Adam's update in place of parameters of one dtype and device, their gradients clipped to the global norm ``max_norm``; returns the
    norm that they had, each times its scale (a float32 scalar on the device, not synchronised). Any number of contiguous tensors, with
    gradients of the parameters' dtype and float32 moments, each parameter once; ``skipped`` as in ``adam_update``."""
    max_norm, n = _check_norm(max_norm), len(params)
    if n == 0 or any(x is not None and len(x) != n for x in (grads, exp_avgs, exp_avg_sqs, grad_scales, zero_grads)):
        raise ValueError("a clipped update needs as many gradients, moments, scales and flags as parameters, and one at least")
    return _adam_clipped(params, grads, exp_avgs, exp_avg_sqs, grad_scales, zero_grads, None, max_norm, step, lr, betas, eps, skipped)[0]


class FusedAdam(torch.optim.Optimizer):

    def __init__(self, params: Iterable[Tensor], lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8):
        if lr < 0 or eps < 0 or not (0 <= betas[0] < 1) or not (0 <= betas[1] < 1):
            raise ValueError("invalid Adam hyper-parameters")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps))
        self._skipped: Dict[torch.device, Tensor] = {}

    def _skip_counter(self, device: torch.device) -> Tensor:
        counter = self._skipped.get(device)
        if counter is None:
            counter = self._skipped[device] = torch.zeros(1, dtype=torch.int32, device=device)
        return counter

    def skipped_elements(self) -> int:
        r"""Elements passed over so far because their gradient was not finite (reads the device: synchronises)."""
        return sum(int(c.item()) for c in self._skipped.values())

    @torch.no_grad()
    def step(self, grad_scale: float = 1.0, zero_grad: bool = False, max_norm: Optional[float] = None) -> Optional[Tensor]:
        r"""Update every parameter that has a gradient.

        ``grad_scale`` multiplies the stored gradients before use; ``zero_grad`` clears the
        gradient buffers (kept allocated) as part of the update kernel. ``max_norm`` clips the
        scaled gradients of all groups to that global norm; the norm that they had is returned
        (a float32 scalar on the device, not synchronised).
        """
        groups = [(group, [p for p in group["params"] if p.grad is not None]) for group in self.param_groups]
        pair = None
        if max_norm is not None:
            max_norm, grads = _check_norm(max_norm), [p.grad for _, live in groups for p in live]
            pair = _norm_factor(grads, [grad_scale] * len(grads), max_norm) if grads else None
        for group, live in groups:
            # an `update` that knows nothing of clipping is not told of it
            self.update(group, live, [p.grad for p in live], [grad_scale] * len(live), [zero_grad] * len(live), *(() if pair is None else (pair,)))
        return None if pair is None else pair[0]

    def watched(self) -> bool:
        r"""Whether something runs with, or counts, calls of ``step``: hooks of this optimizer or of every optimizer, a scheduler."""
        hooks = (self._optimizer_step_pre_hooks, self._optimizer_step_post_hooks, _global_optimizer_pre_hooks, _global_optimizer_post_hooks)
        return any(hooks) or "step" in self.__dict__

    @torch.no_grad()
    def update(self, group, params, grads, grad_scales, zero_grads, pair: Optional[Tensor] = None) -> None:
        r"""``step`` on explicit gradients of some of ``group``'s parameters, each with its own scale and zero flag; ``pair`` is the norm
        and the factor that clips them."""
        batches: Dict[tuple, list] = {}  # tensors of one dtype, device and step go together
        for p, g, scale, zero in zip(params, grads, grad_scales, zero_grads):
            state = self.state[p]
            if not state:
                state["step"] = 0
                state["exp_avg"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
                state["exp_avg_sq"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
            state["step"] += 1
            batches.setdefault((p.dtype, p.device, state["step"]), []).append((p, g, state["exp_avg"], state["exp_avg_sq"], scale, zero))
        for (_, device, step), batch in batches.items():
            columns = [list(c) for c in zip(*batch)]
            hyper = (step, group["lr"], group["betas"], group["eps"], self._skip_counter(device))
            if pair is None:
                adam_updates(*columns, *hyper)
            else:
                _adam_clipped(*columns, pair, 0.0, *hyper)
