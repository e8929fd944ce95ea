r"""Operators of networks wider than the fused MLP: what they are asked to do, their plain form and their exact values.

``listed()`` holds twelve cases, from one token, where the launches and the Python around them count, to a training
batch of a wide layer.  ``draw(rng)`` gives further cases of the same ranges.  ``prepare`` makes inputs, weights and
incoming gradients from a seed; ``run`` is one pass: the plain form in elementary float32 operations, or, where ``own``
is true, the calls a user makes of the framework.

Operators (``case["op"]``):

``norm`` / ``norm_grad``   root-mean-square norm of ``x`` (or of ``x + residual``, which is an output too); with gradients
``int8``                   linear layer with 8-bit integer weights; every token is quantised on the way
``norm_int8``              the norm with 8-bit rows as its output, and the 8-bit linear layer that reads them
``ckpt_grad``              linear layer that keeps its input as 8-bit rows for the backward pass: forward and gradients

8-bit rows are a definition in float32: ``a = max(|x|, 2^-100)`` over a row, ``q = rint(x * (127 / a))``, ``scale = a / 127``;
the storage of ``q`` has a row stride that is a multiple of 16 bytes.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6


def _norm(op, rows, d, dtype, residual=True):
    return dict(op=op, rows=rows, d=d, dtype=dtype, residual=residual)


def _linear(op, rows, d, n, dtype, bias=False, residual=False):
    return dict(op=op, rows=rows, d=d, n=n, dtype=dtype, bias=bias, residual=residual)


def listed():
    named = lambda name, case: dict(case, name=name)  # noqa: E731
    return [
        # one token of a residual stream: latency
        named("norm_token", _norm("norm", 1, 4096, "bf16")),
        # a training batch of a wide residual stream
        named("norm_train", _norm("norm_grad", 16384, 4096, "bf16")),
        # features of an odd width in float32, nothing added
        named("norm_odd", _norm("norm_grad", 4099, 1537, "f32", residual=False)),
        # one token through a norm and the layer behind it: latency, and the weights' bytes
        named("serve_token", _linear("norm_int8", 1, 4096, 4096, "bf16", residual=True)),
        # some tens of requests, one token each, through a norm and a widening layer
        named("serve_batch", _linear("norm_int8", 61, 4096, 11008, "f16", residual=True)),
        # one token through a large layer: the weights' bytes
        named("int8_token", _linear("int8", 1, 8192, 8192, "f16")),
        # a ragged batch with odd widths and float32 results
        named("int8_ragged", _linear("int8", 1023, 2500, 1111, "f32", bias=True)),
        # a long prompt through a widening layer
        named("int8_prompt", _linear("int8", 8192, 4096, 16384, "bf16", bias=True)),
        # a small layer trained on a small batch: latency
        named("ckpt_small", _linear("ckpt_grad", 300, 256, 512, "f16", bias=True)),
        # odd rows and widths in training
        named("ckpt_odd", _linear("ckpt_grad", 3001, 1000, 777, "bf16", bias=True)),
        # a training batch of a square layer
        named("ckpt_train", _linear("ckpt_grad", 8192, 4096, 4096, "bf16", bias=True)),
        # a training batch of a widening layer: the largest case
        named("ckpt_wide", _linear("ckpt_grad", 16384, 4096, 16384, "f16")),
    ]


def _size(rng, low, high, multiple):
    r"""A size between ``low`` and ``high``, even over its logarithm; half of them a multiple of ``multiple``."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return max(multiple, n // multiple * multiple) if rng.random() < 0.5 else n


def draw(rng):
    op = rng.choice(("norm", "norm_grad", "int8", "int8", "norm_int8", "ckpt_grad", "ckpt_grad"))
    if op in ("norm", "norm_grad"):
        d = _size(rng, 16, 16384, 64)
        return _norm(op, _size(rng, 1, min(65536, 2**26 // d), 8), d, rng.choice(("f32", "f16", "bf16")), rng.random() < 0.6)
    d, n = _size(rng, 16, 16384, 64), _size(rng, 16, 16384, 64)
    rows = _size(rng, 1 if op != "ckpt_grad" else 8, min(16384, 2**40 // (d * n)), 8)
    dtype = rng.choice(("f32", "f16", "bf16") if op == "int8" else ("f16", "bf16"))
    return _linear(op, rows, d, n, dtype, rng.random() < 0.5, op == "norm_int8" and rng.random() < 0.7)


# ---- inputs -------------------------------------------------------------------------------------------------


def _quantize(x):
    r"""8-bit rows of a matrix as the module's text defines them, in float32."""
    x = x.float()
    a = x.abs().amax(-1, keepdim=True).clamp_min(2.0**-100)
    top = torch.full_like(a, 127.0)  # tensors on both sides: true divisions
    return torch.round(x * (top / a)), a / top


def prepare(case, seed):
    op, rows, d, dtype = case["op"], case["rows"], case["d"], DTYPES[case["dtype"]]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape, scale=1.0: torch.randn(*shape, device="cuda", generator=gen).mul_(scale)  # noqa: E731
    # a residual stream: tokens of different sizes, and some channels larger than the others
    channels = torch.where(torch.rand(d, device="cuda", generator=gen) < 0.01, 6.0, 1.0)
    sizes = torch.exp(0.5 * normal(rows, 1))
    state = {"op": op, "case": case, "x": (normal(rows, d) * channels * sizes).to(dtype)}
    if case["residual"]:
        state["residual"] = (normal(rows, d) * channels).to(dtype)
    if op.startswith("norm"):
        state["gain"] = (1 + 0.1 * normal(d)).to(dtype)
    if op in ("int8", "norm_int8"):
        q, scale = _quantize(normal(case["n"], d, scale=d**-0.5))
        held = torch.zeros(case["n"], -(-d // 16) * 16, dtype=torch.int8, device="cuda")
        state["q"], state["scale"] = held[:, :d].copy_(q), scale.reshape(-1).contiguous()
    elif op == "ckpt_grad":
        state["weight"] = normal(case["n"], d, scale=d**-0.5).to(dtype)
    if case.get("bias"):
        state["bias"] = normal(case["n"], scale=0.1).to(dtype)
    if op == "norm_grad":
        state["grad"] = normal(rows, d).to(dtype)
        if case["residual"]:
            state["grad_sum"] = normal(rows, d).to(dtype)
    elif op == "ckpt_grad":
        state["grad"] = normal(rows, case["n"], scale=0.1).to(dtype)
    if op.endswith("_grad"):
        for name in ("x", "residual", "gain", "weight", "bias"):
            if name in state:
                state[name].requires_grad_(True)
    return state


# ---- one pass: the framework's calls ------------------------------------------------------------------------


def _own(state):
    op, x, bias, residual = state["op"], state["x"], state.get("bias"), state.get("residual")
    if op in ("norm", "norm_grad"):
        from triton_helpers_b200.layers.rms_norm import rms_norm

        outs = rms_norm(x, state["gain"], residual, EPS)
        outs = outs if residual is not None else (outs,)
        if op == "norm":
            return list(outs)
        wanted = [t for t in (x, residual, state["gain"]) if t is not None]
        grads = torch.autograd.grad(outs, wanted, [state["grad"], state["grad_sum"]] if residual is not None else [state["grad"]])
        return [*(t.detach() for t in outs), *grads]
    if op == "ckpt_grad":
        from triton_helpers_b200.layers.checkpointed_linear import checkpointed_linear

        y = checkpointed_linear(x, state["weight"], bias)
        return [y.detach(), *torch.autograd.grad(y, [t for t in (x, state["weight"], bias) if t is not None], state["grad"])]
    from triton_helpers_b200.layers.int8_linear import Int8Rows, int8_linear

    weight = Int8Rows(state["q"], state["scale"])
    if op == "int8":
        return [int8_linear(x, weight, bias)]
    from triton_helpers_b200.layers.rms_norm import rms_norm_int8

    rows = rms_norm_int8(x, state["gain"], residual, EPS)
    rows, added = rows if residual is not None else (rows, None)
    return [int8_linear(rows, weight, bias, dtype=x.dtype), *([] if added is None else [added])]


# ---- one pass: the plain form -------------------------------------------------------------------------------


def _plain_norm(state):
    r"""(sum that is normalised, its normalised values before the gain, 1 / root mean square), float32."""
    x = state["x"].detach()
    s = x if "residual" not in state else (x.float() + state["residual"].detach().float()).to(x.dtype)
    rstd = torch.rsqrt(s.float().square().mean(-1, keepdim=True) + EPS)
    return s, s.float() * rstd, rstd


def _plain_int8(q, scale, state, dtype):
    y = (q @ state["q"].float().t()) * scale * state["scale"]
    return (y + state["bias"].float() if "bias" in state else y).to(dtype)


def _plain(state):
    op, x = state["op"], state["x"].detach()
    dtype = x.dtype
    if op == "int8":
        return [_plain_int8(*_quantize(x), state, dtype)]
    if op == "ckpt_grad":
        w, go = state["weight"].detach().float(), state["grad"].float()
        y = x.float() @ w.t()
        if "bias" in state:
            y = y + state["bias"].detach().float()
        q, scale = _quantize(x)
        outs = [y.to(dtype), (go @ w).to(dtype), (go.t() @ (q * scale)).to(dtype)]
        return outs + ([go.sum(0).to(dtype)] if "bias" in state else [])
    s, unit, rstd = _plain_norm(state)
    gain = state["gain"].detach().float()
    if op == "norm_int8":
        y = _plain_int8(*_quantize(unit * gain), state, dtype)
        return [y] if "residual" not in state else [y, s]
    outs = [(unit * gain).to(dtype)] + ([s] if "residual" in state else [])
    if op == "norm_grad":
        go = state["grad"].float()
        g = go * gain
        dx = rstd * (g - unit * (g * unit).mean(-1, keepdim=True))
        if "residual" in state:
            dx = dx + state["grad_sum"].float()
        dx = dx.to(dtype)
        outs += [dx, dx] if "residual" in state else [dx]
        outs.append((go * unit).sum(0).to(dtype))
    return outs


def run(state):
    if state["op"].endswith("_grad"):
        return _own(state) if own else _plain(state)
    with torch.no_grad():
        return _own(state) if own else _plain(state)


# ---- the same values in 64 bits -----------------------------------------------------------------------------


def exact(case, seed):
    state = prepare(case, seed)
    op, dtype = case["op"], DTYPES[case["dtype"]]
    val = {k: v.detach().double() for k, v in state.items() if torch.is_tensor(v)}
    added = lambda y: y + val["bias"][None, :] if "bias" in val else y  # noqa: E731

    def rows8(v, rounded):
        # the 8-bit integers follow from float32 arithmetic by definition where the values are float32 (or 16-bit) inputs
        top = v.abs().max(dim=1).values.clamp(min=2.0**-100)
        if rounded:
            steps = torch.round(v.float() * (torch.full_like(top, 127).float() / top.float())[:, None])
        else:
            steps = torch.round(v * (127 / top)[:, None])
        return steps.double(), (top / 127)[:, None]

    if op in ("int8", "norm_int8"):
        table = val["q"] * val["scale"][:, None]
    if op == "int8":
        steps, unit = rows8(val["x"], True)
        return [added(unit * torch.matmul(steps, table.T))]
    if op == "ckpt_grad":
        steps, unit = rows8(val["x"], True)
        out = [added(torch.matmul(val["x"], val["weight"].T)), torch.matmul(val["grad"], val["weight"])]
        out.append(torch.matmul((val["grad"] * unit).T, steps))
        return out + ([torch.sum(val["grad"], dim=0)] if "bias" in val else [])
    total = val["x"]
    if "residual" in val:
        total = (val["x"] + val["residual"]).to(dtype).double()  # what is normalised is the sum as it is passed on
    root = torch.sqrt((total * total).sum(dim=1) / case["d"] + EPS)[:, None]
    hat = total / root
    if op == "norm_int8":
        steps, unit = rows8(hat * val["gain"], False)
        return [added(unit * torch.matmul(steps, table.T))] + ([total] if "residual" in val else [])
    out = [hat * val["gain"]] + ([total] if "residual" in val else [])
    if op == "norm_grad":
        g = val["grad"] * val["gain"]
        back = (g - hat * ((g * hat).sum(dim=1) / case["d"])[:, None]) / root
        if "residual" in val:
            back = back + val["grad_sum"]
        out += [back] * (2 if "residual" in val else 1)
        out.append(torch.einsum("rd,rd->d", val["grad"], hat))
    return out


# ---- what a pass cannot do without --------------------------------------------------------------------------


def work(case):
    op, rows, d, n, size = case["op"], case["rows"], case["d"], case.get("n", 0), BYTES[case["dtype"]]
    sides = 2 if case["residual"] else 1
    if op in ("norm", "norm_grad"):
        total, flops = (2 * sides * rows * d + d) * size, 4 * rows * d
        if op == "norm_grad":  # incoming gradients, the gradient that input and residual share, the gain's
            total += ((sides + 1) * rows * d + d) * size
            flops += 12 * rows * d
        return {"bytes": total, "flops": flops}
    bias = n * size if case["bias"] else 0
    if op == "ckpt_grad":
        total = (2 * rows * d + 2 * rows * n + 2 * n * d) * size + 2 * bias
        return {"bytes": total, "flops": 3 * 2 * rows * d * n}
    total = (rows * d + rows * n) * size + n * (d + 4) + bias
    if op == "norm_int8":
        total += (d + (2 * rows * d if case["residual"] else 0)) * size
    return {"bytes": total, "flops": 2 * rows * d * n}
