r"""Operators of 8-bit floating-point layers, of layers of experts and of clipped updates: what they are asked to do, their plain form
and their exact values.

``listed()`` holds twelve cases, from one token, where the launches and the Python around them count, to a long prompt and a training
batch of a wide layer.  ``draw(rng)`` gives further cases of the same ranges.  ``prepare`` makes inputs, weights and incoming gradients
from a seed; ``run`` is one pass: the plain form in elementary float32 operations, or, where ``own`` is true, the calls a user makes of
the framework.

Operators (``case["op"]``):

``float8``                  linear layer on 8-bit floating-point weights, for serving: the tokens are quantised on the way
``float8_grad``             the same product in training, from 16-bit weights: forward and gradients
``experts`` / ``experts_grad``  linear layers of several experts on rows sorted by expert, ragged sizes; with gradients
``clip``                    the 2-norm of a list of gradients; with ``update`` also Adam's update of the parameters, the gradients clipped
                            to that norm

8-bit blocks are a definition in float32: a block is 128 neighbouring inputs of one row, or of 128 rows of a weight, and

    a = max(|x|, 2^-60) over the block      q = e4m3(x * (448 / a))      scale = a / 448

The 8-bit layer in training: ``y = Q(x) Q(w)^T + b`` and ``dx = Q(dy) Q(w)`` with the products of these values, and
``dw = dy^T Q(x)``.  Experts: rows ``ends[e - 1]`` to ``ends[e] - 1`` belong to expert ``e``; rows behind the last end belong to none,
their results and gradients are zero.  Clipped Adam: every gradient is taken times ``min(1, max_norm / (norm + 1e-6))``.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
LR, BETAS, ADAM_EPS, STEP = 1e-3, (0.9, 0.99), 1e-8, 10


def _linear(op, rows, d, n, dtype, bias=False):
    return dict(op=op, rows=rows, d=d, n=n, dtype=dtype, bias=bias)


def _experts(op, rows, behind, experts, d, n, dtype):
    return dict(op=op, rows=rows, behind=behind, experts=experts, d=d, n=n, dtype=dtype)


def _clip(update, tensors, elements, dtype, norm=0.1):
    return dict(op="clip", update=update, tensors=tensors, elements=elements, dtype=dtype, max_norm=norm)


def listed():
    named = lambda name, case: dict(case, name=name)  # noqa: E731
    return [
        # one token through a layer: latency, and the weights' bytes
        named("float8_token", _linear("float8", 1, 4096, 4096, "bf16")),
        # a ragged batch with odd widths and float32 results
        named("float8_ragged", _linear("float8", 1023, 2500, 1111, "f32", bias=True)),
        # a long prompt through a widening layer: the largest case
        named("float8_prompt", _linear("float8", 8192, 4096, 16384, "bf16")),
        # odd rows and widths in training
        named("float8_train_odd", _linear("float8_grad", 3001, 1000, 777, "f16", bias=True)),
        # a training batch of a square layer
        named("float8_train", _linear("float8_grad", 8192, 4096, 4096, "bf16", bias=True)),
        # some tens of tokens, two experts each: most experts get a row or two, and the weights' bytes count
        named("experts_tokens", _experts("experts", 64, 0, 64, 2048, 1024, "bf16")),
        # a prompt through a layer of many experts, with rows behind the last one in a padded buffer
        named("experts_prompt", _experts("experts", 16000, 384, 64, 2048, 2048, "f16")),
        # few experts, odd sizes, in training
        named("experts_odd", _experts("experts_grad", 3001, 5, 7, 520, 333, "f16")),
        # a training batch of a layer of experts
        named("experts_train", _experts("experts_grad", 16384, 0, 32, 2048, 4096, "bf16")),
        # the gradients of a network of many layers, most of them small
        named("clip_norm", _clip(False, 300, 4_000_000, "f32")),
        # a small network's update: latency
        named("clip_small", _clip(True, 24, 100_000, "f16")),
        # a wide network's update: memory
        named("clip_wide", _clip(True, 60, 100_000_000, "bf16")),
    ]


def _size(rng, low, high, multiple):
    r"""A size between ``low`` and ``high``, even over its logarithm; half of them a multiple of ``multiple``."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return max(multiple, n // multiple * multiple) if rng.random() < 0.5 else n


def draw(rng):
    op = rng.choice(("float8", "float8", "float8_grad", "experts", "experts_grad", "clip", "clip"))
    if op == "clip":
        tensors = _size(rng, 1, 400, 1)
        dtype = rng.choice(("f32", "f16", "bf16"))
        return _clip(rng.random() < 0.5, tensors, max(tensors * 8, _size(rng, 1000, 2**26, 64)), dtype, rng.choice((0.1, 1.0, 1000.0)))
    if op in ("float8", "float8_grad"):
        d, n = _size(rng, 16, 16384, 64), _size(rng, 16, 16384, 64)
        low, most = (1, 2**39) if op == "float8" else (8, 2**36)
        rows = _size(rng, low, max(low, min(16384, most // (d * n))), 8)
        return _linear(op, rows, d, n, rng.choice(("f32", "f16", "bf16") if op == "float8" else ("f16", "bf16")), rng.random() < 0.5)
    d, n = _size(rng, 16, 4096, 64), _size(rng, 16, 4096, 64)
    experts = _size(rng, 1, max(1, min(128, 2**28 // (d * n))), 1)
    rows = _size(rng, 1, min(16384, 2**36 // (d * n)), 8)
    return _experts(op, rows, rng.choice((0, 0, 3, 128)), experts, d, n, rng.choice(("f16", "bf16")))


# ---- inputs -------------------------------------------------------------------------------------------------


def _blocks(x, rows):
    r"""``(q, scale)`` of a matrix in 8-bit blocks of ``rows`` rows (1 or 128) and 128 columns, q as the float32 values it stands for."""
    m, k = x.shape
    held = torch.zeros(-(-m // rows) * rows, -(-k // 128) * 128, device=x.device)
    held[:m, :k] = x
    held = held.view(held.shape[0] // rows, rows, -1, 128)
    a = held.abs().amax((1, 3), keepdim=True).clamp_min(2.0**-60)
    top = torch.full_like(a, 448.0)  # tensors on both sides: true divisions
    q = (held * (top / a)).to(torch.float8_e4m3fn).float()
    return q.view(held.shape[0] * rows, -1)[:m, :k], (a / top)[:, 0, :, 0]


def _sizes(case, gen):
    r"""Rows of each expert: uneven, some of them without any."""
    weights = torch.exp(0.8 * torch.randn(case["experts"], device="cuda", generator=gen))
    picks = torch.multinomial(weights, case["rows"], replacement=True, generator=gen)
    return torch.bincount(picks, minlength=case["experts"])


def _lengths(case):
    r"""Elements of each tensor of a list: a few large ones and many small ones, odd numbers among them."""
    count, left = case["tensors"], case["elements"]
    shares = [1.0 / (1 + i) ** 1.5 for i in range(count)]
    return [max(1, int(left * s / sum(shares))) for s in shares]


def prepare(case, seed):
    op, dtype = case["op"], DTYPES[case["dtype"]]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape, scale=1.0: torch.randn(*shape, device="cuda", generator=gen).mul_(scale)  # noqa: E731
    state = {"op": op, "case": case}
    if op == "clip":
        # tensors of one buffer each for parameters, gradients and moments, as a program keeps them that sums gradients over ranks at once
        lengths = _lengths(case)
        starts = [0]
        for n in lengths:
            starts.append(starts[-1] + -(-n // 64) * 64)
        views = lambda flat: [flat[a : a + n] for a, n in zip(starts, lengths)]  # noqa: E731
        flat = {"grad": normal(starts[-1], scale=0.02).to(dtype)}
        if case["update"]:
            flat["param"] = normal(starts[-1]).to(dtype)
            flat["exp_avg"] = normal(starts[-1], scale=0.01)
            flat["exp_avg_sq"] = normal(starts[-1], scale=0.01).square_()
        state["flat"] = flat
        state.update({name: views(t) for name, t in flat.items()})
        return state
    rows, d, n = case["rows"] + case.get("behind", 0), case["d"], case["n"]
    # a residual stream: tokens of different sizes, and some channels larger than the others
    channels = torch.where(torch.rand(d, device="cuda", generator=gen) < 0.01, 6.0, 1.0)
    sizes = torch.exp(0.5 * normal(rows, 1))
    state["x"] = (normal(rows, d) * channels * sizes).to(dtype)
    if op == "float8":
        q, scale = _blocks(normal(n, d, scale=d**-0.5), 128)
        held = torch.zeros(n, -(-d // 16) * 16, device="cuda").to(torch.float8_e4m3fn)
        held[:, :d] = q.to(torch.float8_e4m3fn)
        state["q"], state["scale"] = held[:, :d], scale.contiguous()
    elif op == "float8_grad":
        state["weight"] = normal(n, d, scale=d**-0.5).to(dtype)
    else:
        state["weight"] = normal(case["experts"], n, d, scale=d**-0.5).to(dtype)
        state["ends"] = _sizes(case, gen).cumsum(0).to(torch.int32)
    if case.get("bias"):
        state["bias"] = normal(n, scale=0.1).to(dtype)
    if op.endswith("_grad"):
        state["grad"] = (normal(rows, n, scale=0.1) * torch.exp(0.5 * normal(rows, 1))).to(dtype)
        for name in ("x", "weight", "bias"):
            if name in state:
                state[name].requires_grad_(True)
    return state


# ---- one pass: the framework's calls ------------------------------------------------------------------------


def _own(state):
    op, x, bias = state["op"], state.get("x"), state.get("bias")
    if op == "clip" and not state["case"]["update"]:
        from triton_helpers_b200.optim import grad_norm

        return [grad_norm(state["grad"])]
    if op == "clip":
        from triton_helpers_b200.optim import clipped_adam_updates

        norm = clipped_adam_updates(
            state["param"], state["grad"], state["exp_avg"], state["exp_avg_sq"], state["case"]["max_norm"], STEP, LR, BETAS, ADAM_EPS
        )
        return [norm, state["flat"]["param"], state["flat"]["exp_avg"], state["flat"]["exp_avg_sq"]]
    if op == "float8":
        from triton_helpers_b200.layers.float8_linear import Float8Blocks, float8_linear

        return [float8_linear(x, Float8Blocks(state["q"], state["scale"]), bias)]
    if op == "float8_grad":
        from triton_helpers_b200.layers.float8_linear import float8_training_linear

        y = float8_training_linear(x, state["weight"], bias)
    else:
        from triton_helpers_b200.layers.expert_linear import expert_linear

        y = expert_linear(x, state["weight"], state["ends"])
        if op == "experts":
            return [y]
    return [y.detach(), *torch.autograd.grad(y, [t for t in (x, state["weight"], bias) if t is not None], state["grad"])]


# ---- one pass: the plain form -------------------------------------------------------------------------------


def _stands_for(x, rows):
    q, scale = _blocks(x.float(), rows)
    return _times(q, scale, rows)


def _times(q, scale, rows):
    return q * scale.repeat_interleave(rows, 0)[: q.shape[0]].repeat_interleave(128, 1)[:, : q.shape[1]]


def _plain_float8(state):
    x, dtype = state["x"].detach(), state["x"].dtype
    xs = _stands_for(x, 1)
    ws = _times(state["q"].float(), state["scale"], 128) if state["op"] == "float8" else _stands_for(state["weight"].detach(), 128)
    y = xs @ ws.t()
    if "bias" in state:
        y = y + state["bias"].detach().float()
    if state["op"] == "float8":
        return [y.to(dtype)]
    go = state["grad"]
    outs = [y.to(dtype), (_stands_for(go, 1) @ ws).to(dtype), (go.float().t() @ xs).to(dtype)]
    return outs + ([go.float().sum(0).to(dtype)] if "bias" in state else [])


def _plain_experts(state):
    x, w, ends, dtype = state["x"].detach(), state["weight"].detach().float(), state["ends"].long(), state["x"].dtype
    # every expert's rows in a matrix of their own, filled up with zeros
    row = torch.arange(x.shape[0], device="cuda")
    expert = torch.searchsorted(ends, row, right=True)
    starts = torch.cat([ends.new_zeros(1), ends])
    at = row - starts[expert]
    belongs = expert < w.shape[0]
    row, expert, at = row[belongs], expert[belongs], at[belongs]
    most = int((starts[1:] - starts[:-1]).max())

    def apart(t):
        held = torch.zeros(w.shape[0], most, t.shape[1], device="cuda")
        held[expert, at] = t[row].float()
        return held

    def together(held):
        out = torch.zeros(x.shape[0], held.shape[2], device="cuda")
        out[row] = held[expert, at]
        return out.to(dtype)

    xs = apart(x)
    y = together(torch.bmm(xs, w.transpose(1, 2)))
    if state["op"] == "experts":
        return [y]
    go = apart(state["grad"])
    return [y, together(torch.bmm(go, w)), torch.bmm(go.transpose(1, 2), xs).to(dtype)]


def _plain_clip(state):
    flat, (b1, b2) = state["flat"], BETAS
    grads = [g.float() for g in state["grad"]]
    norm = torch.sqrt(torch.stack([g.square().sum() for g in grads]).sum())
    if not state["case"]["update"]:
        return [norm]
    factor = (state["case"]["max_norm"] / (norm + 1e-6)).clamp_max(1.0)
    m = [torch.add(b1 * m, (1 - b1) * factor * g) for m, g in zip(state["exp_avg"], grads)]
    v = [torch.add(b2 * v, (1 - b2) * (factor * g).square()) for v, g in zip(state["exp_avg_sq"], grads)]
    root, rate = math.sqrt(1 - b2**STEP), LR / (1 - b1**STEP)
    p = [(p.float() - rate * (a / (b.sqrt() / root + ADAM_EPS))).to(p.dtype) for p, a, b in zip(state["param"], m, v)]
    for name, new in (("param", p), ("exp_avg", m), ("exp_avg_sq", v)):
        torch._foreach_copy_(state[name], new)
    return [norm, flat["param"], flat["exp_avg"], flat["exp_avg_sq"]]


def _plain(state):
    op = state["op"]
    return _plain_clip(state) if op == "clip" else _plain_float8(state) if op.startswith("float8") else _plain_experts(state)


def run(state):
    if state["op"].endswith("_grad"):
        return _own(state) if own else _plain(state)
    with torch.no_grad():
        return _own(state) if own else _plain(state)


# ---- the same values in 64 bits -----------------------------------------------------------------------------


def _exact_blocks(v, tall):
    r"""What a matrix in 8-bit blocks stands for: e4m3 by arithmetic, on the float32 quotients that the definition names."""
    m, k = v.shape
    i = torch.arange(m, device=v.device) // tall
    j = torch.arange(k, device=v.device) // 128
    index = (i[:, None] * (int(j[-1]) + 1) + j[None, :]).reshape(-1)
    top = torch.zeros((int(i[-1]) + 1) * (int(j[-1]) + 1), dtype=torch.float64, device=v.device)
    top = top.scatter_reduce(0, index, v.abs().reshape(-1), "amax").clamp(min=2.0**-60)
    factor = torch.full_like(top, 448).float() / top.float()
    value = (v.float() * factor[index].view(m, k)).double()
    step = torch.exp2(torch.floor(torch.log2(value.abs().clamp(min=2.0**-6))) - 3)  # eight steps from a power of two to the next
    unit = (top.float() / torch.full_like(top, 448).float()).double()
    return torch.clamp(torch.round(value / step) * step, -448, 448) * unit[index].view(m, k)


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "clip":
        total = math.sqrt(sum(float(torch.dot(g.double(), g.double())) for g in state["grad"]))
        norm = torch.tensor(total, dtype=torch.float64, device="cuda")
        if not case["update"]:
            return [norm]
        flat = {name: t.double() for name, t in state["flat"].items()}
        inside = torch.zeros_like(flat["grad"], dtype=torch.bool)
        at = 0
        for n in _lengths(case):  # what lies between the tensors stays as it was
            inside[at : at + n] = True
            at += -(-n // 64) * 64
        g = flat["grad"] * min(1.0, case["max_norm"] / (total + 1e-6))
        m = flat["exp_avg"].lerp(g, 1 - BETAS[0])
        v = flat["exp_avg_sq"].lerp(g * g, 1 - BETAS[1])
        p = flat["param"] - LR * (m / (1 - BETAS[0] ** STEP)) / ((v / (1 - BETAS[1] ** STEP)).sqrt() + ADAM_EPS)
        return [norm, *(torch.where(inside, new, flat[name]) for name, new in (("param", p), ("exp_avg", m), ("exp_avg_sq", v)))]
    val = {k: v.detach().double() for k, v in state.items() if torch.is_tensor(v) and v.dtype != torch.int32}
    if op.startswith("float8"):
        x = _exact_blocks(val["x"], 1)
        if op == "float8":
            unit = torch.kron(val["scale"], torch.ones(128, 128, dtype=torch.float64, device="cuda"))
            w = val["q"] * unit[: case["n"], : case["d"]]
        else:
            w = _exact_blocks(val["weight"], 128)
        y = torch.einsum("rd,nd->rn", x, w)
        out = [y + val["bias"][None, :] if "bias" in val else y]
        if op == "float8_grad":
            out += [torch.einsum("rn,nd->rd", _exact_blocks(val["grad"], 1), w), torch.einsum("rn,rd->nd", val["grad"], x)]
            out += [torch.sum(val["grad"], dim=0)] if "bias" in val else []
        return out
    y = torch.zeros(val["x"].shape[0], case["n"], dtype=torch.float64, device="cuda")
    dx, dw = torch.zeros_like(val["x"]), torch.zeros_like(val["weight"])
    start = 0
    for e, end in enumerate(state["ends"].tolist()):
        mine = slice(start, end)
        y[mine] = torch.matmul(val["x"][mine], val["weight"][e].T)
        if op == "experts_grad":
            dx[mine] = torch.matmul(val["grad"][mine], val["weight"][e])
            dw[e] = torch.matmul(val["grad"][mine].T, val["x"][mine])
        start = end
    return [y] if op == "experts" else [y, dx, dw]


# ---- what a pass cannot do without --------------------------------------------------------------------------


def work(case):
    op, size = case["op"], BYTES[case["dtype"]]
    if op == "clip":
        n = sum(_lengths(case))
        return {"bytes": n * size + 4, "flops": 2 * n} if not case["update"] else {"bytes": n * (3 * size + 16) + 4, "flops": 16 * n}
    rows, d, n = case["rows"], case["d"], case["n"]
    product = 2 * rows * d * n
    if op in ("float8", "float8_grad"):
        bias = n * size if case["bias"] else 0
        if op == "float8":
            return {"bytes": (rows * d + rows * n) * size + n * d + 4 * -(-n // 128) * -(-d // 128) + bias, "flops": product}
        return {"bytes": 2 * (rows * d + rows * n + n * d) * size + 2 * bias, "flops": 3 * product}
    # experts that no row goes to are not read: with rows dealt out evenly so many have one
    used = case["experts"] * (1 - (1 - 1 / case["experts"]) ** rows)
    every = rows + case["behind"]  # results of rows behind the last are written too
    if op == "experts":
        return {"bytes": (rows * d + every * n + used * n * d) * size + 4 * case["experts"], "flops": product}
    total = (rows * d + every * n + rows * n + every * d + used * n * d + case["experts"] * n * d) * size + 4 * case["experts"]
    return {"bytes": total, "flops": 3 * product}
