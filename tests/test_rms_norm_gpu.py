r"""Root-mean-square norm, its gradients and its 8-bit output against float64."""
import pytest
import torch

from triton_helpers_b200.layers.int8_linear import Int8Linear, dequantize_rows
from triton_helpers_b200.layers.rms_norm import RMSNorm, rms_norm, rms_norm_int8

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32]
SHAPES = [(1, 1), (3, 8), (4, 7), (2, 5, 33), (9, 512), (6, 1028), (5, 1537), (3, 4096), (2, 12289), (2, 16384), (300, 40), (2, 70000), (3, 33333)]
# the longest chain of float32 additions in a row's sum: 64 of a thread (70 of a long row's), 10 over the team; each is off by 2^-24 at most
ROUNDINGS = 100 * 2.0**-24


def normal(*shape, seed=0, dtype=torch.float32, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)


def reference(x, gain, residual, eps, gy=None, gs=None):
    r"""float64: s, y, and where gy is given the gradients, each with the magnitude that its roundings are relative to."""
    s = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    v, g = s.double(), gain.double()
    rstd = (v.square().mean(-1, keepdim=True) + eps).rsqrt()
    h = v * rstd
    out = {"s": s, "y": h * g}
    if gy is not None:
        dy = gy.double()
        add = gs.double() if gs is not None else torch.zeros_like(v)
        c = (dy * g * h).mean(-1, keepdim=True)
        out["dx"] = rstd * (dy * g - h * c) + add
        out["dx_reach"] = rstd * ((dy * g).abs() + h.abs() * (dy * g * h).abs().mean(-1, keepdim=True)) + add.abs()
        out["dw"] = (dy * h).reshape(-1, v.shape[-1]).sum(0)
        out["dw_reach"] = (dy * h).abs().reshape(-1, v.shape[-1]).sum(0)
    return out


def near(got, want, reach, extra=0.0):
    bound = (ROUNDINGS + extra) * reach + 1.01 * torch.finfo(got.dtype).eps / 2 * want.abs() + (2.0**-25 if got.dtype == torch.float16 else 1e-38)
    return bool(((got.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("added", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_gradients(shape, added, dtype):
    x = normal(*shape, dtype=dtype).requires_grad_(True)
    residual = normal(*shape, seed=1, dtype=dtype).requires_grad_(True) if added else None
    gain = (1 + 0.3 * normal(shape[-1], seed=2)).to(torch.float32 if shape[-1] % 2 else dtype).requires_grad_(True)
    gy, gs = normal(*shape, seed=3, dtype=dtype), normal(*shape, seed=4, dtype=dtype) if added else None
    out = rms_norm(x, gain, residual, 1e-5)
    y, s = out if added else (out, None)
    wanted = [x, gain] + ([residual] if added else [])
    grads = torch.autograd.grad([y, s] if added else [y], wanted, [gy, gs] if added else [gy])
    ref = reference(x.detach(), gain.detach(), None if residual is None else residual.detach(), 1e-5, gy, gs)
    assert y.dtype == dtype and y.shape == x.shape and near(y.detach(), ref["y"], ref["y"].abs())
    if added:
        assert torch.equal(s.detach(), ref["s"]) and torch.equal(grads[0], grads[2])
    rows = x.numel() // shape[-1]
    assert grads[0].dtype == dtype and near(grads[0], ref["dx"], ref["dx_reach"])
    assert grads[1].dtype == gain.dtype and near(grads[1], ref["dw"], ref["dw_reach"], rows * 2.0**-24)


@pytest.mark.parametrize("d", [24, 200])
def test_gradients_against_differences(d):
    # float64 differences of the definition along random directions; the float32 gradients are held to its second-order error
    x, r, gain = normal(3, d).requires_grad_(True), normal(3, d, seed=1).requires_grad_(True), (1 + 0.2 * normal(d, seed=2)).requires_grad_(True)
    gy, gs = normal(3, d, seed=3), normal(3, d, seed=4)
    grads = torch.autograd.grad(rms_norm(x, gain, r, 1e-3), [x, gain, r], [gy, gs])

    def loss(a, w, b):
        s = a + b
        return (s * (s.square().mean(-1, keepdim=True) + 1e-3).rsqrt() * w * gy.double()).sum() + (s * gs.double()).sum()

    at = [t.detach().double() for t in (x, gain, r)]
    for k, g in enumerate(grads):
        direction = normal(*g.shape, seed=7 + k).double()
        h = 1e-5
        up, down = [t.clone() for t in at], [t.clone() for t in at]
        up[k] += h * direction
        down[k] -= h * direction
        slope = (loss(*up) - loss(*down)) / (2 * h)
        assert abs(float((g.double() * direction).sum() - slope)) <= 1e-6 * float((g.double() * direction).abs().sum()) + 1e-7


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,d", [(20000, 64), (5000, 1024), (1200, 4096), (4099, 1537), (3000, 35), (400, 20000)])
def test_many_rows(rows, d, dtype):
    x, gain = normal(rows, d, dtype=dtype).requires_grad_(True), (1 + 0.3 * normal(d, seed=2)).to(dtype).requires_grad_(True)
    gy = normal(rows, d, seed=3, dtype=dtype)
    y = rms_norm(x, gain)
    dx, dw = torch.autograd.grad(y, [x, gain], gy)
    ref = reference(x.detach(), gain.detach(), None, 1e-6, gy)
    assert near(y.detach(), ref["y"], ref["y"].abs()) and near(dx, ref["dx"], ref["dx_reach"])
    assert near(dw, ref["dw"], ref["dw_reach"], rows * 2.0**-24)
    again = torch.autograd.grad(rms_norm(x, gain), [x, gain], gy)
    assert torch.equal(again[0], dx) and torch.equal(again[1], dw)


@pytest.mark.parametrize("added", [False, True])
def test_only_what_is_wanted(added):
    x, r, gain = normal(6, 48), normal(6, 48, seed=1) if added else None, normal(48, seed=2)
    full = [t.clone().requires_grad_(True) if t is not None else None for t in (x, gain, r)]
    out = rms_norm(*full)
    want = torch.autograd.grad(out[0] if added else out, [t for t in full if t is not None], normal(6, 48, seed=3))
    for k, t in enumerate([x, gain] + ([r] if added else [])):
        args = [x, gain, r]
        args[k] = t.clone().requires_grad_(True)
        out = rms_norm(*args)
        (got,) = torch.autograd.grad(out[0] if added else out, [args[k]], normal(6, 48, seed=3))
        assert torch.equal(got, want[k])
    if added:  # the sum alone
        out = rms_norm(*full)
        gs = normal(6, 48, seed=5)
        gx, gr = torch.autograd.grad(out[1], [full[0], full[2]], gs)
        assert torch.equal(gx, gs) and torch.equal(gr, gs)


def test_layouts():
    base, gain = normal(6, 5, 64, dtype=torch.float16), normal(64, seed=2, dtype=torch.float16)
    for x in (base, base.transpose(0, 1), base[:, 1:], base[:, :1].expand(6, 3, 64), base[:0], base[0, 0]):
        y, s = rms_norm(x, gain, x.contiguous())
        ref = reference(x, gain, x, 1e-6)
        assert y.shape == x.shape and y.is_contiguous() and torch.equal(s, ref["s"]) and near(y, ref["y"], ref["y"].abs())
    for x, w in ((base[..., 1:], gain[1:]), (base[..., ::2], gain[::2])):
        y = rms_norm(x, w)
        ref = reference(x, w, None, 1e-6)
        assert near(y, ref["y"], ref["y"].abs())
    x = base.clone().requires_grad_(True)
    wide = normal(6, 5, 128, seed=8, dtype=torch.float16)
    for gy in (wide[..., :64], wide[..., 1:65], wide[:, :, ::2], wide[:, :1, :64].expand(6, 5, 64)):
        (got,) = torch.autograd.grad(rms_norm(x, gain), [x], gy)
        ref = reference(base, gain, None, 1e-6, gy)
        assert near(got, ref["dx"], ref["dx_reach"])
    x = base[:0].clone().requires_grad_(True)
    w = gain.clone().requires_grad_(True)
    dx, dw = torch.autograd.grad(rms_norm(x, w).sum(), [x, w])
    assert dx.shape == x.shape and bool((dw == 0).all())


def test_zero_rows_and_bad_values_stay_alone():
    x = normal(5, 40)
    x[0], x[2, 3], x[3, 1] = 0, float("nan"), float("inf")
    y = rms_norm(x, torch.ones(40, device="cuda"))
    ref = reference(x, torch.ones(40, device="cuda"), None, 1e-6)["y"]
    assert bool((y[0] == 0).all()) and bool(y[2].isnan().all())
    assert torch.equal(y[3].isnan(), ref[3].isnan()) and near(y[[1, 4]], ref[[1, 4]], ref[[1, 4]].abs())
    rows = rms_norm_int8(x, torch.ones(40, device="cuda"))
    back = dequantize_rows(rows)
    assert bool((back[0] == 0).all()) and bool(back[2].isnan().all()) and bool(back[3].isnan().all()) and bool(back[[1, 4]].isfinite().all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("added", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_int8_output(shape, added, dtype):
    x, gain = normal(*shape, dtype=dtype), (1 + 0.3 * normal(shape[-1], seed=2)).to(dtype)
    residual = normal(*shape, seed=1, dtype=dtype) if added else None
    out = rms_norm_int8(x, gain, residual, 1e-5)
    rows, s = out if added else (out, None)
    ref = reference(x, gain, residual, 1e-5)
    if added:
        assert torch.equal(s, ref["s"])
    top = ref["y"].abs().amax(-1, keepdim=True).clamp_min(2.0**-100)
    assert rows.q.shape == x.shape and rows.scale.shape == x.shape[:-1]
    assert bool(((rows.scale.double()[..., None] - top / 127).abs() <= 2 * ROUNDINGS * top / 127).all())
    # half a step, and the roundings of a value of up to 127 steps
    steps = ref["y"] * 127 / top
    assert bool(((rows.q.double() - steps).abs() <= 0.5 + 127 * 3 * ROUNDINGS).all())


def test_together_as_they_are_served():
    norm, linear = RMSNorm(96).cuda().bfloat16(), torch.nn.Linear(96, 160, bias=False).cuda().bfloat16()
    layer = Int8Linear.from_linear(linear)
    x, residual = normal(7, 96, dtype=torch.bfloat16), normal(7, 96, seed=1, dtype=torch.bfloat16)
    with torch.no_grad():
        rows, s = norm.int8(x, residual)
        y = layer(rows, torch.bfloat16)
    ref = reference(x, norm.weight.detach(), residual, 1e-6)
    w = layer.q.double() * layer.scale.double()[:, None]
    want = ref["y"] @ w.t()
    # the rows' half steps: 1 / 254 of the largest value times the weights' sum (and the roundings before them)
    slack = (1 / 254 + 3 * ROUNDINGS) * ref["y"].abs().amax(-1, keepdim=True) * w.abs().sum(1)
    assert torch.equal(s, ref["s"]) and bool(((y.double() - want).abs() <= slack + 2.0**-8 * (want.abs() + slack)).all())


def test_captured_passes():
    x, gain = normal(64, 256).requires_grad_(True), normal(256, seed=2).requires_grad_(True)
    gy = normal(64, 256, seed=3)
    torch.autograd.grad(rms_norm(x, gain), [x, gain], gy)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = rms_norm(x, gain)
        grads = torch.autograd.grad(y, [x, gain], gy)
    with torch.no_grad():
        x.copy_(normal(64, 256, seed=11))
    graph.replay()
    want = rms_norm(x, gain)
    assert torch.equal(y.detach(), want.detach())
    assert all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad(want, [x, gain], gy)))


def test_refusals():
    x, gain = normal(4, 32), normal(32)
    with pytest.raises(AssertionError, match="Weight shape"):
        rms_norm(x, normal(31))
    with pytest.raises(AssertionError, match="Residual"):
        rms_norm(x, gain, normal(1, 32))
    with pytest.raises(TypeError):
        rms_norm(x, gain, x.half())
    with pytest.raises(TypeError):
        rms_norm(x, gain.half())
    with pytest.raises(TypeError):
        rms_norm(x.double(), gain.double())
    with pytest.raises(AssertionError, match="same device"):
        rms_norm(x, gain.cpu())
    with pytest.raises(RuntimeError, match="no gradient"):
        rms_norm_int8(x, gain.clone().requires_grad_(True))


@pytest.mark.parametrize("d", [33, 64, 1028])
def test_memory_around_rows_is_left(d):
    # inputs inside larger tensors at odd places; what lies beside them is neither used nor written
    for dtype in DTYPES:
        wide = normal(9, d + 5, dtype=dtype)
        wide[:, :3], wide[:, d + 3 :] = float("nan"), float("inf")
        x = wide[:, 3 : d + 3]
        gain = normal(d, seed=2, dtype=dtype)
        before = wide.clone()
        y, ref = rms_norm(x, gain), reference(x, gain, None, 1e-6)
        assert near(y, ref["y"], ref["y"].abs())
        assert torch.equal(rms_norm_int8(x, gain).q, rms_norm_int8(x.contiguous(), gain).q)
        leaf, weight = wide.clone().requires_grad_(True), gain.clone().requires_grad_(True)
        gy = normal(9, d, seed=3, dtype=dtype)
        dwide, dw = torch.autograd.grad(rms_norm(leaf[:, 3 : d + 3], weight), [leaf, weight], gy)
        ref = reference(x, gain, None, 1e-6, gy)
        assert near(dwide[:, 3 : d + 3], ref["dx"], ref["dx_reach"]) and bool((dwide[:, :3] == 0).all()) and bool((dwide[:, d + 3 :] == 0).all())
        assert near(dw, ref["dw"], ref["dw_reach"], 9 * 2.0**-24)
        assert torch.equal(wide.nan_to_num(nan=7.0, posinf=8.0), before.nan_to_num(nan=7.0, posinf=8.0))


@pytest.mark.parametrize("d", [48, 1000, 4097])
def test_rows_at_every_start(d):
    # rows that start at each of the places within 16 bytes, alike and not alike
    for dtype in DTYPES:
        base, other, gain = normal(7 * d + 16, dtype=dtype), normal(7 * d + 16, seed=1, dtype=dtype), normal(d, seed=2, dtype=dtype)
        for at in range(0, 9, 1 if d == 48 else 3):
            x, residual = base[at : at + 7 * d].view(7, d), other[at : at + 7 * d].view(7, d)
            for r in (residual, other[: 7 * d].view(7, d)):
                y, s = rms_norm(x, gain, r)
                ref = reference(x, gain, r, 1e-6)
                assert torch.equal(s, ref["s"]) and near(y, ref["y"], ref["y"].abs())
                assert torch.equal(rms_norm_int8(x, gain, r)[0].q, rms_norm_int8(x.clone(), gain, r.clone())[0].q)


def test_offsets_past_32_bits():
    rows, d = 70000, 32768  # 2.3e9 elements
    x = torch.empty(rows, d, device="cuda", dtype=torch.bfloat16)
    x.copy_(normal(1, d, dtype=torch.bfloat16))
    x[-1] = normal(d, seed=5, dtype=torch.bfloat16)
    gain = normal(d, seed=2, dtype=torch.bfloat16)
    y = rms_norm(x, gain)
    assert torch.equal(y[-1], rms_norm(x[-1], gain)) and torch.equal(y[-2], y[0])
    del y
    rows8 = rms_norm_int8(x, gain)
    assert torch.equal(rows8.q[-1], rms_norm_int8(x[-1], gain).q) and torch.equal(rows8.q[-2], rows8.q[0])
