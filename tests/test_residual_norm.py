"""gated_norm_residual: the reference against torch's layer norm, refusals (host), and the kernels against 64 bits (GPU)."""

from __future__ import annotations

import math

import pytest
import torch
import torch.nn.functional as F

from alphatriangle_amd.ops.residual import gated_norm_residual

U32, U16 = 2.0**-24, 2.0**-8
NAMES = ("x", "z", "scale", "post_weight", "post_bias", "pre_weight", "pre_bias", "gate")


def _inputs(shape, gate="full", tx=torch.float32, tz=torch.float32, tp=torch.float32, device="cpu", seed=0, std=1.0, mean=0.0):  # noqa: ANN001
    g = torch.Generator().manual_seed(seed)
    d = shape[-1]

    def r(*s, dt=torch.float32, m=0.0, k=1.0):  # noqa: ANN002
        return (torch.randn(*s, generator=g, dtype=torch.float64) * k + m).to(dt).to(device)

    t = {"x": r(*shape, dt=tx), "z": r(*shape, dt=tz, k=std, m=mean), "scale": r(d, dt=tp, m=0.5, k=0.3), "post_weight": r(d, dt=tp, m=1.0, k=0.2),
         "post_bias": r(d, dt=tp, k=0.2), "pre_weight": r(d, dt=tp, m=1.0, k=0.2), "pre_bias": r(d, dt=tp, k=0.2),
         "gate": {"none": None, "full": r(*shape, dt=tz, k=2.0), "row": r(*shape[:-1], 1, dt=tz, k=2.0)}[gate]}
    return t, r(*shape, dt=tx), r(*shape, dt=tz)


def _call(t, eps=1e-5):  # noqa: ANN001
    return gated_norm_residual(t["x"], t["z"], t["scale"], t["post_weight"], t["post_bias"], t["pre_weight"], t["pre_bias"], gate=t["gate"], eps=eps)


@pytest.mark.parametrize("gate", ["none", "full", "row"])
def test_reference_is_the_definition(gate):
    t, _, _ = _inputs((3, 5, 12), gate, torch.float64, torch.float64, torch.float64)
    y, h = _call(t, 1e-3)
    branch = t["scale"] * F.layer_norm(t["z"], (12,), t["post_weight"], t["post_bias"], 1e-3)
    want = t["x"] + (branch if gate == "none" else branch * torch.sigmoid(t["gate"]))
    assert torch.allclose(y, want, rtol=1e-12, atol=1e-12)
    assert torch.allclose(h, F.layer_norm(want, (12,), t["pre_weight"], t["pre_bias"], 1e-3), rtol=1e-12, atol=1e-12)
    names = [n for n in NAMES if t[n] is not None]

    def f(*a):  # noqa: ANN002
        return _call({**dict(zip(names, a)), **({"gate": None} if gate == "none" else {})}, 1e-3)

    assert torch.autograd.gradcheck(f, [t[n].requires_grad_(True) for n in names])


def test_refusals():
    t, _, _ = _inputs((4, 16))
    _call(t)
    for change in (
        dict(z=t["z"][:3]), dict(x=t["x"].half(), z=t["z"].half()), dict(x=t["x"].bfloat16()), dict(scale=t["scale"][:15]), dict(pre_bias=t["pre_bias"][None]),
        dict(post_weight=t["post_weight"].long()), dict(gate=t["gate"][:, :2]), dict(gate=t["gate"].bfloat16()), dict(gate=t["gate"][0]),
        dict(x=torch.tensor(1.0), z=torch.tensor(1.0)), dict(scale=t["scale"].to("meta")),
    ):
        with pytest.raises(ValueError):
            _call({**t, **change})
    with pytest.raises(ValueError):
        _call(t, 0.0)
    wide, _, _ = _inputs((1, 4097))
    with pytest.raises(ValueError):
        _call(wide)
    none, _, _ = _inputs((1, 0))
    with pytest.raises(ValueError):
        _call(none)


KINDS = [(torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16)]


def _rel(a: torch.Tensor, b: torch.Tensor) -> float:
    n = float(b.norm())
    e = float((a.double() - b).norm())
    return e / n if n else e


def _compare(t, dy, dh, eps=1e-5, grow=1.0):  # noqa: ANN001
    names = [n for n in NAMES if t[n] is not None]
    s = {n: (t[n].detach().clone().requires_grad_(True) if t[n] is not None else None) for n in NAMES}
    y, h = _call(s, eps)
    grads = torch.autograd.grad([y, h], [s[n] for n in names], [dy, dh])
    with torch.no_grad():
        y2, h2 = _call(t, eps)
    assert torch.equal(y, y2) and torch.equal(h, h2)
    w = {n: (t[n].detach().double().requires_grad_(True) if t[n] is not None else None) for n in NAMES}
    ry, rh = _call({n: (v.cpu() if v is not None else None) for n, v in w.items()}, eps)
    rg = torch.autograd.grad([ry, rh], [w[n] for n in names], [dy.double().cpu(), dh.double().cpu()])
    rows, d = t["x"].numel() // t["x"].shape[-1], t["x"].shape[-1]
    # two sums over a row, two over it again for a gradient (each sqrt(d) u), a few elementwise roundings; parameter
    # gradients sum the rows (sqrt(rows) u); `grow`: how far the inputs lift the condition of the row statistics
    wide = U32 * grow * (8 * math.sqrt(d) + 64)
    for n, a, b in [("y", y, ry), ("h", h, rh), *((n, g, e) for n, g, e in zip(names, grads, rg))]:
        b = b.detach().cpu()
        assert a.shape == b.shape
        like = {"y": t["x"], "h": t["z"]}.get(n, t.get(n)).dtype
        assert a.dtype == like, n
        tol = wide + (U16 if like == torch.bfloat16 else 0.0) + (U32 * 8 * math.sqrt(rows) if n not in ("x", "z", "y", "h", "gate") else 0.0)
        assert _rel(a.detach().cpu(), b) <= tol, (n, _rel(a.detach().cpu(), b), tol)
    return y, h, dict(zip(names, grads))


@pytest.mark.gpu
@pytest.mark.parametrize("kinds", KINDS)
@pytest.mark.parametrize("gate", ["none", "full", "row"])
@pytest.mark.parametrize("n,d", [(1, 128), (3, 8), (17, 120), (130, 256), (33, 512), (21, 1000), (9, 2048), (5, 4096), (4, 2056), (40, 129), (7, 1023), (5, 3001),
                                 (50, 7), (2, 4095)])
def test_sizes(kinds, gate, n, d):
    t, dy, dh = _inputs((n, d), gate, *kinds, device="cuda")
    _compare(t, dy, dh)


@pytest.mark.gpu
def test_one_value_rows():
    """Rows of one value: both norms give their bias; gradients of x through the norm vanish exactly."""
    t, dy, dh = _inputs((6, 1), "none", device="cuda")
    s = {n: (v.requires_grad_(True) if v is not None else None) for n, v in t.items()}
    y, h = _call(s)
    assert torch.equal(h, t["pre_bias"].expand(6, 1)) and torch.allclose(y, t["x"] + t["scale"] * t["post_bias"])
    g = torch.autograd.grad([y, h], [s["x"], s["z"], s["pre_weight"]], [dy, dh])
    assert torch.equal(g[0], dy) and bool((g[1] == 0).all()) and bool((g[2] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("kinds", KINDS)
def test_many_rows_and_unused_outputs(kinds):
    t, dy, dh = _inputs((3, 7001, 128), "full", *kinds, device="cuda")  # more rows than one step of every workgroup
    _, _, grads = _compare(t, dy, dh)
    s = {n: v.detach().requires_grad_(True) for n, v in t.items()}
    for pick, zero in ((0, dh), (1, dy)):
        out = _call(s)
        one = torch.autograd.grad(out[pick], [s[n] for n in NAMES], (dy, dh)[pick], allow_unused=True)
        out = _call(s)
        both = torch.autograd.grad(out, [s[n] for n in NAMES], [dy, torch.zeros_like(dh)] if pick == 0 else [torch.zeros_like(dy), dh])
        for a, b in zip(one, both):
            assert torch.equal(a, b)
        del zero
    again = torch.autograd.grad(_call(s), [s[n] for n in NAMES], [dy, dh])
    for n, g in zip(NAMES, again):
        assert torch.equal(g, grads[n]), n


@pytest.mark.gpu
def test_offset_rows_keep_their_statistics():
    """Rows around 100 with a deviation of 1: a one-pass variance would lose four digits."""
    t, dy, dh = _inputs((64, 512), "full", device="cuda", mean=100.0)
    _compare(t, dy, dh, grow=100.0)


@pytest.mark.gpu
def test_closed_and_open_gates_and_bad_rows():
    t, _, _ = _inputs((8, 256), "row", device="cuda")
    t["gate"][0], t["gate"][1], t["gate"][2], t["gate"][3] = -math.inf, math.inf, -200.0, 200.0
    y, h = _call(t)
    assert torch.equal(y[0], t["x"][0]) and torch.equal(y[2], t["x"][2]) and bool(torch.isfinite(y).all())
    clean = (y.clone(), h.clone())
    t["z"][5, 3] = math.nan
    y, h = _call(t)
    keep = [0, 1, 2, 3, 4, 6, 7]
    assert torch.equal(y[keep], clean[0][keep]) and torch.equal(h[keep], clean[1][keep]) and bool(torch.isnan(y[5]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("d", [128, 1000])
def test_strides_alignment_streams_and_parameter_types(d):
    t, dy, dh = _inputs((6, 10, d), "full", torch.float32, torch.bfloat16, torch.bfloat16, device="cuda")
    _compare(t, dy, dh)
    want = _call(t)
    odd = dict(t)
    odd["x"] = torch.cat([t["x"].reshape(-1)[:1], t["x"].reshape(-1)])[1:].view(t["x"].shape)
    odd["z"] = t["z"].transpose(0, 1).contiguous().transpose(0, 1)
    odd["gate"] = torch.stack([t["gate"], t["gate"]], -1)[..., 0]
    odd["scale"] = torch.cat([t["scale"][:1], t["scale"]])[1:]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = _call(odd)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    empty, dy, dh = _inputs((0, d), "full", device="cuda")
    e = {n: v.requires_grad_(True) for n, v in empty.items()}
    y, h = _call(e)
    assert y.shape == (0, d)
    (y.sum() + h.sum()).backward()
    assert bool((e["scale"].grad == 0).all())


@pytest.mark.gpu
def test_captured_forward_and_backward():
    t, dy, dh = _inputs((500, 128), "full", device="cuda")
    static = {n: v.clone() for n, v in t.items()}

    def step():  # noqa: ANN202
        s = {n: v.detach().requires_grad_(True) for n, v in static.items()}
        y, h = _call(s)
        return (y.detach(), h.detach(), *torch.autograd.grad([y, h], [s[n] for n in NAMES], [dy, dh]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in range(3):
        new, _, _ = _inputs((500, 128), "full", device="cuda", seed=seed)
        for n, v in new.items():
            static[n].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        got = [v.clone() for v in captured]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_gradients_by_differences():
    t, dy, dh = _inputs((5, 24), "full", device="cuda")
    s = {n: v.detach().requires_grad_(True) for n, v in t.items()}
    grads = torch.autograd.grad(_call(s), [s[n] for n in NAMES], [dy, dh])
    eps = 2.0**-6

    def value(u):  # noqa: ANN001, ANN202
        y, h = _call(u)
        return float((y.double() * dy.double()).sum() + (h.double() * dh.double()).sum())

    for n, g in zip(NAMES, grads):
        direction = torch.randn(t[n].shape, generator=torch.Generator().manual_seed(1)).cuda()
        direction /= direction.norm()
        slope = (value({**t, n: t[n] + eps * direction}) - value({**t, n: t[n] - eps * direction})) / (2 * eps)
        # truncation: third derivative (at most about 1e2 here) times eps^2 / 6; rounding: u |f| / eps
        assert abs(slope - float((g.double() * direction.double()).sum())) <= eps**2 / 6 * 100 + 64 * U32 / eps * float(dy.norm() + dh.norm()), n
