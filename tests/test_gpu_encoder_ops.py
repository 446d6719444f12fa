"""Encoder attention operators (relative position bias, two maps) on the GPU against the same formulas in 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U32, U16 = 2.0**-24, 2.0**-8  # half a step of fp32 / bf16, relative


def _tol(dtype: torch.dtype, d: int, lq: int, lk: int) -> float:
    """Relative 2-norm error allowed on an output or gradient.

    fp32: rounding errors of a sum of n products grow like sqrt(n) u; a score (n = d) enters exponentially, the sums
    over keys / queries follow, and a gradient passes through two such chains: u (8 sqrt(d) + 8 sqrt(max(lq, lk)) + 64).
    bf16: one rounding of the probability (or score gradient) that meets the other operand, one of the result: 2 * 2^-8;
    the 32-bit part above is far below."""
    wide = U32 * (8 * math.sqrt(d) + 8 * math.sqrt(max(lq, lk)) + 64)
    return wide if dtype == torch.float32 else 2 * U16 + wide


def _rel(x: torch.Tensor, y: torch.Tensor) -> float:
    y = y.double()
    y = y.detach()
    n = float(y.norm())
    e = float((x.detach().double() - y).norm())
    return e / n if n else e


def _inputs(dtype, maps, b, lq, lk, h, kv, d, buckets, seed=0, std=1.0):  # noqa: ANN001
    g = torch.Generator(device="cuda").manual_seed(seed)

    def r(*s, dt=dtype, m=1.0):  # noqa: ANN002
        return (torch.randn(*s, generator=g, device="cuda") * m).to(dt)

    return {
        "q": r(b, lq, h * maps, d, m=std), "k": r(b, lk, kv * maps, d, m=std), "v": r(b, lk, kv, d * maps),
        "table": r(buckets.num_buckets, h * maps, dt=torch.float32, m=0.5) if buckets else None,
        "lam": (torch.rand(h, generator=g, device="cuda") * 0.6 + 0.1) if maps == 2 else None,
        "dout": r(b, lq, h, d * maps),
    }


def _call(t, buckets, mask, off):  # noqa: ANN001
    from alphatriangle_amd.ops import attention as A

    if t["lam"] is None:
        return A.relative_attention(t["q"], t["k"], t["v"], t["table"], buckets, key_mask=mask, query_offset=off)
    return A.differential_attention(t["q"], t["k"], t["v"], t["lam"], t["table"], buckets, key_mask=mask, query_offset=off)


def _compare(inp, buckets, mask=None, off=0):  # noqa: ANN001
    from alphatriangle_amd.ops.attention import attention_reference

    names = [n for n in ("q", "k", "v", "table", "lam") if inp[n] is not None]
    t = dict(inp)
    for n in names:
        t[n] = inp[n].detach().clone().requires_grad_(True)
    out = _call(t, buckets, mask, off)
    grads = torch.autograd.grad(out, [t[n] for n in names], inp["dout"])
    with torch.no_grad():
        plain = _call(inp, buckets, mask, off)
    w = {n: (inp[n].double().requires_grad_(True) if n in names else None) for n in ("q", "k", "v", "table", "lam")}
    ref = attention_reference(w["q"], w["k"], w["v"], w["lam"], w["table"], buckets, mask, inp["q"].shape[3] ** -0.5, off)
    rg = torch.autograd.grad(ref, [w[n] for n in names], inp["dout"].double())
    torch.cuda.synchronize()
    one_bucket = buckets is not None and buckets.pairs(inp["q"].shape[1], inp["k"].shape[1], off).unique().numel() == 1
    dt, d, lq, lk = inp["q"].dtype, inp["q"].shape[3], inp["q"].shape[1], inp["k"].shape[1]
    if dt == torch.float32:
        assert torch.equal(plain, out), "with and without a backward pass to come"
    assert _rel(plain, ref) <= _tol(dt, d, lq, lk), ("out without gradients", _rel(plain, ref))
    assert _rel(out, ref) <= _tol(dt, d, lq, lk), ("out", _rel(out, ref))
    for n, g, e in zip(names, grads, rg):
        assert g.dtype == t[n].dtype and g.shape == t[n].shape
        # sums over every pair whose terms cancel (softmax gradients add up to zero in a row): 16 times the room
        tol = 16 * _tol(torch.float32, d, lq, lk) if n in ("table", "lam") else _tol(dt, d, lq, lk)
        if (lk == 1 and n in ("q", "k", "table")) or (n == "table" and one_bucket):
            # zero by definition (a row's score gradients add up to delta - delta): what is left are roundings of the terms
            # p (dP - delta), |dP| <= sum |dO| |v|, over the rows that meet in one value
            rows = inp["dout"].shape[0] * lq
            assert float((g.double() - e).abs().max()) <= 64 * U32 * d * float(inp["dout"].abs().max()) * rows
        else:
            assert _rel(g, e) <= tol, (n, _rel(g, e), tol)
    return out, dict(zip(names, grads))


def _plan(kind):  # noqa: ANN001
    from alphatriangle_amd.ops.attention import RelativeBuckets

    if kind is None:
        return None
    return RelativeBuckets.board(*kind, device="cuda") if isinstance(kind, tuple) else RelativeBuckets.log(32, kind, device="cuda")


BOTH = [torch.float32, torch.bfloat16]


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("maps,d", [(1, 8), (1, 32), (1, 40), (1, 64), (1, 96), (1, 128), (2, 8), (2, 32), (2, 48), (2, 64)])
def test_head_widths(dtype, maps, d):
    b, l, h = 2, 97, 3
    _compare(_inputs(dtype, maps, b, l, l, h, h, d, _plan(20)), _plan(20))


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("maps", [1, 2])
@pytest.mark.parametrize("lq,lk", [(1, 1), (1, 2), (2, 1), (1, 64), (16, 17), (63, 65), (64, 64), (65, 63), (128, 129), (1, 700), (130, 700), (700, 5)])
def test_lengths(dtype, maps, lq, lk):
    p = _plan(128)
    _compare(_inputs(dtype, maps, 2, lq, lk, 2, 2, 32, p), p)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("maps", [1, 2])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 9), (9, 1), (3, 5), (8, 15), (12, 21), (20, 30)])
def test_boards(dtype, maps, rows, cols):
    p = _plan((rows, cols))
    n = rows * cols
    _compare(_inputs(dtype, maps, 2, n, n, 2, 2, 32, p), p)


@pytest.mark.parametrize("dtype", BOTH)
def test_widest_board(dtype):
    """1024 cells, 3969 relative positions, two 64-wide maps: the sums by position take one LDS row for all waves."""
    p = _plan((32, 32))
    _compare(_inputs(dtype, 2, 1, 1024, 1024, 1, 1, 64, p), p)
    _compare(_inputs(dtype, 1, 1, 1024, 1024, 2, 1, 128, p), p)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("maps", [1, 2])
@pytest.mark.parametrize("h,kv", [(4, 1), (6, 2), (3, 3)])
def test_shared_heads(dtype, maps, h, kv):
    p = _plan(16)
    _compare(_inputs(dtype, maps, 2, 70, 150, h, kv, 32, p), p)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("maps", [1, 2])
def test_no_bias_and_long_saturated(dtype, maps):
    if maps == 2:
        _compare(_inputs(dtype, 2, 1, 300, 513, 2, 1, 32, None), None)
    p = _plan(9)  # nearly every pair clamped
    _compare(_inputs(dtype, maps, 1, 600, 520, 2, 2, 32, p), p)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("maps", [1, 2])
def test_masks(dtype, maps):
    """Ragged, scattered, whole tiles out, a sample without any key; masked rows hold NaN and infinities."""
    p = _plan(32)
    b, lq, lk = 4, 75, 400
    inp = _inputs(dtype, maps, b, lq, lk, 4, 2, 32, p)
    mask = torch.zeros(b, lk, dtype=torch.bool, device="cuda")
    mask[0, :333] = True
    mask[1] = torch.rand(lk, generator=torch.Generator().manual_seed(1)).cuda() < 0.3
    mask[2, 200] = True
    clean_out, clean = _compare(inp, p, mask)
    assert bool((clean_out[3] == 0).all()) and all(bool((clean[n][3] == 0).all()) for n in ("q", "k", "v"))
    assert bool((clean["k"][~mask] == 0).all()) and bool((clean["v"][~mask] == 0).all())
    bad = dict(inp)
    for n, x in (("k", math.nan), ("v", math.inf)):
        bad[n] = inp[n].clone()
        bad[n][~mask] = x
    bad["k"][3] = -math.inf
    names = [n for n in ("q", "k", "v", "table", "lam") if inp[n] is not None]
    t = {**bad, **{n: bad[n].detach().clone().requires_grad_(True) for n in names}}
    out = _call(t, p, mask, 0)
    grads = torch.autograd.grad(out, [t[n] for n in names], inp["dout"])
    assert torch.equal(out, clean_out)
    for n, g in zip(names, grads):
        assert torch.equal(g, clean[n]), n


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("maps", [1, 2])
def test_table_of_infinities_and_lowest_values(dtype, maps):
    """Buckets of -inf take their pairs out (a row may lose all of them: zeros); buckets of the lowest finite value leave a row that
    has nothing else uniform."""
    p = _plan(16)
    inp = _inputs(dtype, maps, 2, 90, 40, 2, 2, 32, p)
    near = p.pairs(90, 40)
    inp["table"][near[0, 0], :] = -math.inf
    out, g = _compare(inp, p)
    assert bool(torch.isfinite(out).all()) and all(bool(torch.isfinite(x).all()) for x in g.values())
    inp["table"][:] = -math.inf
    out = _call(inp, p, None, 0)
    assert bool((out == 0).all())
    inp["table"][:] = torch.finfo(torch.float32).min
    t = {n: (x.clone().requires_grad_(True) if n != "dout" and x is not None else x) for n, x in inp.items()}
    out = _call(t, p, None, 0)
    mean = inp["v"].double().mean(1, keepdim=True).expand(-1, 90, -1, -1)
    want = mean if maps == 1 else mean * (1 - inp["lam"].double().view(1, 1, -1, 1))
    assert _rel(out, want) <= _tol(dtype, 32, 90, 40)
    dv = torch.autograd.grad(out, t["v"], inp["dout"])[0]
    each = inp["dout"].double().sum(1, keepdim=True).expand(-1, 40, -1, -1) / 40
    assert _rel(dv, each if maps == 1 else each * (1 - inp["lam"].double().view(1, 1, -1, 1))) <= _tol(dtype, 32, 90, 40)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("maps", [1, 2])
def test_one_token_against_a_cache(dtype, maps):
    """Single queries behind caches of different lengths (split keys), with an int and a per-sample offset."""
    p = _plan(128)
    b, lk = 3, 5000
    inp = _inputs(dtype, maps, b, 1, lk, 4, 2, 64, p)
    lengths = torch.tensor([5000, 1, 2777], device="cuda")
    mask = torch.arange(lk, device="cuda")[None] < lengths[:, None]
    _compare(inp, p, mask, (lengths - 1).to(torch.int32))
    _compare(inp, p, None, lk - 1)
    _compare(inp, p, None, 1 << 29)  # everything clamped


@pytest.mark.parametrize("dtype", BOTH)
def test_strides_orders_and_alignment(dtype):
    p = _plan(24)
    b, l, h, d = 3, 77, 2, 32
    packed = torch.randn(l, b, 3, h, d, device="cuda").to(dtype)  # token-major packed projections, read in place
    q, k, v = (packed[:, :, i].transpose(0, 1) for i in range(3))
    base = _inputs(dtype, 1, b, l, l, h, h, d, p)
    inp = {**base, "q": q, "k": k, "v": v}
    want, grads = _compare({**base, "q": q.contiguous(), "k": k.contiguous(), "v": v.contiguous()}, p)
    t = {n: x.detach().requires_grad_(True) for n, x in inp.items() if n in ("q", "k", "v", "table")}
    out = _call({**inp, **t}, p, None, 0)
    assert torch.equal(out, want) and out.stride(1) > out.stride(0)
    got = torch.autograd.grad(out, list(t.values()), base["dout"].transpose(0, 1).contiguous().transpose(0, 1))
    for n, g in zip(t, got):
        assert torch.equal(g, grads[n]), n
    # rows that start off a 16-byte boundary, a last dimension that is not contiguous, an expanded batch
    odd = torch.randn(b * l * h * d + 1, device="cuda").to(dtype)[1:].view(b, l, h, d)
    wide = torch.randn(b, l, h, 2 * d, device="cuda").to(dtype)[..., ::2]
    one = torch.randn(1, l, h, d, device="cuda").to(dtype).expand(b, -1, -1, -1)
    x = _call({**inp, "q": odd, "k": wide, "v": one}, p, None, 0)
    y = _call({**inp, "q": odd.clone(), "k": wide.clone(), "v": one.clone()}, p, None, 0)
    assert torch.equal(x, y)
    rows = torch.zeros(b, 2 * l, dtype=torch.bool, device="cuda")
    rows[:, ::3] = True
    m = rows[:, ::2]
    assert torch.equal(_call(inp, p, m, 0), _call(inp, p, m.contiguous(), 0))


def test_repeatable_and_on_another_stream():
    p = _plan((8, 15))
    inp = _inputs(torch.bfloat16, 2, 16, 120, 120, 2, 2, 32, p)
    first = _compare(inp, p)
    again = _compare(inp, p)
    assert torch.equal(first[0], again[0]) and all(torch.equal(first[1][n], again[1][n]) for n in first[1])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = _compare(inp, p)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(first[0], other[0]) and all(torch.equal(first[1][n], other[1][n]) for n in first[1])


def test_captured_forward_and_backward():
    """One graph of a training call, replayed on new inputs with eager calls and synchronizations in between."""
    p = _plan(64)
    inp = _inputs(torch.float32, 1, 2, 200, 900, 4, 2, 32, p)
    names = ("q", "k", "v", "table")
    static = {n: (x.clone() if x is not None else None) for n, x in inp.items()}
    mask = torch.ones(2, 900, dtype=torch.bool, device="cuda")

    def step():  # noqa: ANN202
        t = {**static, **{n: static[n].detach().requires_grad_(True) for n in names}}
        out = _call(t, p, mask, 0)
        return (out.detach(), *torch.autograd.grad(out, [t[n] for n in names], static["dout"]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in range(4):
        new = _inputs(torch.float32, 1, 2, 200, 900, 4, 2, 32, p, seed=seed)
        mask.fill_(True)
        mask[1, 100 * seed :] = False
        for n, x in new.items():
            if x is not None:
                static[n].copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in captured]
        want = step()
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x, y)


def test_gradients_by_differences():
    """Central differences of a random functional of the output in every argument (fp32, step 2^-6)."""
    p = _plan(12)
    for maps in (1, 2):
        inp = _inputs(torch.float32, maps, 1, 9, 14, 2, 1, 16, p, std=0.5)
        names = [n for n in ("q", "k", "v", "table", "lam") if inp[n] is not None]
        t = {**inp, **{n: inp[n].clone().requires_grad_(True) for n in names}}
        grads = torch.autograd.grad(_call(t, p, None, 0), [t[n] for n in names], inp["dout"])
        eps = 2.0**-6
        for n, g in zip(names, grads):
            direction = torch.randn_like(inp[n])
            direction /= direction.norm()
            vals = []
            for s in (eps, -eps):
                out = _call({**inp, n: inp[n] + s * direction}, p, None, 0)
                vals.append(float((out.double() * inp["dout"].double()).sum()))
            slope = (vals[0] - vals[1]) / (2 * eps)
            want = float((g.double() * direction.double()).sum())
            # truncation: third derivative times eps^2 / 6 (order of |dout| |v| = 1e2 at most); rounding: u |f| / eps
            assert abs(slope - want) <= eps**2 / 6 * 100 + 64 * U32 / eps * float(inp["dout"].norm()), (maps, n, slope, want)


@pytest.mark.parametrize("maps", [1, 2])
def test_empty_calls(maps):
    p = _plan(16)
    for b, lq, lk in ((0, 4, 4), (2, 0, 4), (2, 4, 0)):
        inp = _inputs(torch.float32, maps, b, lq, lk, 2, 2, 32, p)
        t = {n: (x.clone().requires_grad_(True) if n != "dout" and x is not None else x) for n, x in inp.items()}
        out = _call(t, p, None, 0)
        assert out.shape == inp["dout"].shape and bool((out == 0).all())
        out.sum().backward()
        assert all(x.grad is None or bool((x.grad == 0).all()) for n, x in t.items() if n != "dout" and x is not None)


def test_once_differentiable():
    p = _plan(16)
    inp = _inputs(torch.float32, 1, 1, 8, 8, 1, 1, 8, p)
    q = inp["q"].requires_grad_(True)
    g = torch.autograd.grad(_call(inp, p, None, 0).square().sum(), q, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="once"):
        g.sum().backward()


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("maps,kind,lq,lk,h,kv,d,b", [
    (1, (8, 15), 120, 120, 4, 4, 32, 301),  # two key tiles, bias and sums in registers
    (2, (8, 15), 120, 120, 2, 2, 32, 601),
    (1, (10, 16), 160, 160, 4, 4, 24, 203),  # three of the four tiles of the widest register form
    (1, (12, 21), 252, 252, 2, 2, 32, 303),  # a last tile of 60 keys
    (1, (8, 15), 120, 120, 4, 2, 32, 301),  # shared heads: register form for the queries, general form for the keys
    (1, (3, 5), 15, 15, 4, 4, 32, 301),  # one tile
    (1, (8, 15), 120, 120, 4, 4, 64, 301),  # wide heads: general form on a board
    (1, 40, 33, 130, 4, 1, 32, 301),  # sequences
    (2, 40, 70, 65, 2, 1, 64, 601),
])
def test_workgroups_walk_several_samples(dtype, maps, kind, lq, lk, h, kv, d, b):
    """More samples than the card holds workgroups, with masks of every kind; masked rows hold NaN and infinities, and values of
    one sample must not reach the next."""
    p = _plan(kind)
    inp = _inputs(dtype, maps, b, lq, lk, h, kv, d, p, std=0.7)
    g = torch.Generator().manual_seed(3)
    mask = torch.rand(b, lk, generator=g) < torch.rand(b, 1, generator=g)
    mask[1::7] = False  # no key at all
    mask[2::7] = True
    mask[3::7, lk // 2 :] = False
    mask = mask.cuda()
    clean_out, clean = _compare(inp, p, mask)
    assert bool((clean_out[1::7] == 0).all())
    bad = dict(inp)
    for n, x in (("k", math.nan), ("v", math.inf)):
        bad[n] = inp[n].clone()
        bad[n][~mask] = x
    names = [n for n in ("q", "k", "v", "table", "lam") if inp[n] is not None]
    t = {**bad, **{n: bad[n].detach().clone().requires_grad_(True) for n in names}}
    out = _call(t, p, mask, 0)
    grads = torch.autograd.grad(out, [t[n] for n in names], inp["dout"])
    assert torch.equal(out, clean_out)
    for n, x in zip(names, grads):
        assert torch.equal(x, clean[n]), n


def test_many_positions_and_many_sums():
    """4095 relative positions under hundreds of workgroups: the sums by position are joined in two steps."""
    p = _plan(2047)
    _compare(_inputs(torch.bfloat16, 1, 3, 1500, 2100, 6, 2, 32, p), p)
    board = _plan((20, 30))
    _compare(_inputs(torch.float32, 1, 24, 600, 600, 4, 4, 16, board), board)


def test_offsets_beyond_32_bits():
    """Rows 2^25 elements apart: element offsets pass 2^31 and byte offsets 2^32."""
    p = _plan(32)
    n, step = 70, 1 << 25
    for dtype in BOTH:
        store = torch.empty(n * step + (1 << 24), dtype=dtype, device="cuda")
        view = {}
        base = _inputs(dtype, 1, 2, n, n, 1, 1, 32, p)
        for i, name in enumerate(("q", "k", "v", "dout")):
            x = store[i << 20 :].as_strided((2, n, 1, 32), (1 << 22, step, 32, 1), store.storage_offset() + (i << 20))
            x.copy_(base[name])
            view[name] = x
        want, grads = _compare(base, p)
        t = {k: view[k].detach().requires_grad_(True) for k in ("q", "k", "v")}
        out = _call({**base, **t}, p, None, 0)
        got = torch.autograd.grad(out, list(t.values()), view["dout"])
        assert torch.equal(out, want)
        for k, x in zip(t, got):
            assert torch.equal(x, grads[k]), k
        del store, view, t, out, got, x
        torch.cuda.empty_cache()


def test_two_calls_at_once():
    """Calls on two streams share no scratch memory."""
    p, w = _plan((8, 15)), _plan(64)
    a = _inputs(torch.float32, 1, 64, 120, 120, 4, 4, 32, p, seed=1)
    c = _inputs(torch.bfloat16, 2, 2, 150, 1900, 4, 2, 64, w, seed=2)

    def step(inp, plan):  # noqa: ANN001, ANN202
        names = [n for n in ("q", "k", "v", "table", "lam") if inp[n] is not None]
        t = {**inp, **{n: inp[n].detach().requires_grad_(True) for n in names}}
        out = _call(t, plan, None, 0)
        return (out.detach(), *torch.autograd.grad(out, [t[n] for n in names], inp["dout"]))

    want_a, want_c = step(a, p), step(c, w)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got_a, got_c = [], []
    for _ in range(4):
        with torch.cuda.stream(s1):
            got_a.append(step(a, p))
        with torch.cuda.stream(s2):
            got_c.append(step(c, w))
    torch.cuda.synchronize()
    for got, want in ((got_a, want_a), (got_c, want_c)):
        for r in got:
            for x, y in zip(r, want):
                assert torch.equal(x, y)


def test_two_graphs_of_two_maps():
    """Two captured training calls of different shapes, replayed in turn beside eager ones, on new inputs."""
    p = _plan((8, 15))
    shapes = ((3, 120, 4, 4), (40, 120, 2, 2))
    graphs = []
    for b, l, h, kv in shapes:
        static = {n: (x.clone() if x is not None else None) for n, x in _inputs(torch.bfloat16, 2, b, l, l, h, kv, 32, p).items()}
        names = ("q", "k", "v", "table", "lam")

        def step(static=static, names=names):  # noqa: ANN202
            t = {**static, **{n: static[n].detach().requires_grad_(True) for n in names}}
            out = _call(t, p, None, 0)
            return (out.detach(), *torch.autograd.grad(out, [t[n] for n in names], static["dout"]))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        graphs.append((graph, held, static, step))
    for seed in range(3):
        for (b, l, h, kv), (graph, _, static, _) in zip(shapes, graphs):
            for n, x in _inputs(torch.bfloat16, 2, b, l, l, h, kv, 32, p, seed=seed).items():
                if x is not None:
                    static[n].copy_(x)
            graph.replay()
        torch.cuda.synchronize()
        for _, held, _, step in graphs:
            for x, y in zip([x.clone() for x in held], step()):
                assert torch.equal(x, y)


def test_inputs_changed_in_place_are_noticed():
    p = _plan(16)
    inp = _inputs(torch.float32, 1, 1, 20, 20, 1, 1, 32, p)
    for name in ("k", "table"):
        t = {**inp, name: inp[name].clone(), "q": inp["q"].clone().requires_grad_(True)}
        out = _call(t, p, None, 0)
        t[name].mul_(2)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.sum().backward()


def test_half_of_a_batch_equals_the_whole():
    """Results do not depend on how many samples share a launch (no sum runs over samples except the table's)."""
    p = _plan((8, 15))
    for dtype in BOTH:
        inp = _inputs(dtype, 1, 400, 120, 120, 4, 4, 32, p)
        whole = _call(inp, p, None, 0)
        part = {n: (x[390:] if n in ("q", "k", "v") else x) for n, x in inp.items()}
        assert torch.equal(_call(part, p, None, 0), whole[390:])


def test_long_rows_stay_accurate():
    """fp32 against 64 bits over 32 tiles with few workgroups to split them.  A probability is off by two roundings of the exponential
    and that of its score (below 8 in units of its rounding in the root mean square); sums per tile add half a rounding times
    the root of 32: 8 u in all, and nothing may grow with the number of maxima a row runs through."""
    p = _plan(128)
    inp = _inputs(torch.float32, 1, 4, 2000, 2000, 8, 8, 32, p)
    names = ("q", "k", "v", "table")
    t = {**inp, **{n: inp[n].clone().requires_grad_(True) for n in names}}
    out = _call(t, p, None, 0)
    got = torch.autograd.grad(out, [t[n] for n in names], inp["dout"])
    from alphatriangle_amd.ops.attention import attention_reference

    w = {n: inp[n].double().requires_grad_(True) for n in names}
    ref = attention_reference(w["q"], w["k"], w["v"], None, w["table"], p, None, 32**-0.5, 0)
    want = torch.autograd.grad(ref, [w[n] for n in names], inp["dout"].double())
    assert _rel(out, ref) <= 8 * U32
    for n, g, e in zip(names[:3], got, want):
        assert _rel(g, e) <= 8 * U32, n


@pytest.mark.parametrize("dtype", BOTH)
def test_table_gradient_adds_up_to_zero(dtype):
    """Over all buckets a head's table gradient is zero by definition (softmax gradients of a row add up to zero).  What is left are
    roundings of dP - delta, |dP| about sqrt(64) = 8: one per row that does not average out in it, of random sign, over 3000 rows: 8 u sqrt(3000),
    twice that allowed.  A rounding that always goes one way would leave 3000 of them."""
    p = _plan(128)
    inp = _inputs(dtype, 1, 1, 3000, 3000, 8, 2, 64, p)
    table = inp["table"].clone().requires_grad_(True)
    g = torch.autograd.grad(_call({**inp, "table": table}, p, None, 0), table, inp["dout"])[0]
    assert float(g.double().sum(0).abs().max()) <= 2 * 8 * U32 * math.sqrt(3000)


def test_rows_with_a_single_key():
    """Their score gradients are zero by definition: dP - delta leaves roundings of products of the size of |dO| |v| only."""
    p = _plan(16)
    for dtype in BOTH:
        for maps in (1, 2):
            inp = _inputs(dtype, maps, 64, 5, 3, 2, 2, 64, p)
            mask = torch.zeros(64, 3, dtype=torch.bool, device="cuda")
            mask[torch.arange(64), torch.arange(64) % 3] = True
            t = {**inp, **{n: inp[n].clone().requires_grad_(True) for n in ("q", "k", "table")}}
            grads = torch.autograd.grad(_call(t, p, mask, 0), [t[n] for n in ("q", "k", "table")], inp["dout"])
            # one rounding of the probability, and of o, times |dP| <= |dO| |v|, times |k| scale or |q| scale, over the five queries
            size = float(inp["dout"].float().norm(dim=-1).max() * inp["v"].float().norm(dim=-1).max())
            side = float(torch.maximum(inp["q"].float().norm(dim=-1).max(), inp["k"].float().norm(dim=-1).max())) * 64**-0.5
            for g in grads[:2]:
                assert float(g.float().abs().max()) <= 8 * U32 * size * side * 5
            assert float(grads[2].abs().max()) <= 8 * U32 * size * 64 * 5


def test_broadcast_keys_add_their_gradients():
    p = _plan(24)
    inp = _inputs(torch.float32, 1, 3, 40, 50, 2, 2, 32, p)
    one = {n: inp[n][:1].clone().requires_grad_(True) for n in ("k", "v")}
    out = _call({**inp, **{n: x.expand(3, -1, -1, -1) for n, x in one.items()}}, p, None, 0)
    got = torch.autograd.grad(out, list(one.values()), inp["dout"])
    full = {n: inp[n][:1].repeat(3, 1, 1, 1).requires_grad_(True) for n in ("k", "v")}
    same = _call({**inp, **full}, p, None, 0)
    want = torch.autograd.grad(same, list(full.values()), inp["dout"])
    assert torch.equal(out, same)
    for x, y in zip(got, want):
        assert torch.equal(x, y.sum(0, keepdim=True))


@pytest.mark.parametrize("dtype,maps,kind,lq,lk,h,kv,d,b", [
    (torch.bfloat16, 1, (8, 15), 120, 120, 4, 4, 32, 64),
    (torch.bfloat16, 1, (12, 21), 252, 252, 4, 4, 32, 16),
    (torch.bfloat16, 2, (8, 15), 120, 120, 2, 2, 32, 32),
    (torch.bfloat16, 1, 128, 700, 900, 4, 2, 64, 1),
    (torch.bfloat16, 1, 128, 1, 4001, 8, 8, 64, 4),
    (torch.bfloat16, 2, None, 300, 600, 2, 1, 64, 1),
])
def test_inference_rounds_once(dtype, maps, kind, lq, lk, h, kv, d, b):
    """Without a backward pass to come the output is off by its own rounding.  Half a step of bf16 in an output, 2^-16 of every
    probability (two bf16 parts), and 2^-20 for the 32-bit parts (scores below 16, the exponential, sums), each times |v|."""
    from alphatriangle_amd.ops.attention import attention_reference

    p = _plan(kind)
    inp = _inputs(dtype, maps, b, lq, lk, h, kv, d, p)
    out = _call(inp, p, None, 0).double()
    w = {n: (x.double() if x is not None else None) for n, x in inp.items()}
    size = attention_reference(w["q"], w["k"], w["v"].abs(), -w["lam"] if maps == 2 else None, w["table"], p, None, d**-0.5, 0)
    ref = attention_reference(w["q"], w["k"], w["v"], w["lam"], w["table"], p, None, d**-0.5, 0)
    assert float(((out - ref).abs() - U16 * ref.abs() - (2.0**-16 + 2.0**-20) * size).max()) <= 0


@pytest.mark.parametrize("maps,kind,lq,lk,h,kv,d,b", [
    (1, (8, 15), 120, 120, 4, 4, 32, 16),
    (1, (12, 21), 252, 252, 2, 2, 32, 8),
    (2, (8, 15), 120, 120, 2, 2, 32, 16),
    (1, 128, 600, 700, 4, 2, 64, 1),
    (1, 128, 200, 300, 2, 1, 128, 1),
    (2, None, 300, 400, 2, 2, 64, 1),
    (2, 64, 300, 400, 2, 1, 48, 1),
])
def test_bf16_gradients_round_once(maps, kind, lq, lk, h, kv, d, b):
    """Half a step of bf16 in a gradient, 2^-16 of every probability and score gradient (two bf16 parts), and for the 32-bit parts
    2^-20 of p and of p (|dO| |v| + |delta|), each times the rows they meet."""
    p = _plan(kind)
    inp = _inputs(torch.bfloat16, maps, b, lq, lk, h, kv, d, p)
    t = {**inp, **{n: inp[n].clone().requires_grad_(True) for n in ("q", "k", "v")}}
    got = dict(zip(("q", "k", "v"), torch.autograd.grad(_call(t, p, None, 0), [t[n] for n in ("q", "k", "v")], inp["dout"])))
    group, scale = h // kv, d**-0.5
    q = inp["q"].double().view(b, lq, h, maps, d).permute(0, 2, 3, 1, 4)  # [b, h, maps, lq, d]
    k = inp["k"].double().view(b, lk, kv, maps, d).permute(0, 2, 3, 1, 4).repeat_interleave(group, 1)
    v, do = inp["v"].double().transpose(1, 2).repeat_interleave(group, 1), inp["dout"].double().transpose(1, 2)
    s = torch.matmul(q, k.transpose(-1, -2)) * scale
    if p is not None:
        s = s + inp["table"].double()[p.pairs(lq, lk)].view(lq, lk, h, maps).permute(2, 3, 0, 1)
    prob = s.softmax(-1)
    lam = torch.stack([torch.ones(h, device="cuda"), -inp["lam"]], 1).double().view(1, h, maps, 1, 1) if maps == 2 else 1.0
    dp, size = (torch.matmul(x, y.transpose(-1, -2)).unsqueeze(2) for x, y in ((do, v), (do.abs(), v.abs())))
    delta = (prob * dp).sum(-1, keepdim=True)
    ds = lam * prob * (dp - delta)
    off_ds = 2.0**-16 * ds.abs() + 2.0**-20 * abs(lam) * prob * (size + (prob * size).sum(-1, keepdim=True))
    mixed, off_mixed = (lam * prob).sum(2), (2.0**-16 + 2.0**-20) * (abs(lam) * prob).sum(2)

    def keys(x):  # noqa: ANN001, ANN202  [b, h, (maps,) lk, width] summed over the heads that share them
        x = x.view(b, kv, group, -1, lk, x.shape[-1]).sum(2)
        return x.permute(0, 3, 1, 2, 4).reshape(b, lk, -1, x.shape[-1])

    want = {"q": (torch.matmul(ds, k), torch.matmul(off_ds, k.abs())), "k": (torch.matmul(ds.transpose(-1, -2), q), torch.matmul(off_ds.transpose(-1, -2), q.abs())),
            "v": (torch.matmul(mixed.transpose(-1, -2), do), torch.matmul(off_mixed.transpose(-1, -2), do.abs()))}
    for n, (ref, off) in want.items():
        if n != "v":
            ref, off = ref * scale, off * scale
        ref, off = (x.permute(0, 3, 1, 2, 4).reshape(b, lq, h * maps, d) if n == "q" else keys(x) for x in (ref, off))
        assert float(((got[n].double() - ref).abs() - U16 * ref.abs() - off).max()) <= 0, n


@pytest.mark.parametrize("maps,kind,l,h,d,b", [(1, (8, 15), 120, 4, 32, 64), (2, (8, 15), 120, 2, 32, 64), (2, (20, 20), 400, 2, 64, 4), (2, 128, 300, 2, 40, 4),
                                               (2, None, 2000, 2, 64, 1), (2, 128, 2000, 2, 64, 1)])
def test_fp32_is_no_further_off_than_the_plain_form(maps, kind, l, h, d, b):  # noqa: E741
    """Output and gradients against 64 bits: at most as far off as the same formulas in elementary fp32 operations."""
    from alphatriangle_amd.ops.attention import attention_reference

    p = _plan(kind)
    inp = _inputs(torch.float32, maps, b, l, l, h, h, d, p)

    def results(dtype, call):  # noqa: ANN001, ANN202
        t = {n: (x.to(dtype).requires_grad_(n != "dout") if x is not None else None) for n, x in inp.items()}
        out = call(t)
        return [out, *torch.autograd.grad(out, [t[n] for n in ("q", "k", "v")], t["dout"])]

    def plain(t):  # noqa: ANN001, ANN202
        return attention_reference(t["q"], t["k"], t["v"], t["lam"], t["table"], p, None, d**-0.5, 0)

    exact = results(torch.float64, plain)
    for n, own, other, e in zip(("out", "q", "k", "v"), results(torch.float32, lambda t: _call(t, p, None, 0)), results(torch.float32, plain), exact):
        assert _rel(own, e) <= _rel(other, e), (n, _rel(own, e), _rel(other, e))


@pytest.mark.parametrize("maps", [1, 2])
def test_outputs_take_in_place_operations(maps):
    """In token order as in batch order; the gradients are those of the same operations out of place."""
    p = _plan(16)
    inp = _inputs(torch.bfloat16, maps, 3, 20, 20, 2, 2, 32, p)
    for order in (lambda x: x, lambda x: x.transpose(0, 1).contiguous().transpose(0, 1)):
        grads = []
        for in_place in (False, True):
            t = {**inp, **{n: order(inp[n]).detach().requires_grad_(True) for n in ("q", "k", "v")}}
            out = _call(t, p, None, 0)
            out = out.mul_(2).relu_() if in_place else out.mul(2).relu()
            grads.append((out.detach(), *torch.autograd.grad(out, [t[n] for n in ("q", "k", "v")], inp["dout"])))
        for x, y in zip(*grads):
            assert torch.equal(x, y) and x.stride() == y.stride()


def test_forward_mode_tangents_are_refused():
    from torch.autograd import forward_ad

    p = _plan(16)
    inp = _inputs(torch.float32, 1, 1, 8, 8, 1, 1, 8, p)
    with forward_ad.dual_level():
        for n in ("q", "table"):
            with pytest.raises(NotImplementedError, match="reverse mode"):
                _call({**inp, n: forward_ad.make_dual(inp[n], torch.ones_like(inp[n]))}, p, None, 0)
        _call(inp, p, None, 0)


def test_tracing_is_refused():
    from torch.fx.experimental.proxy_tensor import make_fx

    p = _plan(16)
    inp = _inputs(torch.float32, 1, 1, 8, 8, 1, 1, 8, p)

    def call(q):  # noqa: ANN001, ANN202
        return _call({**inp, "q": q}, p, None, 0)

    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(call, (inp["q"],), check_trace=False)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        make_fx(call)(inp["q"])


def test_plans_under_a_gpu_default_device():
    from alphatriangle_amd.ops.attention import RelativeBuckets

    with torch.device("cuda"):
        made = RelativeBuckets.log(32, 16), RelativeBuckets.board(3, 5)
        held = RelativeBuckets(**{n: getattr(made[1], n) for n in ("num_buckets", "radius", "rows", "cols", "lut", "order", "start")})
    for p, want in zip((*made, held), (RelativeBuckets.log(32, 16), RelativeBuckets.board(3, 5), RelativeBuckets.board(3, 5))):
        assert p.device.type == "cuda" and want.device.type == "cpu"
        assert all(torch.equal(getattr(p, n).cpu(), getattr(want, n)) for n in ("lut", "order", "start"))


@pytest.mark.parametrize("maps", [1, 2])
def test_smallest_scale_keeps_the_bias(maps):
    """At a scale of 1e-30 products of queries and keys are nothing beside the bias, which the kernels hold 1e30 times as large."""
    from alphatriangle_amd.ops.attention import attention_reference, differential_attention, relative_attention

    p = _plan(16)
    inp = _inputs(torch.float32, maps, 2, 40, 50, 2, 2, 32, p)
    more = {"scale": 1e-30}
    args = [inp["q"], inp["k"], inp["v"]]
    out = relative_attention(*args, inp["table"], p, **more) if maps == 1 else differential_attention(*args, inp["lam"], inp["table"], p, **more)
    ref = attention_reference(*(x.double() for x in args), inp["lam"].double() if maps == 2 else None, inp["table"].double(), p, None, 1e-30, 0)
    assert _rel(out, ref) <= _tol(torch.float32, 32, 40, 50)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("maps,kind,l", [(1, (8, 15), 120), (1, 16, 90), (2, 16, 90)])
def test_infinities_reach_their_column_only(dtype, maps, kind, l):  # noqa: E741
    """An infinity in one value of ``v`` (or of the output's gradient) leaves every other column of the output (of ``v``'s gradient) as it is."""
    p = _plan(kind)
    inp = _inputs(dtype, maps, 2, l, l, 2, 2, 32, p)

    def results(t, train):  # noqa: ANN001, ANN202
        if not train:
            return _call(t, p, None, 0), None
        v = t["v"].clone().requires_grad_(True)
        out = _call({**t, "v": v}, p, None, 0)
        return out.detach(), torch.autograd.grad(out, v, t["dout"])[0]

    for train in (False, True):
        want, grad = results(inp, train)
        v, dout = inp["v"].clone(), inp["dout"].clone()
        v[1, 3, 1, 5] = math.inf
        got, _ = results({**inp, "v": v}, train)
        assert not bool(torch.isfinite(got[1, :, 1, 5]).any())
        got[1, :, 1, 5] = want[1, :, 1, 5]
        assert torch.equal(got, want)
        if train:
            dout[0, 7, 0, 9] = -math.inf
            _, got = results({**inp, "dout": dout}, True)
            assert not bool(torch.isfinite(got[0, :, 0, 9]).any())
            got[0, :, 0, 9] = grad[0, :, 0, 9]
            assert torch.equal(got, grad)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("maps,kind,l,h,kv", [(1, (8, 15), 120, 2, 2), (1, 40, 700, 4, 2), (2, (8, 15), 120, 2, 2), (2, 40, 300, 2, 1), (2, None, 300, 2, 2)])
def test_gradients_of_some_arguments(dtype, maps, kind, l, h, kv):  # noqa: E741
    """Any subset of the arguments may be frozen: the other gradients keep their bits, and keys and values take no work where both are."""
    p = _plan(kind)
    inp = _inputs(dtype, maps, 2, l, l, h, kv, 32, p)
    names = [n for n in ("q", "k", "v", "table", "lam") if inp[n] is not None]

    def grads(wanted):  # noqa: ANN001, ANN202
        t = {**inp, **{n: inp[n].clone().requires_grad_(n in wanted) for n in names}}
        out = _call(t, p, None, 0)
        node = out.grad_fn(inp["dout"])
        assert (node[1] is None) == (node[2] is None) == (not {"k", "v"} & set(wanted))
        return dict(zip(wanted, torch.autograd.grad(out, [t[n] for n in wanted], inp["dout"])))

    every = grads(names)
    for bits in range(1, 1 << len(names)):
        wanted = [n for i, n in enumerate(names) if bits >> i & 1]
        for n, g in grads(wanted).items():
            assert torch.equal(g, every[n]), (wanted, n)


@pytest.mark.parametrize("op", ["relative", "differential", "joint"])
def test_capture_beside_an_eager_graph_of_the_same_leaves(op):
    """Refused at the forward call, before the backward pass would reach out of the capture; without the eager graph, captured and
    replayed on new values beside eager calls."""
    from alphatriangle_amd.ops.residual import gated_norm_residual

    if op == "joint":
        g = torch.Generator(device="cuda").manual_seed(0)
        leaves = [torch.randn(*s, generator=g, device="cuda").requires_grad_(True) for s in ((64, 40), (64, 40), (40,), (40,), (40,), (40,), (40,))]

        def forward(*t):  # noqa: ANN002, ANN202
            return gated_norm_residual(*t)[1]
    else:
        p = _plan((3, 5))
        inp = _inputs(torch.float32, 1 if op == "relative" else 2, 3, 15, 15, 2, 2, 32, p)
        names = [n for n in ("q", "k", "v", "table", "lam") if inp[n] is not None]
        leaves = [inp[n].requires_grad_(True) for n in names]

        def forward(*t):  # noqa: ANN002, ANN202
            return _call({**inp, **dict(zip(names, t))}, p, None, 0)

    eager = forward(*leaves)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager graph"), torch.cuda.graph(graph):
        forward(*leaves)
    torch.cuda.synchronize()
    detached = torch.cuda.CUDAGraph()  # other leaves of the same values: nothing to reach out to
    with torch.cuda.graph(detached):
        again = [t.detach().requires_grad_(True) for t in leaves]
        held = torch.autograd.grad(forward(*again).sum(), again)
    del eager
    own = torch.cuda.CUDAGraph()
    with torch.cuda.graph(own):
        kept = torch.autograd.grad(forward(*leaves).sum(), leaves)
    for seed in range(3):
        with torch.no_grad():
            for t in leaves:
                t.add_(0.1 * (seed + 1))
        detached.replay()
        own.replay()
        torch.cuda.synchronize()
        want = torch.autograd.grad(forward(*leaves).sum(), leaves)
        torch.cuda.synchronize()
        for x, y, z in zip(held, kept, want):
            assert torch.equal(x, z) and torch.equal(y, z)
