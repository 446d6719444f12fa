"""The encoder's attention and residual operators, as cases to be measured: what a user's program holds, one pass through
an operator, and what that pass cannot do without.

``own`` picks the side: false computes every operator from elementary torch operations in 32 bits (the plain form), true
makes the calls a user of this package makes (``alphatriangle_amd.ops.attention``, ``alphatriangle_amd.ops.residual``).
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-5
BUCKETS, MAX_DISTANCE = 32, 128  # sequences: half of each side's buckets exact, the rest logarithmic up to the distance


# ---------------------------------------------------------------------------------------------------------------- cases
def listed() -> list[dict]:
    return [
        # one learner step's encoder attention at the default configuration: 256 boards of 8 x 15 cells, fp32 training
        _attention("relative_board_train", "relative", "fp32", True, batch=256, rows=8, cols=15, heads=4, dim=32),
        # the leaves of 4096 concurrent games in bf16, forward only (one evaluation of a search wave)
        _attention("relative_leaves", "relative", "bf16", False, batch=4096, rows=8, cols=15, heads=4, dim=32),
        # the 12 x 21 board (252 cells: more than one tile) in a bf16 autocast learner step
        _attention("relative_large_board_train", "relative", "bf16", True, batch=256, rows=12, cols=21, heads=4, dim=32),
        # long ragged sequences with key/value heads shared by four query heads, logarithmic distance buckets
        _attention("relative_long_train", "relative", "bf16", True, batch=2, lq=4095, lk=4095, heads=8, kv_heads=2, dim=64, ragged=True),
        # one new token of each of four sequences against everything before it: what latency and bandwidth allow
        _attention("relative_one_token", "relative", "bf16", False, batch=4, lq=1, lk=8190, heads=8, dim=64, ragged=True),
        # the learner step again with the two-map attention (two pairs of 32-wide maps over 64-wide values)
        _attention("differential_board_train", "differential", "fp32", True, batch=256, rows=8, cols=15, heads=2, dim=32),
        # two-map attention over a long odd-sized sequence, no position bias, 64-wide maps
        _attention("differential_long_train", "differential", "bf16", True, batch=1, lq=3001, lk=3001, heads=4, dim=64, bias=False),
        # the smallest call: one token of one sequence against 600 others in fp32
        _attention("differential_one_token", "differential", "fp32", False, batch=1, lq=1, lk=600, heads=2, dim=32, bias=False),
        # residual joint of one encoder block in the default learner step: 256 boards x 120 tokens, a gate per value
        _norm("norm_board_train", "fp32", "fp32", "full", True, tokens=120 * 256, width=128),
        # the same joint for the leaves of 4096 games: fp32 residual stream, bf16 branch, forward only
        _norm("norm_leaves", "fp32", "bf16", "none", False, tokens=120 * 4096, width=128),
        # one board, forward only: a launch and little else
        _norm("norm_one_board", "fp32", "fp32", "full", False, tokens=120, width=128),
        # a wide model with an odd number of rows, a width that is no power of two, and one gate per token
        _norm("norm_wide_train", "bf16", "bf16", "token", True, tokens=16381, width=2000),
    ]


def _attention(name, op, dtype, train, *, batch, heads, dim, rows=0, cols=0, lq=0, lk=0, kv_heads=0, ragged=False, bias=True):  # noqa: ANN001
    return {"name": name, "op": op, "dtype": dtype, "train": train, "batch": batch, "rows": rows, "cols": cols,
            "lq": rows * cols if rows else lq, "lk": rows * cols if rows else lk, "heads": heads, "kv_heads": kv_heads or heads,
            "dim": dim, "ragged": ragged, "bias": bias}


def _norm(name, stream, branch, gate, train, *, tokens, width):  # noqa: ANN001
    return {"name": name, "op": "norm", "dtype": branch, "stream": stream, "gate": gate, "train": train, "tokens": tokens, "width": width}


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


def draw(rng: random.Random) -> dict:
    op = rng.choice(["relative", "relative", "differential", "differential", "norm"])
    if op == "norm":
        branch = rng.choice(["fp32", "bf16"])
        stream = "fp32" if branch == "fp32" else rng.choice(["fp32", "bf16"])
        width = rng.choice([64, 128, 256, 384, 512, 777, 1000, 1024, 2000, 4096, 129, 40, _log_int(rng, 1, 4096)])
        tokens = _log_int(rng, 1, max(1, min(400_000, 30_000_000 // width)))
        case = _norm("", stream, branch, rng.choice(["none", "full", "token"]), rng.random() < 0.6, tokens=tokens, width=width)
    else:
        dtype = rng.choice(["fp32", "bf16"])
        dim = rng.choice([8, 16, 24, 32, 40, 48, 64] + ([80, 96, 128] if op == "relative" else []))
        kv = rng.choice([1, 1, 2, 3, 4])
        heads = kv * rng.choice([1, 1, 2, 4])
        bias = op == "relative" or rng.random() < 0.5
        form = rng.choice(["board", "sequence", "sequence", "token"])
        if form == "board":
            rows, cols = rng.randint(2, 16), rng.randint(2, 24)
            size = dict(rows=rows, cols=cols)
            lq = lk = rows * cols
        else:
            # two keys at least: with a single one the gradients of queries and keys are zero by definition
            lk = _log_int(rng, 2, 2000 if form == "sequence" else 16000)
            lq = 1 if form == "token" else rng.choice([lk, lk, _log_int(rng, 1, lk)])
            size = dict(lq=lq, lk=lk)
        most = max(1, min(1024, int(1e8 / (heads * max(lq, 64) * max(lk, 64))), int(2e7 / (heads * (lq + lk) * dim))))
        train = form != "token" and rng.random() < 0.6
        case = _attention("", op, dtype, train, batch=_log_int(rng, 1, most), heads=heads, kv_heads=kv, dim=dim, ragged=rng.random() < 0.4,
                          bias=bias, **size)
    del case["name"]
    return case


# ----------------------------------------------------------------------------------------------------------- what it needs
def _lengths(case: dict) -> list[int]:
    """Keys each sample has: all, or spread from all of them down (the last of three or more samples has none)."""
    b, lk = case["batch"], case["lk"]
    if not case["ragged"]:
        return [lk] * b
    if b < 3:
        return [max(1, lk - (i * lk) // (b + 1)) for i in range(b)]
    return [(lk * (b - 1 - i)) // (b - 1) for i in range(b)]


def work(case: dict) -> dict:
    size = {"fp32": 4, "bf16": 2}
    if case["op"] == "norm":
        n, d = case["tokens"], case["width"]
        sx, sz = size[case["stream"]], size[case["dtype"]]
        g = {"none": 0, "token": n, "full": n * d}[case["gate"]] * sz
        forward = n * d * (sx + sz) + g + 5 * d * 4 + n * d * (sx + sz)
        if not case["train"]:
            return {"bytes": forward, "flops": 20 * n * d}
        back = n * d * (sx + sz) + n * d * (sx + sz) + g + 5 * d * 4  # both output gradients in, three gradients out
        return {"bytes": forward + back, "flops": 60 * n * d}
    e, h, kv, d, lq, lk, b = size[case["dtype"]], case["heads"], case["kv_heads"], case["dim"], case["lq"], case["lk"], case["batch"]
    keys = sum(_lengths(case))
    maps = 2 if case["op"] == "differential" else 1
    dv = d * maps
    q_bytes, o_bytes, kv_bytes = b * lq * h * maps * d * e, b * lq * h * dv * e, keys * kv * (maps * d + dv) * e
    table = (_bucket_count(case) * h * maps * 4 if case["bias"] else 0) + (h * 4 if maps == 2 else 0)
    pairs = lq * keys * h
    nbytes, flops = q_bytes + kv_bytes + o_bytes + table, pairs * 2 * (maps * d + dv)
    if case["train"]:
        nbytes += o_bytes + q_bytes + kv_bytes + table
        flops += pairs * 2 * (3 * maps * d + 2 * dv)  # the scores again, dQ and dK of each map; dP and dV once
    return {"bytes": nbytes, "flops": flops}


def _bucket_count(case: dict) -> int:
    return (2 * case["rows"] - 1) * (2 * case["cols"] - 1) if case["rows"] else BUCKETS


# ------------------------------------------------------------------------------------------------------------------ inputs
def _buckets_of(case: dict, dev: torch.device) -> torch.Tensor:
    """``[lq, lk]`` bucket of every (query, key) pair; a single token stands behind the last key of its sample (``[batch, 1, lk]``)."""
    if case["rows"]:
        rows, cols = case["rows"], case["cols"]
        t = torch.arange(rows * cols, device=dev)
        r, c = t // cols, t % cols
        return (r[None, :] - r[:, None] + rows - 1) * (2 * cols - 1) + (c[None, :] - c[:, None] + cols - 1)
    rel = torch.arange(case["lk"], device=dev)[None, None, :] - (_offsets(case, dev)[:, None, None] + torch.arange(case["lq"], device=dev)[None, :, None])
    half = BUCKETS // 2
    exact = half // 2
    dist = rel.abs()
    far = exact + (torch.log(dist.clamp(min=1).double() / exact) / math.log(MAX_DISTANCE / exact) * (half - exact) + 1e-9).floor().long()
    bucket = torch.where(dist < exact, dist, far.clamp(max=half - 1)) + half * (rel > 0)
    return bucket[0] if case["lq"] > 1 else bucket


def _offsets(case: dict, dev: torch.device) -> torch.Tensor:
    if case["lq"] == 1 and not case["rows"]:
        return torch.tensor([max(0, n - 1) for n in _lengths(case)], dtype=torch.int32, device=dev)
    return torch.zeros(1, dtype=torch.int32, device=dev)


def prepare(case: dict, seed: int) -> dict:
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, dtype=torch.float32, std=1.0, mean=0.0):  # noqa: ANN002, ANN202
        return (torch.randn(*shape, generator=gen, device=dev) * std + mean).to(dtype)

    dt = DTYPES[case["dtype"]]
    if case["op"] == "norm":
        n, d = case["tokens"], case["width"]
        sx = DTYPES[case["stream"]]
        st = {"case": case, "x": normal(n, d, dtype=sx), "z": normal(n, d, dtype=dt, std=0.7, mean=0.1),
              "gate": {"none": None, "token": normal(n, 1, dtype=dt), "full": normal(n, d, dtype=dt)}[case["gate"]],
              "scale": normal(d, std=0.2, mean=0.5), "post_weight": normal(d, std=0.2, mean=1.0), "post_bias": normal(d, std=0.2),
              "pre_weight": normal(d, std=0.2, mean=1.0), "pre_bias": normal(d, std=0.2)}
        if case["train"]:
            st["dy"], st["dh"] = normal(n, d, dtype=sx), normal(n, d, dtype=dt)
        return st
    b, lq, lk, h, kv, d = (case[k] for k in ("batch", "lq", "lk", "heads", "kv_heads", "dim"))
    maps = 2 if case["op"] == "differential" else 1
    st = {"case": case, "q": normal(b, lq, h * maps, d, dtype=dt), "k": normal(b, lk, kv * maps, d, dtype=dt), "v": normal(b, lk, kv, d * maps, dtype=dt),
          "table": normal(_bucket_count(case), h * maps, std=0.5) if case["bias"] else None,
          "lam": torch.rand(h, generator=gen, device=dev) * 0.6 + 0.1 if maps == 2 else None, "mask": None, "dout": None}
    if case["ragged"]:
        lengths = torch.tensor(_lengths(case), device=dev)
        st["mask"] = torch.arange(lk, device=dev)[None, :] < lengths[:, None]
    if case["train"]:
        st["dout"] = normal(b, lq, h, d * maps, dtype=dt)
    if case["bias"]:
        st["bucket"] = _buckets_of(case, dev)
    st["offset"] = _offsets(case, dev) if case["lq"] == 1 and not case["rows"] else 0
    if own and case["bias"]:  # the plan a model builds once
        from alphatriangle_amd.ops.attention import RelativeBuckets

        st["plan"] = RelativeBuckets.board(case["rows"], case["cols"], device=dev) if case["rows"] else RelativeBuckets.log(BUCKETS, MAX_DISTANCE, device=dev)
    return st


# ---------------------------------------------------------------------------------------------------------------- one pass
def run(state: dict):  # noqa: ANN201
    if own:
        return _own_norm(state) if state["case"]["op"] == "norm" else _own_attention(state)
    return _plain_norm(state) if state["case"]["op"] == "norm" else _plain_attention(state)


def _own_attention(st: dict) -> dict:
    from alphatriangle_amd.ops import attention

    case = st["case"]
    names = [n for n in ("q", "k", "v", "table", "lam") if st[n] is not None]
    t = {n: st[n].detach().requires_grad_(case["train"]) for n in names}
    more = {"key_mask": st["mask"], "query_offset": st["offset"]}
    if case["op"] == "relative":
        out = attention.relative_attention(t["q"], t["k"], t["v"], t["table"], st["plan"], **more)
    else:
        out = attention.differential_attention(t["q"], t["k"], t["v"], t["lam"], t.get("table"), st.get("plan"), **more)
    if not case["train"]:
        return {"out": out}
    grads = torch.autograd.grad(out, [t[n] for n in names], st["dout"])
    return {"out": out.detach(), **{"d" + n: g for n, g in zip(names, grads)}}


def _own_norm(st: dict) -> dict:
    from alphatriangle_amd.ops.residual import gated_norm_residual

    case = st["case"]
    names = [n for n in ("x", "z", "gate", "scale", "post_weight", "post_bias", "pre_weight", "pre_bias") if st[n] is not None]
    t = {n: st[n].detach().requires_grad_(case["train"]) for n in names}
    y, h = gated_norm_residual(t["x"], t["z"], t["scale"], t["post_weight"], t["post_bias"], t["pre_weight"], t["pre_bias"], gate=t.get("gate"), eps=EPS)
    if not case["train"]:
        return {"y": y, "h": h}
    grads = torch.autograd.grad([y, h], [t[n] for n in names], [st["dy"], st["dh"]])
    return {"y": y.detach(), "h": h.detach(), **{"d" + n: g for n, g in zip(names, grads)}}


def _softmax(s: torch.Tensor) -> torch.Tensor:
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total == 0, 1.0, total)


def _plain_attention(st: dict) -> dict:
    """Maps are a dimension of their own: q ``[B, H, M, Lq, D]``, k ``[B, KV, M, Lk, D]`` (repeated to H), v ``[B, H, 1, Lk, M D]``."""
    case = st["case"]
    dt = st["q"].dtype
    b, lq, lk, h, kv, d = (case[k] for k in ("batch", "lq", "lk", "heads", "kv_heads", "dim"))
    maps = 2 if case["op"] == "differential" else 1
    group, scale = h // kv, d**-0.5
    q = st["q"].float().view(b, lq, h, maps, d).permute(0, 2, 3, 1, 4).contiguous()
    k = st["k"].float().view(b, lk, kv, maps, d).permute(0, 2, 3, 1, 4).repeat_interleave(group, 1)
    v = st["v"].float().view(b, lk, kv, 1, d * maps).permute(0, 2, 3, 1, 4).repeat_interleave(group, 1)
    s = q @ k.transpose(-1, -2) * scale
    if case["bias"]:
        bias = st["table"][st["bucket"]]  # [lq, lk, maps h] or, for single tokens, [b, 1, lk, maps h]
        lead = bias.shape[:-1]
        bias = bias.view(*lead, h, maps)
        s = s + (bias.permute(2, 3, 0, 1) if bias.dim() == 4 else bias.permute(0, 3, 4, 1, 2))
    if st["mask"] is not None:
        s = s.masked_fill(~st["mask"][:, None, None, None, :], -math.inf)
    p = _softmax(s)
    lam = st["lam"].view(h, 1, 1) if maps == 2 else None
    mixed = p[:, :, 0] - lam * p[:, :, 1] if maps == 2 else p[:, :, 0]  # [B, H, Lq, Lk]
    v0 = v[:, :, 0]
    out = (mixed @ v0).permute(0, 2, 1, 3).to(dt).contiguous()
    if not case["train"]:
        return {"out": out}
    do = st["dout"].float().permute(0, 2, 1, 3).contiguous()
    d_mixed = do @ v0.transpose(-1, -2)
    dv = mixed.transpose(-1, -2) @ do
    dp = torch.stack([d_mixed, -lam * d_mixed], 2) if maps == 2 else d_mixed[:, :, None]
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    dq = (ds @ k * scale).permute(0, 3, 1, 2, 4).reshape(b, lq, h * maps, d)
    dk = (ds.transpose(-1, -2) @ q * scale).view(b, kv, group, maps, lk, d).sum(2).permute(0, 3, 1, 2, 4).reshape(b, lk, kv * maps, d)
    dv = dv.view(b, kv, group, lk, d * maps).sum(2).permute(0, 2, 1, 3)
    res = {"out": out, "dq": dq.to(dt), "dk": dk.to(dt), "dv": dv.to(dt).contiguous()}
    if case["bias"]:
        # per query row, a product with the buckets' indicator; 64 bits, for these are long sums whose terms cancel
        pairs = ds.view(b, h * maps, lq, lk)
        pairs = pairs.sum(0).transpose(0, 1) if st["bucket"].dim() == 2 else pairs[:, :, 0]
        bucket = st["bucket"] if st["bucket"].dim() == 2 else st["bucket"][:, 0]
        indicator = (bucket[:, :, None] == torch.arange(st["table"].shape[0], device=ds.device)).double()
        table = (pairs.double() @ indicator).sum(0).t()
        res["dtable"] = table.float().contiguous()
    if maps == 2:
        res["dlam"] = -(p[:, :, 1] * d_mixed).sum(-1).double().sum((0, 2)).float()
    return res


def _standard(t: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    centred = t - t.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt((centred * centred).mean(-1, keepdim=True) + EPS)
    return centred * rstd, rstd


def _standard_back(g: torch.Tensor, unit: torch.Tensor, rstd: torch.Tensor) -> torch.Tensor:
    return rstd * (g - g.mean(-1, keepdim=True) - unit * (g * unit).mean(-1, keepdim=True))


def _plain_norm(st: dict) -> dict:
    x, z, gate = st["x"].float(), st["z"].float(), st["gate"]
    open_ = 1.0 / (1.0 + torch.exp(-gate.float())) if gate is not None else None
    zu, zr = _standard(z)
    n = zu * st["post_weight"] + st["post_bias"]
    scaled = st["scale"] * n
    y = x + (scaled * open_ if gate is not None else scaled)
    yu, yr = _standard(y)
    h = yu * st["pre_weight"] + st["pre_bias"]
    res = {"y": y.to(st["x"].dtype), "h": h.to(st["z"].dtype)}
    if not st["case"]["train"]:
        return res
    dh = st["dh"].float()
    dy = st["dy"].float() + _standard_back(dh * st["pre_weight"], yu, yr)
    opened = dy * open_ if gate is not None else dy
    dn = opened * st["scale"]
    res["dx"] = dy.to(st["x"].dtype)
    res["dz"] = _standard_back(dn * st["post_weight"], zu, zr).to(st["z"].dtype)
    if gate is not None:
        dg = dy * scaled * open_ * (1.0 - open_)
        res["dgate"] = (dg.sum(-1, keepdim=True) if gate.shape[-1] == 1 and dg.shape[-1] != 1 else dg).to(gate.dtype)
    res["dscale"] = (opened * n).sum(0)
    res["dpost_weight"], res["dpost_bias"] = (dn * zu).sum(0), dn.sum(0)
    res["dpre_weight"], res["dpre_bias"] = (dh * yu).sum(0), dh.sum(0)
    return res


# ---------------------------------------------------------------------------------------------------------------- 64 bits
def exact(case: dict, seed: int):  # noqa: ANN201
    """The definitions in 64 bits, their gradients by automatic differentiation."""
    st = prepare(case, seed)
    wide = {k: (v.double().requires_grad_(bool(case["train"])) if torch.is_tensor(v) and v.is_floating_point() else v) for k, v in st.items()}
    if case["op"] == "norm":
        names = [n for n in ("x", "z", "gate", "scale", "post_weight", "post_bias", "pre_weight", "pre_bias") if wide[n] is not None]

        def layer_norm(t, w, c):  # noqa: ANN001, ANN202
            var, mean = torch.var_mean(t, -1, correction=0, keepdim=True)
            return (t - mean) * (var + EPS) ** -0.5 * w + c

        branch = wide["scale"] * layer_norm(wide["z"], wide["post_weight"], wide["post_bias"])
        y = wide["x"] + (branch * torch.sigmoid(wide["gate"]) if wide["gate"] is not None else branch)
        h = layer_norm(y, wide["pre_weight"], wide["pre_bias"])
        if not case["train"]:
            return {"y": y, "h": h}
        grads = torch.autograd.grad((y * wide["dy"].detach()).sum() + (h * wide["dh"].detach()).sum(), [wide[n] for n in names])
        return {"y": y.detach(), "h": h.detach(), **{"d" + n: g for n, g in zip(names, grads)}}
    maps = 2 if case["op"] == "differential" else 1
    group = case["heads"] // case["kv_heads"]
    visible = st["mask"] if st["mask"] is not None else torch.ones(case["batch"], case["lk"], dtype=torch.bool, device=st["q"].device)
    bias_leaf = None
    if case["bias"]:  # one leaf value per pair (and head), summed into the buckets afterwards
        bias_leaf = wide["table"].detach()[st["bucket"]].requires_grad_(bool(case["train"]))
        bias = bias_leaf.movedim(-1, -3)  # [heads, lq, lk] or [b, heads, 1, lk]

    def softmax_of(m: int) -> torch.Tensor:
        queries = wide["q"][:, :, m::maps].transpose(1, 2)
        keys = wide["k"][:, :, m::maps].transpose(1, 2).repeat_interleave(group, 1)
        logits = torch.matmul(queries, keys.transpose(2, 3)) / math.sqrt(case["dim"])
        if case["bias"]:
            logits = logits + bias[..., m::maps, :, :]
        weights = torch.exp(logits - logits.detach().amax(-1, keepdim=True)) * visible[:, None, None, :]
        mass = weights.sum(-1, keepdim=True)
        return weights / torch.where(mass > 0, mass, torch.ones_like(mass))

    att = softmax_of(0)
    if maps == 2:
        att = att - wide["lam"][:, None, None] * softmax_of(1)
    out = torch.matmul(att, wide["v"].transpose(1, 2).repeat_interleave(group, 1)).transpose(1, 2)
    if not case["train"]:
        return {"out": out}
    names = [n for n in ("q", "k", "v", "table", "lam") if wide[n] is not None]
    leaves = [bias_leaf if n == "table" else wide[n] for n in names]
    grads = dict(zip(names, torch.autograd.grad((out * wide["dout"].detach()).sum(), leaves)))
    if case["bias"]:
        flat = grads["table"].reshape(-1, grads["table"].shape[-1])
        which = st["bucket"].reshape(-1)
        grads["table"] = torch.stack([torch.bincount(which, weights=column, minlength=_bucket_count(case)) for column in flat.t().contiguous()], 1)
    return {"out": out.detach(), **{"d" + n: grads[n] for n in names}}


