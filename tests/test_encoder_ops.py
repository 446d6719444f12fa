"""Encoder attention operators on the host: bucket plans, the reference formulas against plain loops, refusals."""

from __future__ import annotations

import math
import shutil
import subprocess
from pathlib import Path

import numpy
import pytest
import torch

from alphatriangle_amd.ops.attention import MAX_OFFSET, RelativeBuckets, differential_attention, relative_attention


def test_log_buckets():
    p = RelativeBuckets.log(32, 128)
    lut = p.lut.tolist()
    assert p.radius == 128 and len(lut) == 257 and lut[128] == 0
    assert [lut[128 - n] for n in range(8)] == list(range(8))        # keys at or before the query, one bucket each
    assert [lut[128 + n] for n in range(1, 8)] == list(range(17, 24))  # keys behind it
    assert lut[0] == 15 and lut[-1] == 31
    assert all(a >= b for a, b in zip(lut[:128], lut[1:129]))
    assert p.start[0] == 0 and p.start[-1] == 257 and sorted(p.order.tolist()) == list(range(257))
    for b in range(32):
        assert all(lut[i] == b for i in p.order[p.start[b] : p.start[b + 1]].tolist())
    far = p.pairs(3, 1000, 500)
    assert far[0, 0] == 15 and far[0, 999] == 31 and far[1, 501] == 0
    each = p.pairs(1, 10, torch.tensor([0, 9], dtype=torch.int32))
    assert each.shape == (2, 1, 10) and each[1, 0, 9] == 0 and each[0, 0, 0] == 0


def test_board_buckets():
    p = RelativeBuckets.board(4, 7)
    got = p.pairs(28, 28)
    for i in range(28):
        for j in range(28):
            dr, dc = j // 7 - i // 7, j % 7 - i % 7
            assert got[i, j] == (dr + 3) * 13 + dc + 6
    assert p.num_buckets == 7 * 13 == p.lut.numel()
    assert RelativeBuckets.board(32, 32).num_buckets == 63 * 63


@pytest.mark.parametrize("bad", [lambda: RelativeBuckets.log(31), lambda: RelativeBuckets.log(2), lambda: RelativeBuckets.log(32, 8),
                                 lambda: RelativeBuckets.log(32, 4096), lambda: RelativeBuckets.board(0, 3), lambda: RelativeBuckets.board(40, 40)])
def test_plan_refusals(bad):
    with pytest.raises(ValueError):
        bad()


def _loops(q, k, v, lam, table, pairs, mask, scale):  # noqa: ANN001
    b, lq, hm, d = q.shape
    lk, kv = k.shape[1], v.shape[2]
    maps = 1 if lam is None else 2
    h = hm // maps
    out = torch.zeros(b, lq, h, d * maps, dtype=torch.float64)
    for s in range(b):
        for i in range(lq):
            for n in range(h):
                g = n // (h // kv)
                for m in range(maps):
                    keys = [j for j in range(lk) if mask is None or bool(mask[s, j])]
                    x = [scale * float(q[s, i, n * maps + m] @ k[s, j, g * maps + m]) + (float(table[pairs[i, j], n * maps + m]) if table is not None else 0.0)
                         for j in keys]
                    if not x:
                        continue
                    top = max(x)
                    e = [math.exp(a - top) for a in x]
                    c = 1.0 if m == 0 else -float(lam[n])
                    for j, a in zip(keys, e):
                        out[s, i, n] += c * a / sum(e) * v[s, j, g]
    return out


@pytest.mark.parametrize("maps", [1, 2])
@pytest.mark.parametrize("form", ["board", "sequence"])
def test_reference_is_the_definition(maps, form):
    torch.manual_seed(maps)
    p = RelativeBuckets.board(2, 3) if form == "board" else RelativeBuckets.log(8, 5)
    b, lq, lk, h, kv, d = 2, 6 if form == "board" else 4, 6 if form == "board" else 9, 4, 2, 8
    q, k, v = (torch.randn(*s, dtype=torch.float64) for s in ((b, lq, h * maps, d), (b, lk, kv * maps, d), (b, lk, kv, d * maps)))
    table = torch.randn(p.num_buckets, h * maps, dtype=torch.float64)
    lam = torch.rand(h, dtype=torch.float64) if maps == 2 else None
    mask = torch.rand(b, lk) < 0.6
    mask[1] = False
    off = 0 if form == "board" else 3
    if maps == 1:
        out = relative_attention(q, k, v, table, p, key_mask=mask, scale=0.4, query_offset=off)
    else:
        out = differential_attention(q, k, v, lam, table, p, key_mask=mask, scale=0.4, query_offset=off)
    want = _loops(q, k, v, lam, table, p.pairs(lq, lk, off), mask, 0.4)
    assert torch.allclose(out, want, rtol=1e-12, atol=1e-12) and bool((out[1] == 0).all())


def test_reference_gradients_by_differences():
    torch.manual_seed(3)
    p = RelativeBuckets.log(8, 5)
    mk = lambda *s: torch.randn(*s, dtype=torch.float64, requires_grad=True)  # noqa: E731
    mask = torch.tensor([[True, False, True, True, True], [False] * 5])
    assert torch.autograd.gradcheck(lambda q, k, v, t: relative_attention(q, k, v, t, p, key_mask=mask), (mk(2, 3, 2, 8), mk(2, 5, 1, 8), mk(2, 5, 1, 8), mk(8, 2)))
    assert torch.autograd.gradcheck(lambda q, k, v, lam, t: differential_attention(q, k, v, lam, t, p, key_mask=mask),
                                    (mk(2, 3, 4, 8), mk(2, 5, 2, 8), mk(2, 5, 1, 16), mk(2), mk(8, 4)))


def test_masked_rows_may_hold_anything():
    p = RelativeBuckets.log(8, 5)
    q, k, v, t = torch.randn(1, 3, 1, 8), torch.randn(1, 4, 1, 8), torch.randn(1, 4, 1, 8), torch.randn(8, 1)
    mask = torch.tensor([[True, True, False, True]])
    want = relative_attention(q, k, v, t, p, key_mask=mask)
    k[0, 2], v[0, 2] = math.nan, math.inf
    assert torch.equal(relative_attention(q, k, v, t, p, key_mask=mask), want)


def test_refusals():
    p, board = RelativeBuckets.log(8, 5), RelativeBuckets.board(2, 2)
    q = k = v = torch.randn(2, 4, 2, 16)
    t, tb = torch.randn(8, 2), torch.randn(9, 2)
    ok = dict(q=q, k=k, v=v, table=t, buckets=p)
    relative_attention(**ok)
    relative_attention(q, k, v, tb, board)
    half = torch.randn(2, 4, 2, 16, dtype=torch.float16)
    for change in (
        dict(q=q[0]), dict(q=half, k=half, v=half), dict(k=k.bfloat16()), dict(q=q[..., :12], k=k[..., :12], v=v[..., :12]), dict(k=k[:1]), dict(v=v[:, :3]),
        dict(k=torch.randn(2, 4, 3, 16), v=torch.randn(2, 4, 3, 16)), dict(k=k[:, :, :1]), dict(v=v[..., :8]), dict(table=t[:, :1]), dict(table=t[:7]),
        dict(table=t.long()), dict(buckets=board), dict(buckets=None), dict(key_mask=torch.ones(2, 4)), dict(key_mask=torch.ones(2, 3, dtype=torch.bool)),
        dict(query_offset=torch.zeros(2)), dict(query_offset=torch.zeros(3, dtype=torch.int32)), dict(query_offset=MAX_OFFSET + 1),
        dict(table=tb, buckets=board, query_offset=1), dict(table=tb, buckets=board, query_offset=torch.zeros(2, dtype=torch.int32)),
        dict(table=tb, buckets=board, q=q[:, :3]), dict(k=k.to("meta")), dict(table=t.to("meta")),
    ):
        with pytest.raises(ValueError):
            relative_attention(**{**ok, **change})
    wide = torch.randn(1, 2, 1, 136)
    with pytest.raises(ValueError):
        relative_attention(wide, wide, wide, t[:, :1], p)
    q2, k2, v2, lam = torch.randn(2, 4, 4, 16), torch.randn(2, 5, 2, 16), torch.randn(2, 5, 1, 32), torch.rand(2)
    differential_attention(q2, k2, v2, lam)
    differential_attention(q2, k2, v2, lam, query_offset=7)  # positions have no effect without a bias
    for args in ((q2[:, :, :3], k2, v2, lam), (q2, k2, v2[..., :16], lam), (q2, k2[:, :, :1], v2, lam), (q2, k2, v2, lam[:1]), (q2, k2, v2, None),
                 (q2, k2, v2, lam.long()), (q2, k2, v2, lam, torch.randn(8, 4)), (q2, k2, v2, lam, torch.randn(8, 2), p)):
        with pytest.raises(ValueError):
            differential_attention(*args)
    w = torch.randn(1, 2, 2, 72)
    with pytest.raises(ValueError):
        differential_attention(w, w, torch.randn(1, 2, 1, 144), torch.rand(1))


def test_plans_that_would_lead_outside_are_refused():
    good = RelativeBuckets.log(8, 6)
    fields = dict(num_buckets=8, radius=6, rows=0, cols=0, lut=good.lut, order=good.order, start=good.start)
    RelativeBuckets(**fields)
    low, high = good.lut.clone(), good.lut.clone()
    low[0], high[3] = -1, 8
    twice = good.order.clone()
    twice[0] = twice[1]
    for change in (dict(radius=7), dict(radius=-1), dict(radius=1 << 20), dict(num_buckets=9), dict(num_buckets=0), dict(cols=5), dict(rows=2, cols=3),
                   dict(lut=low), dict(lut=high), dict(order=twice), dict(order=good.order.flip(0).contiguous()), dict(lut=good.lut.long()),
                   dict(start=good.start + 1), dict(lut=torch.stack([good.lut, good.lut], 1)[:, 0])):
        with pytest.raises(ValueError, match="RelativeBuckets"):
            RelativeBuckets(**{**fields, **change})
    board = RelativeBuckets.board(3, 4)
    assert board.radius == 2 * 7 + 3 and board.num_buckets == 5 * 7


def _rules(tmp_path, body):  # noqa: ANN001, ANN202
    """Lines of whitespace-separated numbers printed by a program over the rules the kernels and their host side share."""
    if shutil.which("g++") is None:
        pytest.skip("no host compiler")
    header = Path(__file__).parent.parent / "alphatriangle_amd" / "csrc" / "hip" / "encoder_ops.h"
    src = tmp_path / "rules.cpp"
    src.write_text(f'#include "{header}"\n#include <cstdio>\n#include <initializer_list>\nusing namespace atrihip;\nint main() {{ {body} }}\n')
    subprocess.check_call(["g++", "-std=c++17", "-O1", str(src), "-o", str(tmp_path / "rules")])
    return [[int(x) for x in line.split()] for line in subprocess.check_output([str(tmp_path / "rules")], text=True).splitlines()]


def test_sums_by_position_share_a_row_only_where_it_pays(tmp_path):
    """One row of sums for all four waves (which then take turns) only where four rows do not fit or cost a workgroup per unit."""
    rows = _rules(tmp_path, """
      const int widths[5][2] = {{32, 1}, {64, 1}, {128, 1}, {32, 2}, {64, 2}};
      for (auto& w : widths) for (int bf16 = 0; bf16 < 2; ++bf16) for (int slots : {1, 65, 257, 455, 1001, 2416, 2417, 4095}) {
        const int form = enc_query_form(bf16, w[0], w[1], slots), waves = enc_waves(w[0], w[1], 0, enc_columns_of(w[0], w[1], 0, bf16, kEncQueries), bf16, kEncQueries);
        const int rows = enc_hist_rows(form, w[0], w[1], 0, slots, waves);
        std::printf("%d %d %d %d %d %d %d %d %d\\n", w[0], w[1], bf16, slots, form, waves, rows, enc_lds_bytes(form, w[0], w[1], 0, kEncQueries, slots, 1),
                    enc_lds_bytes(form, w[0], w[1], 0, kEncQueries, slots, 4));
      }""")
    assert len(rows) == 80
    chosen = {}
    for width, maps, bf16, slots, form, waves, n, one, four in rows:
        most = 160 * 1024
        assert one <= most and (n == 1 or four <= most)
        fits_one, fits_four = min(waves, most // one), min(waves, most // four)
        assert n == (4 if fits_four == fits_one else 1)
        assert form == (0 if bf16 else 2 if (width, maps) == (64, 2) and slots > 2416 else 1)
        chosen[width, maps, bf16, slots] = n
    assert chosen[64, 2, 0, 65] == chosen[64, 2, 0, 257] == chosen[32, 2, 0, 455] == chosen[64, 1, 0, 4095] == chosen[128, 1, 1, 4095] == 4
    assert chosen[64, 2, 0, 4095] == chosen[64, 1, 0, 1001] == 1


def test_planned_workgroups_fit_a_compute_unit(tmp_path):
    """What the launch planning counts as resident is what both the registers and the LDS of a unit hold."""
    rows = _rules(tmp_path, """
      for (int bf16 = 0; bf16 < 2; ++bf16) for (int maps = 1; maps < 3; ++maps) for (int d : {8, 32, 40, 64, 128}) {
        if (maps == 2 && d > 64) continue;
        for (int r : {-1, 0, 128, 500, 2047}) for (int pass = 0; pass < 3; ++pass) {
          if (maps == 1 && r < 0) continue;
          const int width = d <= 32 ? 32 : d <= 64 ? 64 : 128, slots = r < 0 ? 0 : 2 * r + 1;
          const int form = pass == kEncQueries ? enc_query_form(bf16, width, maps, slots) : bf16 ? kRowsBf16 : kRowsParts;
          const int waves = enc_waves(width, maps, 0, enc_columns(0, 4000, 4000, d, maps, bf16, pass), bf16, pass);
          const int lds = enc_lds_bytes(form, width, maps, 0, pass, slots, slots ? enc_hist_rows(form, width, maps, 0, slots, waves) : 0);
          std::printf("%d %d %d %d %d %d %d %d\\n", bf16, maps, d, r, pass, waves, lds, enc_workgroups(bf16, d, maps, r, 0, 4000, 4000, true, pass, true));
        }
      }""")
    held = {}
    for bf16, maps, d, r, which, waves, lds, n in rows:
        assert n == min(waves, 160 * 1024 // lds) >= 1
        held[bf16, maps, d, r, which] = n
    assert held[0, 2, 40, 128, 1] == held[0, 1, 64, 2047, 1] == held[1, 1, 128, 2047, 1] == 1  # the LDS holds fewer than the registers
    assert held[1, 1, 64, 128, 1] == held[0, 1, 32, 128, 1] == 2


def _kernels_host_side():  # noqa: ANN202
    """The extension without kernels bound to it: what it refuses, it refuses before a launch."""
    try:
        import alphatriangle_amd._atri_torch as ops
    except ImportError as exc:
        pytest.skip(f"extension not built: {exc}")
    return ops


def _raw_calls(ops):  # noqa: ANN001, ANN202  name -> (call of one tensor list, the tensors)
    q, table, lam = torch.randn(1, 4, 2, 8), torch.randn(8, 2), torch.rand(1)
    p = RelativeBuckets.log(8, 5)
    rows, row = torch.randn(3, 16), torch.randn(16)
    return {
        "relative": (lambda q, k, v, t: ops.attention(q, k, v, t, None, p.lut, p.order, p.start, p.radius, 0, 8, None, None, 0, 0.5), [q, q.clone(), q.clone(), table]),
        "differential": (lambda q, k, v, m: ops.attention(q, k, v, None, m, None, None, None, 0, 0, 0, None, None, 0, 0.5), [q, q.clone(), torch.randn(1, 4, 1, 16), lam]),
        "joint": (lambda x, z, g, *params: ops.gated_norm_residual(x, z, *params, g, 1e-5), [rows, rows.clone(), rows.clone(), *(row.clone() for _ in range(5))]),
    }


@pytest.mark.parametrize("name", ["relative", "differential", "joint"])
def test_forward_mode_tangents_are_refused(name):
    from torch.autograd import forward_ad

    call, args = _raw_calls(_kernels_host_side())[name]
    for i in range(len(args)):
        for leaf in (False, True):
            with forward_ad.dual_level():
                given = list(args)
                given[i] = forward_ad.make_dual(args[i].clone().requires_grad_(leaf), torch.ones_like(args[i]))
                with pytest.raises(NotImplementedError, match="reverse mode"):
                    call(*given)


@pytest.mark.parametrize("name", ["relative", "differential", "joint"])
def test_tracing_is_refused(name):
    """A trace would hold the output's allocation alone.  (The host path's elementary operations are traced as any.)"""
    from torch.fx.experimental.proxy_tensor import make_fx

    call, args = _raw_calls(_kernels_host_side())[name]
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(call, tuple(args), check_trace=False)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        make_fx(call)(*args)


def test_host_path_is_traced():
    p = RelativeBuckets.log(8, 5)
    q, t = torch.randn(1, 4, 2, 8), torch.randn(8, 2)
    traced = torch.jit.trace(lambda a, b: relative_attention(a, a, a, b, p), (q, t), check_trace=False)
    other = torch.randn(1, 4, 2, 8)
    assert torch.allclose(traced(other, t), relative_attention(other, other, other, t, p), rtol=1e-5, atol=1e-6)


def test_plans_under_another_default_device():
    """Their tables are values: made on the host, and held there where the default device holds none."""
    want = RelativeBuckets.log(8, 5), RelativeBuckets.board(2, 3)
    with torch.device("meta"):
        got = RelativeBuckets.log(8, 5), RelativeBuckets.board(2, 3)
    for a, b in zip(want, got):
        assert a.device == b.device == torch.device("cpu")
        assert all(torch.equal(getattr(a, n), getattr(b, n)) for n in ("lut", "order", "start"))


def test_one_map_needs_its_bias():
    q = torch.randn(1, 4, 2, 8)
    with pytest.raises(ValueError, match="table"):
        relative_attention(q, q, q, None, None)


@pytest.mark.parametrize("offset", [1.5, 2.0, True, None, "1", [1, 2], numpy.array(1.5), numpy.float32(2)])
def test_offsets_are_whole_numbers(offset):
    q, p = torch.randn(2, 4, 2, 8), RelativeBuckets.log(8, 5)
    with pytest.raises(ValueError, match="query_offset"):
        relative_attention(q, q, q, torch.randn(8, 2), p, query_offset=offset)
    relative_attention(q, q, q, torch.randn(8, 2), p, query_offset=numpy.int64(3))


@pytest.mark.parametrize("scale", [0.0, -1.0, 1e-38, 9e-31, 1e30, math.inf, math.nan])
def test_scales_that_would_lose_the_bias_are_refused(scale):
    q, t, p = torch.randn(1, 4, 2, 8), torch.randn(8, 2), RelativeBuckets.log(8, 5)
    with pytest.raises(ValueError, match="scale"):
        relative_attention(q, q, q, t, p, scale=scale)
    relative_attention(q, q, q, t, p, scale=1e-30)
