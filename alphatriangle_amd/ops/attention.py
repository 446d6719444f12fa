"""Attention operators for encoders beyond the default one: a learned relative position bias by buckets, and two-map
("differential") attention.

``relative_attention`` and ``differential_attention`` run the hand-written gfx950 kernels for CUDA tensors
(csrc/hip/encoder_attn_*.hip; they raise when the kernel library is missing) and the elementary composition of the same formulas
(:func:`attention_reference`) for host tensors.  Both are differentiable once in every tensor argument.

* Types: fp32 or bf16 ``q`` / ``k`` / ``v`` of one type; ``table`` and ``lam`` in any floating type (used in fp32, their gradients
  are summed in at least 32 bits).  fp32 products are true fp32 products.
* Layouts: ``[batch, tokens, heads, dim]`` with any strides; a contiguous last dimension with 16-byte aligned rows is read in
  place, anything else is copied first.  Outputs and gradients follow the token / batch order of the tensor they belong to.
* Shared heads: ``k`` and ``v`` may have fewer heads than ``q`` (a divisor); their gradients are summed over the group.
* Masks: ``key_mask[b, j] == False`` takes key ``j`` of sample ``b`` out whatever its rows hold (NaN included); a sample without
  keys gives zero outputs and zero gradients.
* Results do not depend on the order in which workgroups run: no floating-point atomics.
"""

from __future__ import annotations

import ctypes as C
import math
from dataclasses import dataclass

import torch
from torch.autograd.function import once_differentiable

from . import hipbind as hb

MAX_RADIUS = 2047     # largest position difference the kernels keep apart
MAX_OFFSET = 1 << 29  # positions beyond this would let differences leave 32 bits


@dataclass(frozen=True)
class RelativeBuckets:
    """Which bucket a (query, key) pair's relative position falls into; built once per model (:meth:`log`, :meth:`board`).

    ``lut[d + radius]`` is the bucket of position difference ``d = pos(key) - pos(query)``, clamped to ``+-radius``;
    ``order`` / ``start`` list the differences of every bucket (the gradient's summation order)."""

    num_buckets: int
    radius: int
    rows: int  # board size; 0: a sequence
    cols: int
    lut: torch.Tensor
    order: torch.Tensor
    start: torch.Tensor

    @classmethod
    def _make(cls, lut: torch.Tensor, num_buckets: int, radius: int, rows: int, cols: int, device: torch.device | str | None) -> "RelativeBuckets":
        n = lut.numel()
        tables = torch.zeros(2 * n + num_buckets + 1, dtype=torch.int32)  # one upload
        tables[:n] = lut
        tables[n : 2 * n] = torch.argsort(lut, stable=True)
        tables[2 * n + 1 :] = torch.bincount(lut, minlength=num_buckets).cumsum(0)
        tables = tables.to("cpu" if device is None else device)
        return cls(num_buckets, radius, rows, cols, tables[:n], tables[n : 2 * n], tables[2 * n :])

    @classmethod
    def log(cls, num_buckets: int = 32, max_distance: int = 128, *, device: torch.device | str | None = None) -> "RelativeBuckets":
        """Sequences: half of the buckets for keys at or before the query, half for keys behind it; within each half one
        bucket per distance up to a quarter of ``num_buckets``, then logarithmically wider ones up to ``max_distance``."""
        if num_buckets < 4 or num_buckets % 2:
            raise ValueError(f"num_buckets must be even and at least 4, got {num_buckets}")
        half = num_buckets // 2
        exact = half // 2
        if not exact < max_distance <= MAX_RADIUS:
            raise ValueError(f"max_distance must be in ({exact}, {MAX_RADIUS}], got {max_distance}")

        def bucket(d: int) -> int:
            n = abs(d)
            if n >= exact:
                n = min(half - 1, exact + math.floor(math.log(n / exact) / math.log(max_distance / exact) * (half - exact) + 1e-9))
            return n + (half if d > 0 else 0)

        lut = torch.tensor([bucket(d) for d in range(-max_distance, max_distance + 1)], dtype=torch.int64)
        return cls._make(lut, num_buckets, max_distance, 0, 0, device)

    @classmethod
    def board(cls, rows: int, cols: int, *, device: torch.device | str | None = None) -> "RelativeBuckets":
        """Cells of a ``rows x cols`` board in row-major order: one bucket per (row difference, column difference),
        ``(dr + rows - 1) * (2 cols - 1) + dc + cols - 1``."""
        if rows < 1 or cols < 1:
            raise ValueError(f"a board needs rows and columns, got {rows} x {cols}")
        radius = (rows - 1) * (2 * cols - 1) + cols - 1
        if radius > MAX_RADIUS:
            raise ValueError(f"a {rows} x {cols} board has {2 * radius + 1} relative positions; at most {2 * MAX_RADIUS + 1} are supported")
        n = (2 * rows - 1) * (2 * cols - 1)
        return cls._make(torch.arange(n, dtype=torch.int64), n, radius, rows, cols, device)

    @property
    def device(self) -> torch.device:
        return self.lut.device

    def to(self, device: torch.device | str) -> "RelativeBuckets":
        dev = torch.device(device)
        if dev == self.device:
            return self
        return RelativeBuckets(self.num_buckets, self.radius, self.rows, self.cols, self.lut.to(dev), self.order.to(dev), self.start.to(dev))

    def pairs(self, lq: int, lk: int, query_offset: int | torch.Tensor = 0) -> torch.Tensor:
        """Bucket of every pair, ``[lq, lk]`` (``[batch, lq, lk]`` for per-sample offsets): what the kernels look up."""
        dev = self.device
        qt, kt = torch.arange(lq, device=dev), torch.arange(lk, device=dev)
        if self.rows:
            qp, kp = (t + torch.div(t, self.cols, rounding_mode="floor") * (self.cols - 1) for t in (qt, kt))
        else:
            off = query_offset.to(dev).long().view(-1, 1) if torch.is_tensor(query_offset) else query_offset
            qp, kp = qt + off, kt
        diff = (kp - qp.unsqueeze(-1)).clamp(-self.radius, self.radius)
        return self.lut.long()[diff + self.radius]


# -------------------------------------------------------------------------------------------------------- reference
def attention_reference(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lam: torch.Tensor | None, table: torch.Tensor | None,
                        buckets: RelativeBuckets | None, key_mask: torch.Tensor | None, scale: float,
                        query_offset: int | torch.Tensor = 0) -> torch.Tensor:
    """The formulas in elementary differentiable operations, computed in the inputs' type (at least fp32), any device."""
    maps = 1 if lam is None else 2
    wide = torch.promote_types(q.dtype, torch.float32)
    b, lq, hm, d = q.shape
    lk, kv = k.shape[1], v.shape[2]
    h = hm // maps
    qq = q.to(wide).view(b, lq, h, maps, d).permute(0, 2, 3, 1, 4)
    kk = k.to(wide).view(b, lk, kv, maps, d).permute(0, 2, 3, 1, 4)
    vv = v.to(wide).permute(0, 2, 1, 3)
    if key_mask is not None:  # masked rows may hold anything
        kk = torch.where(key_mask[:, None, None, :, None], kk, 0.0)
        vv = torch.where(key_mask[:, None, :, None], vv, 0.0)
    kk, vv = kk.repeat_interleave(h // kv, 1), vv.repeat_interleave(h // kv, 1)
    s = torch.matmul(qq.contiguous(), kk.transpose(-1, -2).contiguous()) * scale
    if table is not None and buckets is not None:
        bias = table.to(wide)[buckets.pairs(lq, lk, query_offset)]
        bias = bias.view(*bias.shape[:-1], h, maps)
        s = s + (bias.permute(2, 3, 0, 1) if bias.dim() == 4 else bias.permute(0, 3, 4, 1, 2))
    if key_mask is not None:
        s = s.masked_fill(~key_mask[:, None, None, None, :], -math.inf)
    top = s.detach().amax(-1, keepdim=True) if lk else s.new_zeros(*s.shape[:-1], 1)
    e = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, 1.0, total)
    att = p[:, :, 0] if lam is None else p[:, :, 0] - lam.to(wide).view(h, 1, 1) * p[:, :, 1]
    return torch.matmul(att.contiguous(), vv.contiguous()).permute(0, 2, 1, 3).to(q.dtype)


# ---------------------------------------------------------------------------------------------------------- kernels
class _ArgsC(C.Structure):
    _fields_ = (
        [(n, hb.VP) for n in ("q", "k", "v", "dout", "out", "dq", "dk", "dv", "table", "lut", "lam", "words", "qoff", "stat", "o32",
                              "delta", "part_o", "part_ml", "hist")]
        + [(n, C.c_longlong * 3) for n in ("qs", "ks", "vs", "os", "gs", "dqs", "dks", "dvs")]
        + [("o32s", C.c_longlong * 4)]
        + [(n, C.c_int) for n in ("B", "Lq", "Lk", "H", "KV", "D", "DV", "M", "R", "W", "q0", "bf16", "splits", "hist_rows")]
        + [("scale", C.c_float)]
    )


_abi_checked = False


def _check_abi() -> None:
    global _abi_checked
    if not _abi_checked:
        fn = hb.lib().atri_sizeof_encattn
        fn.restype = C.c_int
        if fn() != C.sizeof(_ArgsC):
            raise hb.HipError(f"ABI mismatch: atri_sizeof_encattn() = {fn()} but ctypes has {C.sizeof(_ArgsC)} bytes")
        _abi_checked = True


def _rows_ok(t: torch.Tensor) -> bool:
    vec = 16 // t.element_size()
    return t.data_ptr() % 16 == 0 and (t.stride(3) == 1 or t.shape[3] == 1) and all(t.stride(i) % vec == 0 for i in range(3) if t.shape[i] > 1)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` as the kernels can read it: in place when its rows are contiguous and 16-byte aligned, else a copy."""
    return t if _rows_ok(t) else t.contiguous()


def _strides(t: torch.Tensor) -> tuple[int, int, int]:
    return tuple(0 if t.shape[i] == 1 else t.stride(i) for i in range(3))  # type: ignore[return-value]


def _empty_like_rows(t: torch.Tensor, heads: int, width: int, dtype: torch.dtype) -> torch.Tensor:
    """New ``[B, L, heads, width]`` in the token / batch order of ``t``."""
    b, n = t.shape[:2]
    if b > 1 and n > 1 and t.stride(0) < t.stride(1):
        return torch.empty(n, b, heads, width, dtype=dtype, device=t.device).transpose(0, 1)
    return torch.empty(b, n, heads, width, dtype=dtype, device=t.device)


def _fill(a: _ArgsC, **tensors: tuple[torch.Tensor, str] | torch.Tensor | None) -> None:
    for name, t in tensors.items():
        if t is None:
            continue
        if isinstance(t, tuple):
            getattr(a, t[1])[:] = _strides(t[0])
            t = t[0]
        setattr(a, name, t.data_ptr())


def _splits(b: int, h: int, lq: int, lk: int, wide: bool) -> int:
    """Key ranges per query tile: one unless the (sample, head, query tile) workgroups leave compute units idle, then about
    four workgroups per CU with at least four key tiles each (a range's partial output costs a write, a read and the join)."""
    groups = b * h * -(-lq // (128 if wide else 64))
    tiles = -(-lk // 64)
    if groups >= 512 or tiles < 8:
        return 1
    return max(1, min(-(-1024 // groups), tiles // 4, 256))


@dataclass
class _Call:
    """What one call fixes besides its tensors."""

    buckets: RelativeBuckets | None
    mask: torch.Tensor | None
    qoff: torch.Tensor | None
    q0: int
    scale: float
    maps: int


def _base_args(c: _Call, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor | None, lam: torch.Tensor | None,
               words: torch.Tensor | None) -> _ArgsC:
    a = _ArgsC()
    a.B, a.Lq, a.Lk = q.shape[0], q.shape[1], k.shape[1]
    a.H, a.KV, a.D, a.DV, a.M = q.shape[2] // c.maps, v.shape[2], q.shape[3], v.shape[3], c.maps
    a.bf16, a.splits, a.hist_rows, a.q0, a.scale = int(q.dtype == torch.bfloat16), 1, 4, c.q0, c.scale
    _fill(a, q=(q, "qs"), k=(k, "ks"), v=(v, "vs"), table=table, lam=lam, words=words, qoff=c.qoff)
    if table is not None and c.buckets is not None:
        a.R, a.W, a.lut = c.buckets.radius, c.buckets.cols, c.buckets.lut.data_ptr()
    return a


def _forward(c: _Call, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor | None, lam: torch.Tensor | None,
             train: bool) -> tuple[torch.Tensor, torch.Tensor | None, torch.Tensor | None, torch.Tensor | None]:
    """``out`` and, for a backward pass, (stat, o32, words); operands as the kernels read them, fp32 table and lam."""
    _check_abi()
    b, lq, hm, _ = q.shape
    lk, h, dv = k.shape[1], hm // c.maps, v.shape[3]
    dev = q.device
    out = _empty_like_rows(q, h, dv, q.dtype)
    words = None
    if c.mask is not None:
        words = torch.empty(b, -(-lk // 64), dtype=torch.int64, device=dev)
        hb.call("atri_enc_key_words", hb.ptr(c.mask), hb.i64(c.mask.stride(0)), hb.i64(c.mask.stride(1)), hb.ptr(words), hb.i32(b), hb.i32(lk))
    a = _base_args(c, q, k, v, table, lam, words)
    _fill(a, out=(out, "os"))
    stat = o32 = None
    if train:
        stat = torch.empty(c.maps, b * h * lq, 2, dtype=torch.float32, device=dev)
        if c.maps == 2 or q.dtype != torch.float32:  # delta = dO . o needs every map's output in 32 bits
            o32 = torch.empty(c.maps, b, h, lq, dv, dtype=torch.float32, device=dev)
            a.o32s[:] = (o32.stride(1), o32.stride(3), o32.stride(2), o32.stride(0))
        _fill(a, stat=stat, o32=o32)
    a.splits = _splits(b, h, lq, lk, c.maps == 1 and q.shape[3] <= 64 and lq > 64)
    part = None
    if a.splits > 1:
        rows = a.splits * c.maps * b * h * lq
        part = torch.empty(rows * (dv + 2), dtype=torch.float32, device=dev)
        a.part_o, a.part_ml = part.data_ptr(), part.data_ptr() + 4 * rows * dv
    hb.call("atri_enc_attn_fwd", C.byref(a))
    return out, stat, o32, words


def _backward(c: _Call, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor | None, lam: torch.Tensor | None,
              o32: torch.Tensor, stat: torch.Tensor, words: torch.Tensor | None, dout: torch.Tensor, dq: torch.Tensor, dk: torch.Tensor,
              dv: torch.Tensor, want_table: bool, want_lam: bool) -> tuple[torch.Tensor | None, torch.Tensor | None]:
    """Fills ``dq`` / ``dk`` / ``dv`` (strided, every element) and returns ``(dtable, dlam)`` in fp32.  ``o32`` is the per-map
    output ``[M, B, H, Lq, DV]`` or, for one fp32 map, the output itself ``[B, Lq, H, DV]``."""
    b, lq, hm, d = q.shape
    h, dev = hm // c.maps, q.device
    a = _base_args(c, q, k, v, table, lam, words)
    delta = torch.empty(c.maps, b * h * lq, dtype=torch.float32, device=dev)
    _fill(a, dout=(dout, "gs"), dq=(dq, "dqs"), dk=(dk, "dks"), dv=(dv, "dvs"), stat=stat, delta=delta, o32=o32)
    a.o32s[:] = (o32.stride(1), o32.stride(3), o32.stride(2), o32.stride(0)) if o32.dim() == 5 else (*_strides(o32), 0)
    hist, nqt, slots = None, 0, 0
    if want_table and table is not None and c.buckets is not None:
        per = hb.lib().atri_enc_attn_bwd_queries
        per.restype = C.c_int
        nqt, slots = -(-lq // per(C.c_int(d), C.c_int(c.maps))), 2 * c.buckets.radius + 1
        hist = torch.empty(b * h * nqt, c.maps, slots, dtype=torch.float32, device=dev)
        a.hist = hist.data_ptr()
    hb.call("atri_enc_attn_bwd", C.byref(a))
    dtable = dlam = None
    if hist is not None and table is not None and c.buckets is not None:
        shares = max(1, min(64, b * nqt // 16))
        mid = torch.empty(shares, hm, slots, dtype=torch.float32, device=dev)
        dtable = torch.empty(c.buckets.num_buckets, hm, dtype=torch.float32, device=dev)
        hb.call("atri_enc_table_grad", hb.ptr(hist), hb.ptr(mid), hb.ptr(c.buckets.order), hb.ptr(c.buckets.start), hb.ptr(dtable), hb.i32(b),
                hb.i32(h), hb.i32(c.maps), hb.i32(nqt), hb.i32(slots), hb.i32(c.buckets.num_buckets), hb.i32(shares))
    if want_lam and lam is not None:
        dlam = torch.empty(h, dtype=torch.float32, device=dev)
        hb.call("atri_enc_dlam", hb.ptr(delta[1]), hb.ptr(dlam), hb.i32(b), hb.i32(h), hb.i32(lq))
    return dtable, dlam


def _f32(t: torch.Tensor | None) -> torch.Tensor | None:
    return None if t is None else t.detach().float().contiguous()


class _EncoderAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, table, lam, call):  # noqa: ANN001
        qr, kr, vr = _rows(q.detach()), _rows(k.detach()), _rows(v.detach())
        t32, l32 = _f32(table), _f32(lam)
        with torch.cuda.device(q.device):
            out, stat, o32, words = _forward(call, qr, kr, vr, t32, l32, True)
        ctx.call = call
        ctx.like = (table.dtype if table is not None else None, lam.dtype if lam is not None else None)
        ctx.save_for_backward(qr, kr, vr, t32, l32, out if o32 is None else o32, stat, words)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):  # noqa: ANN001
        q, k, v, table, lam, o32, stat, words = ctx.saved_tensors
        c = ctx.call
        with torch.cuda.device(q.device):
            dq, dk, dv = (_empty_like_rows(t, t.shape[2], t.shape[3], t.dtype) for t in (q, k, v))
            dtable, dlam = _backward(c, q, k, v, table, lam, o32, stat, words, _rows(dout.to(q.dtype)), dq, dk, dv, ctx.needs_input_grad[3],
                                     ctx.needs_input_grad[4])
            if dtable is not None:
                dtable = dtable.to(ctx.like[0])
            if dlam is not None:
                dlam = dlam.to(ctx.like[1])
        return dq, dk, dv, dtable, dlam, None


def _check(name: str, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor | None, lam: torch.Tensor | None,
           buckets: RelativeBuckets | None, key_mask: torch.Tensor | None, query_offset: int | torch.Tensor) -> None:
    maps = 1 if lam is None else 2
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError(f"{name}: q, k and v are [batch, tokens, heads, dim], got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if q.dtype not in (torch.float32, torch.bfloat16) and (q.is_cuda or q.dtype != torch.float64):
        raise ValueError(f"{name}: fp32 or bf16 operands, got {q.dtype}")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"{name}: q, k and v of one type, got {q.dtype}, {k.dtype}, {v.dtype}")
    b, _, hm, d = q.shape
    lk, kv = k.shape[1], v.shape[2]
    most = 128 if maps == 1 else 64
    if d % 8 or not 8 <= d <= most:
        raise ValueError(f"{name}: head widths are multiples of 8 up to {most}, got {d}")
    if hm % maps or hm < maps or k.shape[0] != b or k.shape[3] != d or k.shape[2] != kv * maps or tuple(v.shape[:2]) != (b, lk) or v.shape[3] != d * maps:
        raise ValueError(f"{name}: shapes do not belong together: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}")
    if kv < 1 or (hm // maps) % kv:
        raise ValueError(f"{name}: {hm // maps} heads cannot share {kv} key / value heads")
    if lam is not None and (tuple(lam.shape) != (hm // maps,) or not lam.is_floating_point()):
        raise ValueError(f"{name}: lam is one floating value per head, got {tuple(lam.shape)} {lam.dtype} for {hm // maps} heads")
    if (table is None) != (buckets is None):
        raise ValueError(f"{name}: table and buckets go together")
    if table is not None and buckets is not None:
        if tuple(table.shape) != (buckets.num_buckets, hm) or not table.is_floating_point():
            raise ValueError(f"{name}: table is a floating [{buckets.num_buckets}, {hm}], got {tuple(table.shape)} {table.dtype}")
        if buckets.rows and not (q.shape[1] == lk == buckets.rows * buckets.cols):
            raise ValueError(f"{name}: a {buckets.rows} x {buckets.cols} board has {buckets.rows * buckets.cols} tokens, got {q.shape[1]} queries and {lk} keys")
    if key_mask is not None and (key_mask.dtype != torch.bool or tuple(key_mask.shape) != (b, lk)):
        raise ValueError(f"{name}: key_mask is a bool [{b}, {lk}], got {tuple(key_mask.shape)} {key_mask.dtype}")
    if torch.is_tensor(query_offset):
        if tuple(query_offset.shape) not in ((b,), (1,)) or query_offset.dtype != torch.int32:
            raise ValueError(f"{name}: query_offset is an int or an int32 [{b}], got {tuple(query_offset.shape)} {query_offset.dtype}")
        if buckets is not None and buckets.rows:
            raise ValueError(f"{name}: query_offset moves queries along a sequence, not on a board")
    elif query_offset and buckets is not None and buckets.rows:
        raise ValueError(f"{name}: query_offset moves queries along a sequence, not on a board")
    elif abs(int(query_offset)) > MAX_OFFSET:
        raise ValueError(f"{name}: query_offset beyond {MAX_OFFSET}")
    if max(q.shape[1], lk) > MAX_OFFSET:
        raise ValueError(f"{name}: sequences of at most {MAX_OFFSET} tokens")
    others = [t for t in (k, v, table, lam, key_mask, query_offset if torch.is_tensor(query_offset) else None, buckets.lut if buckets else None)
              if t is not None]
    if any(t.device != q.device for t in others):
        raise ValueError(f"{name}: all tensors (and the buckets) on {q.device}, got {[str(t.device) for t in others]}")


def _attend(name: str, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lam: torch.Tensor | None, table: torch.Tensor | None,
            buckets: RelativeBuckets | None, key_mask: torch.Tensor | None, scale: float | None, query_offset: int | torch.Tensor) -> torch.Tensor:
    _check(name, q, k, v, table, lam, buckets, key_mask, query_offset)
    scale = q.shape[3] ** -0.5 if scale is None else float(scale)
    if not q.is_cuda or q.numel() == 0 or k.numel() == 0:
        return attention_reference(q, k, v, lam, table, buckets, key_mask, scale, query_offset)
    qoff = None
    if torch.is_tensor(query_offset):
        qoff = query_offset.expand(q.shape[0]).contiguous()
        query_offset = 0
    call = _Call(buckets, key_mask, qoff, int(query_offset), scale, 1 if lam is None else 2)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, table, lam)):
        return _EncoderAttention.apply(q, k, v, table, lam, call)
    with torch.cuda.device(q.device):
        return _forward(call, _rows(q.detach()), _rows(k.detach()), _rows(v.detach()), _f32(table), _f32(lam), False)[0]


def relative_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, buckets: RelativeBuckets, *,
                       key_mask: torch.Tensor | None = None, scale: float | None = None, query_offset: int | torch.Tensor = 0) -> torch.Tensor:
    """``softmax(scale q k^T + table[bucket(pos(key) - pos(query))]) v`` -> ``[B, Lq, H, D]``.

    ``q [B, Lq, H, D]``, ``k`` / ``v [B, Lk, KV, D]`` (``KV`` divides ``H``), ``D`` a multiple of 8 up to 128;
    ``table [buckets.num_buckets, H]`` is learned.  ``scale`` defaults to ``D ** -0.5``.  For sequences query ``i`` stands at
    position ``query_offset + i`` (an int, or an int32 ``[B]`` tensor: a new token behind each sample's own cache) and
    key ``j`` at ``j`` (without a bias positions have no effect); boards take all their cells as queries and keys.
    """
    return _attend("relative_attention", q, k, v, None, table, buckets, key_mask, scale, query_offset)


def differential_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lam: torch.Tensor, table: torch.Tensor | None = None,
                           buckets: RelativeBuckets | None = None, *, key_mask: torch.Tensor | None = None, scale: float | None = None,
                           query_offset: int | torch.Tensor = 0) -> torch.Tensor:
    """``(softmax(scale q1 k1^T + b1) - lam softmax(scale q2 k2^T + b2)) v`` -> ``[B, Lq, H, 2 D]``.

    Map ``m`` of head ``h`` is head ``2 h + m`` of ``q [B, Lq, 2 H, D]`` and ``k [B, Lk, 2 KV, D]`` (and column ``2 h + m`` of
    ``table``, if there is a bias); ``v`` is ``[B, Lk, KV, 2 D]``, ``lam [H]`` the learned weight of the second map, ``D`` a multiple
    of 8 up to 64.  Everything else as in :func:`relative_attention`.
    """
    if lam is None:
        raise ValueError("differential_attention: lam is one floating value per head")
    return _attend("differential_attention", q, k, v, lam, table, buckets, key_mask, scale, query_offset)
