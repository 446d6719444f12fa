"""Attention operators for encoders beyond the default one: a learned relative position bias by buckets, and two-map
("differential") attention.

``relative_attention`` and ``differential_attention`` run the hand-written gfx950 kernels for CUDA tensors
(csrc/hip/encoder_attn_*.hip; they raise when the kernel library is missing) and the elementary composition of the same formulas
(:func:`attention_reference`) for host tensors.  Both are differentiable once, in reverse mode, in every tensor argument; on
the GPU they refuse tensors that carry a forward-mode tangent, and to be traced (``torch.jit.trace``, ``make_fx``).

* Types: fp32 or bf16 ``q`` / ``k`` / ``v`` of one type; ``table`` and ``lam`` in any floating type (used in fp32, their gradients
  are summed in at least 32 bits).  fp32 products carry all 24 bits of their operands, most of them as three bf16 parts.
* Infinities (in fp32 also values above 3.38e38) in rows that take part make the results they reach NaN, for an operand in several
  parts meets them as inf - inf or 0 inf: in fp32 those of every tensor, in bf16 those of ``v`` and of the output's gradient.
* bf16 results are rounded once, when they are written: in between, probabilities and score gradients meet the bf16 operands in 16 bits at
  least.  Where a backward pass is to come the output's probabilities carry 24 bits, so the last bit of some values may
  differ from a call without one; in fp32 the two are equal.
* Layouts: ``[batch, tokens, heads, dim]`` with any strides; a contiguous last dimension with 16-byte aligned rows is read in
  place, anything else is copied first.  Outputs and gradients follow the token / batch order of the tensor they belong to.
* Shared heads: ``k`` and ``v`` may have fewer heads than ``q`` (a divisor); their gradients are summed over the group.
* Masks: ``key_mask[b, j] == False`` takes key ``j`` of sample ``b`` out whatever its rows hold (NaN included); a sample without
  keys gives zero outputs and zero gradients.
* Results do not depend on the order in which workgroups run: no floating-point atomics.
* Graphs: forward and backward passes can be captured.  A call that takes gradients is refused inside a capture while an eager graph of
  one of its leaves lives that was made on the default stream.
"""

from __future__ import annotations

import copy
import math
import operator
from collections.abc import Callable
from dataclasses import dataclass

import torch

from .. import native

MAX_RADIUS = 2047     # largest position difference the kernels keep apart
MIN_SCALE = 1e-30     # the kernels hold the bias in units of 1 / scale, which has to stay a finite number
MAX_OFFSET = 1 << 29  # positions beyond this would let differences leave 32 bits


@dataclass(frozen=True)
class RelativeBuckets:
    """Which bucket a (query, key) pair's relative position falls into; built once per model (:meth:`log`, :meth:`board`).

    ``lut[d + radius]`` is the bucket of position difference ``d = pos(key) - pos(query)``, clamped to ``+-radius``;
    ``order`` / ``start`` list the differences of every bucket (the gradient's summation order).  Without a ``device`` plans are
    placed on the default one (on the host where that is ``meta``); :meth:`to` moves them."""

    num_buckets: int
    radius: int
    rows: int  # board size; 0: a sequence
    cols: int
    lut: torch.Tensor
    order: torch.Tensor
    start: torch.Tensor

    def __post_init__(self) -> None:
        """The kernels index with these tables: refuses what would lead them outside."""
        n = 2 * self.radius + 1
        if not 0 <= self.radius <= MAX_RADIUS or self.num_buckets < 1:
            raise ValueError(f"RelativeBuckets: a radius of 0 to {MAX_RADIUS} and a bucket, got {self.radius} and {self.num_buckets}")
        if (self.rows, self.cols) != (0, 0) and (self.rows < 1 or self.cols < 1 or self.radius != (self.rows - 1) * (2 * self.cols - 1) + self.cols - 1):
            raise ValueError(f"RelativeBuckets: radius {self.radius} is not that of a {self.rows} x {self.cols} board")
        tables = (self.lut, self.order, self.start)
        if [tuple(t.shape) for t in tables] != [(n,), (n,), (self.num_buckets + 1,)] or any(
            t.dtype != torch.int32 or not t.is_contiguous() or t.device != self.lut.device for t in tables
        ):
            raise ValueError(f"RelativeBuckets: lut and order are contiguous int32 [{n}], start [{self.num_buckets + 1}], on one device")
        lut, order, start = (t.cpu().long() for t in tables)
        if int(lut.min()) < 0 or int(lut.max()) >= self.num_buckets or not torch.equal(order.sort().values, torch.arange(n, device="cpu")):
            raise ValueError("RelativeBuckets: lut names buckets, order every difference once")
        if not torch.equal(start[1:], torch.bincount(lut, minlength=self.num_buckets).cumsum(0)) or int(start[0]) != 0 or not torch.equal(
            lut[order], lut.sort().values
        ):
            raise ValueError("RelativeBuckets: order lists the differences bucket by bucket, start where each bucket begins")

    @classmethod
    def _make(cls, lut: torch.Tensor, num_buckets: int, radius: int, rows: int, cols: int, device: torch.device | str | None) -> "RelativeBuckets":
        n = lut.numel()
        tables = torch.zeros(2 * n + num_buckets + 1, dtype=torch.int32, device="cpu")
        tables[:n] = lut
        tables[n : 2 * n] = torch.argsort(lut, stable=True)
        tables[2 * n + 1 :] = torch.bincount(lut, minlength=num_buckets).cumsum(0)
        plan = cls(num_buckets, radius, rows, cols, tables[:n], tables[n : 2 * n], tables[2 * n :])
        device = torch.get_default_device() if device is None else torch.device(device)
        return plan if device.type == "meta" else plan.to(device)

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

        lut = torch.tensor([bucket(d) for d in range(-max_distance, max_distance + 1)], dtype=torch.int64, device="cpu")
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
        return cls._make(torch.arange(n, dtype=torch.int64, device="cpu"), n, radius, rows, cols, device)

    @property
    def device(self) -> torch.device:
        return self.lut.device

    def to(self, device: torch.device | str) -> "RelativeBuckets":
        dev = torch.device(device)
        if dev == self.device:
            return self
        moved = copy.copy(self)  # checked when it was made: not read back from the device again
        for name in ("lut", "order", "start"):
            object.__setattr__(moved, name, getattr(self, name).to(dev))
        return moved

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


# ---------------------------------------------------------------------------------------------------------- operators
def _whole(x: object) -> bool:
    try:
        return not isinstance(x, bool) and operator.index(x) is not None  # type: ignore[arg-type]
    except TypeError:
        return False


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
    if table is None and lam is None:
        raise ValueError(f"{name}: a table and its buckets are needed")
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
    elif not _whole(query_offset):
        raise ValueError(f"{name}: query_offset is an int or an int32 [{b}], got {query_offset!r}")
    elif query_offset and buckets is not None and buckets.rows:
        raise ValueError(f"{name}: query_offset moves queries along a sequence, not on a board")
    elif abs(int(query_offset)) > MAX_OFFSET:
        raise ValueError(f"{name}: query_offset beyond {MAX_OFFSET}")
    if max(q.shape[1], lk) > MAX_OFFSET:
        raise ValueError(f"{name}: sequences of at most {MAX_OFFSET} tokens")
    dev = q.device
    for t in (k, v, table, lam, key_mask, query_offset if torch.is_tensor(query_offset) else None, buckets.lut if buckets is not None else None):
        if t is not None and t.device != dev:
            raise ValueError(f"{name}: all tensors (and the buckets) on {dev}, got one on {t.device}")


def _attend(name: str, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lam: torch.Tensor | None, table: torch.Tensor | None,
            buckets: RelativeBuckets | None, key_mask: torch.Tensor | None, scale: float | None, query_offset: int | torch.Tensor) -> torch.Tensor:
    _check(name, q, k, v, table, lam, buckets, key_mask, query_offset)
    scale = q.shape[3] ** -0.5 if scale is None else float(scale)
    if not MIN_SCALE <= scale < 1e30:
        raise ValueError(f"{name}: scale is in [{MIN_SCALE}, 1e30), got {scale}")
    if not q.is_cuda or q.numel() == 0 or k.numel() == 0:
        return attention_reference(q, k, v, lam, table, buckets, key_mask, scale, query_offset)
    qoff = None
    if torch.is_tensor(query_offset):
        qoff, query_offset = query_offset.expand(q.shape[0]).contiguous(), 0
    call = _ops or _load()
    if buckets is None:
        return call(q, k, v, None, lam, None, None, None, 0, 0, 0, key_mask, None, 0, scale)
    return call(q, k, v, table, lam, buckets.lut, buckets.order, buckets.start, buckets.radius, buckets.cols, buckets.num_buckets, key_mask, qoff,
                int(query_offset), scale)


_ops: Callable[..., torch.Tensor] | None = None


def _load() -> Callable[..., torch.Tensor]:
    """The kernels' host side (csrc/torch/encoder_ops.cpp)."""
    global _ops
    _ops = native.torch_ops().attention
    return _ops


def relative_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, buckets: RelativeBuckets, *,
                       key_mask: torch.Tensor | None = None, scale: float | None = None, query_offset: int | torch.Tensor = 0) -> torch.Tensor:
    """``softmax(scale q k^T + table[bucket(pos(key) - pos(query))]) v`` -> ``[B, Lq, H, D]``.

    ``q [B, Lq, H, D]``, ``k`` / ``v [B, Lk, KV, D]`` (``KV`` divides ``H``), ``D`` a multiple of 8 up to 128;
    ``table [buckets.num_buckets, H]`` is learned; values beyond ``3.4e38 scale`` count as that (-inf takes a pair out).  ``scale``
    defaults to ``D ** -0.5``.  For sequences query ``i`` stands at
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
