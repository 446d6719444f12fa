"""The joint between two blocks of a residual stream: the norm after a block, its gate and residual scale, the residual add
and the norm in front of the next block, as one operator.

``gated_norm_residual`` runs the gfx950 kernels for CUDA tensors (csrc/hip/residual_norm_kernels.hip: one launch forward, two
backward; it raises when the kernel library is missing) and the elementary composition (:func:`gated_norm_residual_reference`)
for host tensors.  It is differentiable once in every tensor argument; parameter gradients are summed in 32 bits in a fixed
order (no atomics).
"""

from __future__ import annotations

import ctypes as C

import torch
from torch.autograd.function import once_differentiable

from . import hipbind as hb

MAX_WIDTH = 4096


def gated_norm_residual_reference(x: torch.Tensor, z: torch.Tensor, scale: torch.Tensor, post_weight: torch.Tensor, post_bias: torch.Tensor,
                                  pre_weight: torch.Tensor, pre_bias: torch.Tensor, gate: torch.Tensor | None = None,
                                  eps: float = 1e-5) -> tuple[torch.Tensor, torch.Tensor]:
    """The formulas in elementary differentiable operations, in the inputs' type (at least fp32)."""
    wide = torch.promote_types(x.dtype, torch.float32)

    def norm(t: torch.Tensor, w: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
        c = t - t.mean(-1, keepdim=True)
        return c * torch.rsqrt((c * c).mean(-1, keepdim=True) + eps) * w.to(wide) + b.to(wide)

    branch = scale.to(wide) * norm(z.to(wide), post_weight, post_bias)
    y = x.to(wide) + (branch if gate is None else torch.sigmoid(gate.to(wide)) * branch)
    return y.to(x.dtype), norm(y, pre_weight, pre_bias).to(z.dtype)


class _ArgsC(C.Structure):
    _fields_ = (
        [(n, hb.VP) for n in ("x", "z", "gate", "scale", "post_w", "post_b", "pre_w", "pre_b", "y", "h", "stats", "dy", "dh", "dx", "dz", "dgate",
                              "part", "dparams")]
        + [("N", C.c_longlong)]
        + [(n, C.c_int) for n in ("D", "gate_mode", "groups")]
        + [("eps", C.c_float)]
    )


_rows_per_step: dict[int, int] = {}  # by width


def _workgroups(n: int, d: int, most: int) -> int:
    """Workgroups of a launch: one step each while there are few rows, then ``most`` that walk the rest."""
    per = _rows_per_step.get(d)
    if per is None:
        lib = hb.lib()
        size, rows = lib.atri_sizeof_resnorm, lib.atri_resnorm_rows
        size.restype = rows.restype = C.c_int
        if size() != C.sizeof(_ArgsC):
            raise hb.HipError(f"ABI mismatch: atri_sizeof_resnorm() = {size()} but ctypes has {C.sizeof(_ArgsC)} bytes")
        per = _rows_per_step[d] = int(rows(C.c_int(d)))
    return max(1, min(-(-n // per), most))


def _args(x: torch.Tensor, z: torch.Tensor, gate: torch.Tensor | None, params: list[torch.Tensor], eps: float) -> _ArgsC:
    a = _ArgsC()
    a.N, a.D, a.eps = x.numel() // x.shape[-1], x.shape[-1], eps
    a.gate_mode = 0 if gate is None else 2 if gate.shape == z.shape else 1
    for name, t in zip(("x", "z", "gate", "scale", "post_w", "post_b", "pre_w", "pre_b"), (x, z, gate, *params)):
        if t is not None:
            setattr(a, name, t.data_ptr())
    return a


def _types(x: torch.Tensor, z: torch.Tensor) -> tuple[C.c_int, C.c_int]:
    return hb.i32(x.dtype == torch.bfloat16), hb.i32(z.dtype == torch.bfloat16)


def _rows(t: torch.Tensor | None) -> torch.Tensor | None:
    """Contiguous rows on a 16-byte boundary (a copy where they are not)."""
    if t is None:
        return None
    t = t.detach().contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _forward(x, z, gate, params, eps, train):  # noqa: ANN001, ANN202
    y, h = torch.empty_like(x), torch.empty_like(z)
    a = _args(x, z, gate, params, eps)
    a.y, a.h = y.data_ptr(), h.data_ptr()
    stats = None
    if train:
        stats = torch.empty(a.N, 4, dtype=torch.float32, device=x.device)
        a.stats = stats.data_ptr()
    a.groups = _workgroups(a.N, a.D, 2048)
    hb.call("atri_resnorm_fwd", C.byref(a), *_types(x, z))
    return y, h, stats


class _GatedNormResidual(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, z, scale, post_weight, post_bias, pre_weight, pre_bias, gate, eps):  # noqa: ANN001
        given = (scale, post_weight, post_bias, pre_weight, pre_bias)
        with torch.cuda.device(x.device):
            xr, zr, gr = _rows(x), _rows(z), _rows(gate)
            params = [_rows(p.float()) for p in given]
            y, h, stats = _forward(xr, zr, gr, params, eps, True)
        ctx.save_for_backward(xr, zr, gr, stats, *params)
        ctx.like = [p.dtype for p in given]
        ctx.eps = eps
        ctx.set_materialize_grads(False)
        return y, h

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh):  # noqa: ANN001
        if dy is None and dh is None:
            return (None,) * 9
        x, z, gate, stats, *params = ctx.saved_tensors
        with torch.cuda.device(x.device):
            dy = _rows(dy.to(x.dtype)) if dy is not None else None
            dh = _rows(dh.to(z.dtype)) if dh is not None else None
            dx, dz = torch.empty_like(x), torch.empty_like(z)
            dgate = torch.empty_like(gate) if gate is not None else None
            a = _args(x, z, gate, params, ctx.eps)
            # many rows per workgroup keep the partial sums small beside the rows: 5 of a row each
            a.groups = _workgroups(a.N, a.D, 1024 if a.D <= 512 else 512)
            part = torch.empty(a.groups, 5, a.D, dtype=torch.float32, device=x.device)
            dparams = torch.empty(5, a.D, dtype=torch.float32, device=x.device)
            for name, t in (("stats", stats), ("dy", dy), ("dh", dh), ("dx", dx), ("dz", dz), ("dgate", dgate), ("part", part), ("dparams", dparams)):
                if t is not None:
                    setattr(a, name, t.data_ptr())
            hb.call("atri_resnorm_bwd", C.byref(a), *_types(x, z))
            each = [g.to(t) for g, t in zip(dparams.unbind(0), ctx.like)]
        return (dx, dz, *each, dgate, None)


def gated_norm_residual(x: torch.Tensor, z: torch.Tensor, scale: torch.Tensor, post_weight: torch.Tensor, post_bias: torch.Tensor,
                        pre_weight: torch.Tensor, pre_bias: torch.Tensor, *, gate: torch.Tensor | None = None,
                        eps: float = 1e-5) -> tuple[torch.Tensor, torch.Tensor]:
    """``y = x + scale * sigmoid(gate) * LN(z; post)`` and ``h = LN(y; pre)`` -> ``(y, h)``.

    ``x [..., D]`` is the residual stream (fp32, or bf16 with a bf16 branch), ``z [..., D]`` the block's output (fp32 or bf16),
    ``scale`` / ``post_*`` / ``pre_*`` are learned ``[D]`` parameters of any floating type (used in fp32), ``gate`` holds logits in
    ``z``'s type, one per value ``[..., D]`` or one per row ``[..., 1]``; without it the branch is open.  ``y`` comes in ``x``'s type,
    ``h`` (taken from the unrounded ``y``) in ``z``'s.  ``D`` is at most 4096.
    """
    name = "gated_norm_residual"
    if x.dim() < 1 or x.shape != z.shape:
        raise ValueError(f"{name}: x and z of one shape, got {tuple(x.shape)} and {tuple(z.shape)}")
    d = x.shape[-1]
    kinds = ((torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16))
    if (x.dtype, z.dtype) not in kinds and (x.is_cuda or x.dtype != torch.float64 or z.dtype != torch.float64):
        raise ValueError(f"{name}: x / z in fp32 / fp32, fp32 / bf16 or bf16 / bf16, got {x.dtype} / {z.dtype}")
    if not 1 <= d <= MAX_WIDTH:
        raise ValueError(f"{name}: widths of 1 to {MAX_WIDTH}, got {d}")
    for p in (scale, post_weight, post_bias, pre_weight, pre_bias):
        if tuple(p.shape) != (d,) or not p.is_floating_point():
            raise ValueError(f"{name}: parameters are floating [{d}], got {tuple(p.shape)} {p.dtype}")
    if gate is not None and (gate.dtype != z.dtype or tuple(gate.shape) not in (tuple(z.shape), (*z.shape[:-1], 1))):
        raise ValueError(f"{name}: gate is [..., {d}] or [..., 1] in {z.dtype}, got {tuple(gate.shape)} {gate.dtype}")
    if not eps > 0:
        raise ValueError(f"{name}: eps must be positive, got {eps}")
    tensors = [t for t in (x, z, scale, post_weight, post_bias, pre_weight, pre_bias, gate) if t is not None]
    if any(t.device != x.device for t in tensors):
        raise ValueError(f"{name}: all tensors on {x.device}, got {[str(t.device) for t in tensors]}")
    if not x.is_cuda or x.numel() == 0:
        return gated_norm_residual_reference(x, z, scale, post_weight, post_bias, pre_weight, pre_bias, gate, eps)
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        return _GatedNormResidual.apply(x, z, scale, post_weight, post_bias, pre_weight, pre_bias, gate, float(eps))
    with torch.cuda.device(x.device):
        params = [_rows(p.float()) for p in (scale, post_weight, post_bias, pre_weight, pre_bias)]
        return _forward(_rows(x), _rows(z), _rows(gate), params, float(eps), False)[:2]
