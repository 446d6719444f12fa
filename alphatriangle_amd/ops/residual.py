"""The joint between two blocks of a residual stream: the norm after a block, its gate and residual scale, the residual add
and the norm in front of the next block, as one operator.

``gated_norm_residual`` runs the gfx950 kernels for CUDA tensors (csrc/hip/residual_norm_kernels.hip: one launch forward, two
backward; it raises when the kernel library is missing) and the elementary composition (:func:`gated_norm_residual_reference`)
for host tensors.  It is differentiable once in every tensor argument; parameter gradients are summed in 32 bits in a fixed
order (no atomics).
"""

from __future__ import annotations

import ctypes as C
import struct

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


# ResNormArgs of csrc/hip/residual_norm_kernels.hip: 18 pointers, the row count, 5 ints, 1 float.
_PACK = struct.Struct("=18qq5if")
_rows_per_step: dict[int, int] = {}  # by width


def _workgroups(n: int, d: int, most: int) -> int:
    """Workgroups of a launch: one step each while there are few rows, then ``most`` that walk the rest."""
    per = _rows_per_step.get(d)
    if per is None:
        lib = hb.lib()
        size, rows = lib.atri_sizeof_resnorm, lib.atri_resnorm_rows
        size.restype = rows.restype = C.c_int
        if size() != _PACK.size:
            raise hb.HipError(f"ABI mismatch: atri_sizeof_resnorm() = {size()} but {_PACK.size} bytes are packed")
        per = _rows_per_step[d] = int(rows(C.c_int(d)))
    return max(1, min(-(-n // per), most))


def _rows(t: torch.Tensor) -> torch.Tensor:
    """Contiguous rows on a 16-byte boundary (a copy where they are not)."""
    t = t.detach().contiguous()
    return t if not t.data_ptr() & 15 else t.clone()


def _param(t: torch.Tensor) -> torch.Tensor:
    return _rows(t if t.dtype == torch.float32 else t.float())


def _gate_mode(z: torch.Tensor, gate: torch.Tensor | None) -> int:
    return 0 if gate is None else 2 if gate.shape == z.shape else 1


def _forward(x: torch.Tensor, z: torch.Tensor, gate: torch.Tensor | None, params: tuple[torch.Tensor, ...], eps: float,
             train: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
    y, h = torch.empty_like(x), torch.empty_like(z)
    d = x.shape[-1]
    n = x.numel() // d
    stats = torch.empty(n, 4, dtype=torch.float32, device=x.device) if train else None
    hb.call_packed("atri_resnorm_fwd", _PACK.pack(
        x.data_ptr(), z.data_ptr(), gate.data_ptr() if gate is not None else 0, *[p.data_ptr() for p in params], y.data_ptr(), h.data_ptr(),
        stats.data_ptr() if stats is not None else 0, 0, 0, 0, 0, 0, 0, 0, n, d, _gate_mode(z, gate), _workgroups(n, d, 2048),
        x.dtype == torch.bfloat16, z.dtype == torch.bfloat16, eps), x.device.index)
    return y, h, stats


class _GatedNormResidual(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, z, scale, post_weight, post_bias, pre_weight, pre_bias, gate, eps):  # noqa: ANN001
        given = (scale, post_weight, post_bias, pre_weight, pre_bias)
        with hb.on_device(x.device.index):
            xr, zr, gr = _rows(x), _rows(z), _rows(gate) if gate is not None else None
            params = tuple(_param(p) for p in given)
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
        with hb.on_device(x.device.index):
            dy = _rows(dy.to(x.dtype)) if dy is not None else None
            dh = _rows(dh.to(z.dtype)) if dh is not None else None
            dx, dz = torch.empty_like(x), torch.empty_like(z)
            dgate = torch.empty_like(gate) if gate is not None else None
            d = x.shape[-1]
            n = x.numel() // d
            # many rows per workgroup keep the partial sums small beside the rows: 5 of a row each
            groups = _workgroups(n, d, 1024 if d <= 512 else 512)
            part = torch.empty(groups, 5, d, dtype=torch.float32, device=x.device)
            dparams = torch.empty(5, d, dtype=torch.float32, device=x.device)
            hb.call_packed("atri_resnorm_bwd", _PACK.pack(
                x.data_ptr(), z.data_ptr(), gate.data_ptr() if gate is not None else 0, *[p.data_ptr() for p in params], 0, 0, stats.data_ptr(),
                dy.data_ptr() if dy is not None else 0, dh.data_ptr() if dh is not None else 0, dx.data_ptr(), dz.data_ptr(),
                dgate.data_ptr() if gate is not None else 0, part.data_ptr(), dparams.data_ptr(), n, d, _gate_mode(z, gate), groups,
                x.dtype == torch.bfloat16, z.dtype == torch.bfloat16, ctx.eps), x.device.index)
            each = [g if t == torch.float32 else g.to(t) for g, t in zip(dparams.unbind(0), ctx.like)]
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
    params = (scale, post_weight, post_bias, pre_weight, pre_bias)
    dev = x.device
    grads = x.requires_grad or z.requires_grad or (gate is not None and gate.requires_grad)
    for t in (z, *params, gate):
        if t is not None and t.device != dev:
            raise ValueError(f"{name}: all tensors on {dev}, got one on {t.device}")
    if not x.is_cuda or x.numel() == 0:
        return gated_norm_residual_reference(x, z, *params, gate, eps)
    if torch.is_grad_enabled() and (grads or any([p.requires_grad for p in params])):
        return _GatedNormResidual.apply(x, z, *params, gate, float(eps))
    with hb.on_device(dev.index):
        return _forward(_rows(x), _rows(z), _rows(gate) if gate is not None else None, tuple(_param(p) for p in params), float(eps), False)[:2]
