"""The joint between two blocks of a residual stream: the norm after a block, its gate and residual scale, the residual add
and the norm in front of the next block, as one operator.

``gated_norm_residual`` runs the gfx950 kernels for CUDA tensors (csrc/hip/residual_norm_kernels.hip: one launch forward, two
backward; it raises when the kernel library is missing) and the elementary composition (:func:`gated_norm_residual_reference`)
for host tensors.  It is differentiable once, in reverse mode, in every tensor argument (on the GPU it refuses tensors that carry a
forward-mode tangent, to be traced by ``torch.jit.trace`` or ``make_fx``, and to be captured with gradients beside an eager
graph of the same leaves); parameter gradients are summed in 32 bits in a fixed order (no atomics).
"""

from __future__ import annotations

import torch

from .. import native

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
    params = (scale, post_weight, post_bias, pre_weight, pre_bias)
    for p in params:
        if tuple(p.shape) != (d,) or not p.is_floating_point():
            raise ValueError(f"{name}: parameters are floating [{d}], got {tuple(p.shape)} {p.dtype}")
    if gate is not None and (gate.dtype != z.dtype or tuple(gate.shape) not in (tuple(z.shape), (*z.shape[:-1], 1))):
        raise ValueError(f"{name}: gate is [..., {d}] or [..., 1] in {z.dtype}, got {tuple(gate.shape)} {gate.dtype}")
    if not eps > 0:
        raise ValueError(f"{name}: eps must be positive, got {eps}")
    dev = x.device
    for t in (z, *params, gate):
        if t is not None and t.device != dev:
            raise ValueError(f"{name}: all tensors on {dev}, got one on {t.device}")
    if not x.is_cuda or x.numel() == 0:
        return gated_norm_residual_reference(x, z, *params, gate, eps)
    return native.torch_ops().gated_norm_residual(x, z, *params, gate, float(eps))
