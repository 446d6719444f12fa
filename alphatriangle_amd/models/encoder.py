"""Encoder variants of the policy / value network (``ModelConfig.TRANSFORMER_ATTENTION``, ``TRANSFORMER_NORM``).

Beside the default pre-norm softmax layer (:class:`~alphatriangle_amd.models.model.EncoderLayer`, the reference's
architecture) an encoder layer may use

* ``relative`` attention: a learned bias per relative board position and head (``ops.attention.relative_attention``);
* ``differential`` attention: pairs of heads whose softmax maps are subtracted with a learned weight
  (``ops.attention.differential_attention``, with the same kind of bias per map), the pair's output normalised;
* the ``sandwich`` norm: a norm behind each block as well as in front of it, a learned residual scale per channel and a
  sigmoid gate computed from the block's input (``ops.residual.gated_norm_residual``).

All three run on the GPU through hand-written kernels and on the host through the same formulas in PyTorch.
Probabilities of the relative and differential forms take no dropout (the branches and the feed-forward layer do).
"""

from __future__ import annotations

import math

import torch
import torch.nn as nn
import torch.nn.functional as F

from ..ops.attention import RelativeBuckets, differential_attention, relative_attention
from ..ops.residual import gated_norm_residual
from .model import EncoderLayer, FastLayerNorm, _linear_rows


def _rows(x: torch.Tensor, lin: nn.Linear | tuple[torch.Tensor, torch.Tensor]) -> torch.Tensor:
    """``lin`` over the last dimension: the learner's split-K rows on a GPU, the stock product on the host."""
    weight, bias = (lin.weight, lin.bias) if isinstance(lin, nn.Linear) else lin
    return _linear_rows(x, weight, bias) if x.is_cuda else F.linear(x, weight, bias)


class BoardEncoderLayer(EncoderLayer):
    """An encoder layer over the cells of a ``board = (rows, cols)``; ``[tokens, batch, dim]`` in and out."""

    def __init__(self, board: tuple[int, int], attention: str, sandwich: bool, index: int, **kwargs) -> None:  # noqa: ANN003
        super().__init__(**kwargs)
        d, heads = self.self_attn.embed_dim, self.self_attn.num_heads
        self.board, self.attention, self.sandwich = board, attention, sandwich
        if attention != "softmax":
            self.buckets = RelativeBuckets.board(*board)
            self.position_bias = nn.Parameter(torch.zeros(self.buckets.num_buckets, heads))
        if attention == "differential":
            hd = d // heads
            # the subtracted map starts at this weight: a fifth in the first layer, towards 0.8 in deep ones
            self.lambda_init = 0.8 - 0.6 * math.exp(-0.3 * index)
            for name in ("lambda_q1", "lambda_k1", "lambda_q2", "lambda_k2"):
                self.register_parameter(name, nn.Parameter(torch.randn(heads // 2, hd) * 0.1))
            self.head_norm = FastLayerNorm(2 * hd)
        if sandwich:
            for i in (1, 2):
                self.register_module(f"post_norm{i}", nn.LayerNorm(d))
                self.register_parameter(f"residual_scale{i}", nn.Parameter(torch.ones(d)))
                gate = nn.Linear(d, d)
                nn.init.zeros_(gate.weight)
                nn.init.constant_(gate.bias, 2.0)  # nearly open to begin with
                self.register_module(f"gate{i}", gate)

    def _lambda(self) -> torch.Tensor:
        """Weight of the subtracted map, one per pair of heads (fp32)."""
        with torch.autocast(device_type=self.lambda_q1.device.type, enabled=False):
            first = torch.exp((self.lambda_q1 * self.lambda_k1).sum(-1))
            second = torch.exp((self.lambda_q2 * self.lambda_k2).sum(-1))
            return first - second + self.lambda_init

    def _attend(self, y: torch.Tensor) -> torch.Tensor:
        """Self-attention of normalised tokens ``y`` including the output projection."""
        attn = self.self_attn
        seq, batch, d = y.shape
        heads, hd = attn.num_heads, d // attn.num_heads
        qkv = _rows(y, (attn.in_proj_weight, attn.in_proj_bias))
        if self.attention == "softmax":
            ctx = self._attention(qkv, seq, batch, d, heads)
        else:
            if self.buckets.device != y.device:
                self.buckets = self.buckets.to(y.device)
            q, k, v = (t.transpose(0, 1) for t in qkv.view(seq, batch, 3, heads, hd).unbind(2))  # [B, L, heads, hd]: read in place
            if self.attention == "relative":
                ctx = relative_attention(q, k, v, self.position_bias, self.buckets)
            else:
                ctx = differential_attention(q, k, v.reshape(batch, seq, heads // 2, 2 * hd), self._lambda(), self.position_bias, self.buckets)
                ctx = self.head_norm(ctx) * (1.0 - self.lambda_init)
            ctx = ctx.transpose(0, 1).reshape(seq, batch, d)
        return _rows(ctx, attn.out_proj)

    def _feed_forward(self, y: torch.Tensor) -> torch.Tensor:
        hidden = _rows(y, self.linear1)
        hidden = self._act_dropout(hidden) if hidden.is_cuda else self.dropout(self.activation(hidden))
        return _rows(hidden, self.linear2)

    def _join(self, x: torch.Tensor, y: torch.Tensor, z: torch.Tensor, drop: nn.Dropout, i: int, pre: nn.LayerNorm) -> tuple[torch.Tensor, torch.Tensor]:
        """Residual stream and the next block's normalised input behind block ``i`` (input ``y``, output ``z``)."""
        post, gate, scale = getattr(self, f"post_norm{i}"), getattr(self, f"gate{i}"), getattr(self, f"residual_scale{i}")
        z = drop(z)
        if x.dtype != torch.float32 and z.dtype == torch.float32:
            x = x.float()
        return gated_norm_residual(x, z, scale, post.weight, post.bias, pre.weight, pre.bias, gate=_rows(y, gate).to(z.dtype), eps=post.eps)

    def step(self, x: torch.Tensor, y: torch.Tensor, pre_next: nn.LayerNorm) -> tuple[torch.Tensor, torch.Tensor]:
        """Sandwich form: residual stream ``x`` and its norm ``y`` in; the same behind this layer out (``pre_next``: whose norm)."""
        x, y = self._join(x, y, self._attend(y), self.dropout1, 1, self.norm2)
        return self._join(x, y, self._feed_forward(y), self.dropout2, 2, pre_next)

    def forward(self, src, src_mask=None, src_key_padding_mask=None, is_causal=False):  # noqa: ANN001
        if src_mask is not None or src_key_padding_mask is not None or is_causal:
            raise ValueError("BoardEncoderLayer takes no masks")
        if self.sandwich:
            raise ValueError("sandwich layers run inside BoardEncoder: a layer's last norm belongs to the next one")
        src, y = self._norm_fork(self.norm1, src)
        x = src + self.dropout1(self._attend(y))
        x, y = self._norm_fork(self.norm2, x)
        return x + self.dropout2(self._feed_forward(y))


class BoardEncoder(nn.Module):
    """A stack of :class:`BoardEncoderLayer` with a final norm (``layers`` and ``norm`` as in ``nn.TransformerEncoder``)."""

    def __init__(self, board: tuple[int, int], num_layers: int, attention: str, sandwich: bool, d_model: int, **kwargs) -> None:  # noqa: ANN003
        super().__init__()
        self.layers = nn.ModuleList(BoardEncoderLayer(board, attention, sandwich, i, d_model=d_model, **kwargs) for i in range(num_layers))
        self.norm = FastLayerNorm(d_model)
        self.sandwich = sandwich

    def forward(self, src: torch.Tensor) -> torch.Tensor:
        if not self.sandwich:
            for layer in self.layers:
                src = layer(src)
            return self.norm(src)
        y = self.layers[0].norm1(src)
        for i, layer in enumerate(self.layers):
            src, y = layer.step(src, y, self.layers[i + 1].norm1 if i + 1 < len(self.layers) else self.norm)
        return y
