"""8-bit inference of the order-flow model: a frozen teacher, or evaluation.

Every projection (q/k/v, o, gate/up, down and the tied output) runs as an int8
matrix product: activations are quantised per token, by the RMSNorm in front of
the projection where there is one and by a row quantisation otherwise (the
attention output, the gate's output); weights once, per output channel.
Residual stream (fp32), RoPE, attention and the SwiGLU gate are those of
:class:`~mega_trading_b200.model.TradingModelB200`.  The reference evaluates its
model in bf16 (duoan/mega-trading ``src/mega_trading/model.py:20-147``); there
is no counterpart of this path.
"""

from __future__ import annotations

import torch

from .kernels.embedding import scaled_embedding
from .kernels.fused_blocks import qkv_rope_attention, swiglu_packed
from .kernels.int8 import add_rms_norm_int8, int8_linear, quantize_rows_int8, rms_norm_int8
from .model import TradingModelB200, top_of_projection

__all__ = ["Int8TradingModel"]


class _Int8Block:
    def __init__(self, block) -> None:
        att, ffn = block.attention, block.feed_forward
        self.heads, self.kv_heads, self.head_dim = att.heads, att.kv_heads, att.head_dim
        self.cos, self.sin = att.cos, att.sin
        self.attention_norm, self.ffn_norm = _Norm(block.attention_norm), _Norm(block.ffn_norm)
        self.qkv = quantize_rows_int8(torch.cat([att.q_proj.weight, att.k_proj.weight, att.v_proj.weight]))
        self.o = quantize_rows_int8(att.o_proj.weight)
        self.gate_up = quantize_rows_int8(torch.cat([ffn.w1.weight, ffn.w3.weight]))
        self.down = quantize_rows_int8(ffn.w2.weight)

    def attention(self, q: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
        qkv = int8_linear(q, scale, *self.qkv)
        o = qkv_rope_attention(qkv, self.cos, self.sin, self.heads, self.kv_heads, self.head_dim)
        b, _, t, _ = o.shape  # stored [B, T, H, D]
        return int8_linear(*quantize_rows_int8(o.transpose(1, 2).reshape(b, t, -1)), *self.o)

    def feed_forward(self, q: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
        return int8_linear(*quantize_rows_int8(swiglu_packed(int8_linear(q, scale, *self.gate_up))), *self.down)


class _Norm:
    def __init__(self, norm) -> None:
        self.weight, self.eps = norm.weight.detach().clone(), norm.eps


class Int8TradingModel:
    """An 8-bit copy of a :class:`TradingModelB200` for inference (its weights are not shared).

    Calling it gives the logits ``[batch, time, vocab]`` (fp32, like the bf16 model);
    :meth:`top_logits` gives what a student's distillation loss takes.  hidden_dim and
    intermediate_dim must be multiples of 16."""

    @torch.no_grad()
    def __init__(self, model: TradingModelB200) -> None:
        self.cfg = model.cfg
        if self.cfg.hidden_dim % 16 or self.cfg.intermediate_dim % 16:
            raise ValueError("Int8TradingModel needs hidden_dim and intermediate_dim that are multiples of 16")
        self.table = model.token_embedding.weight.detach().clone()
        self.blocks = [_Int8Block(b) for b in model.blocks]
        self.norm = _Norm(model.norm)
        self.output = quantize_rows_int8(self.table)

    def _hidden(self, input_ids: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """The final norm's 8-bit rows and scales."""
        if input_ids.ndim != 2:
            raise ValueError("input_ids must have shape [batch, time]")
        if input_ids.shape[1] > self.cfg.block_size:
            raise ValueError(f"sequence length {input_ids.shape[1]} exceeds block_size {self.cfg.block_size}")
        h = scaled_embedding(input_ids, self.table)  # fp32 residual stream
        norms = [b.attention_norm for b in self.blocks[1:]] + [self.norm]
        first = self.blocks[0].attention_norm if self.blocks else self.norm
        q, s = rms_norm_int8(h, first.weight, eps=first.eps)
        for block, following in zip(self.blocks, norms):
            h, q, s = add_rms_norm_int8(block.attention(q, s), h, block.ffn_norm.weight, eps=block.ffn_norm.eps)
            h, q, s = add_rms_norm_int8(block.feed_forward(q, s), h, following.weight, eps=following.eps)
        return q, s

    @torch.no_grad()
    def __call__(self, input_ids: torch.Tensor) -> torch.Tensor:
        return int8_linear(*self._hidden(input_ids), *self.output, out_dtype=torch.float32)

    @torch.no_grad()
    def top_logits(self, input_ids: torch.Tensor, top: int) -> tuple[torch.Tensor, torch.Tensor]:
        """``(ids, logits)`` of each position's ``top`` largest logits (fp32)."""
        q, scale = self._hidden(input_ids)
        rows, scales = q.reshape(-1, q.shape[-1]), scale.reshape(-1)
        return top_of_projection(input_ids.shape, top, lambda lo, hi: int8_linear(
            rows[lo:hi], scales[lo:hi], *self.output, out_dtype=torch.float32))
