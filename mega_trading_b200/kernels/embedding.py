"""Token embedding with a scale on sm_100a, and its gradient by sorted tokens.

Reference: ``nn.Embedding`` of the model (duoan/mega-trading
``src/mega_trading/model.py:20-147``).  The lookup, the scale (models that
multiply their embeddings by ``sqrt(dim)``) and the rounding to the output
dtype are one pass.  The gradient sorts the token positions by id and sums the
neighbouring rows in fp32: it is dense, written completely, rounded once to the
weight's dtype, and the same bits every time (torch's own gradient adds with
atomics).
"""

from __future__ import annotations

import torch

from .. import _lib

__all__ = ["scaled_embedding"]

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


def _lookup(weight, ids, scale, out_dtype):
    """Contiguous ids and the scaled rows."""
    w, ids = weight.contiguous(), ids.contiguous()
    vocab, dim = w.shape
    dev = w.device
    out = w.new_empty((*ids.shape, dim), dtype=out_dtype)
    st = _lib.call(
        _lib.load().mt_embedding_fwd, dev, ids.data_ptr(), 1 if ids.dtype is torch.int64 else 0, ids.numel(),
        w.data_ptr(), _lib.dtype_code(w.dtype), vocab, dim, scale, out.data_ptr(), _lib.dtype_code(out_dtype),
        _lib.status_ptr(dev, "scaled_embedding"), _lib.stream_ptr(dev),
    )
    if st:
        _lib.check(st, "scaled_embedding forward")
    return ids, out


class _ScaledEmbedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, ids, scale, padding_idx, out_dtype):
        ids, out = _lookup(weight, ids, scale, out_dtype)
        ctx.save_for_backward(ids)
        ctx.save_for_forward(ids)
        ctx.args, ctx.out_dtype = (scale, padding_idx, *weight.shape, weight.dtype), out_dtype
        return out

    @staticmethod
    def jvp(ctx, weight_tangent, *_):
        (ids,) = ctx.saved_tensors
        return scaled_embedding(ids, weight_tangent, scale=ctx.args[0], out_dtype=ctx.out_dtype)

    @staticmethod
    def backward(ctx, grad_output):
        (ids,) = ctx.saved_tensors
        if torch.is_grad_enabled() and grad_output.requires_grad or _lib.has_tangent(grad_output):
            return _EmbeddingGradient.apply(grad_output, ids, ctx.args), None, None, None, None
        return _gradient(grad_output, ids, *ctx.args), None, None, None, None


def _gradient(grad_output, ids, scale, padding_idx, vocab, dim, dtype):
    """The table's dense gradient in ``dtype``."""
    op = "scaled_embedding"
    lib = _lib.load()
    g = grad_output.contiguous()
    dev = g.device
    n = ids.numel()
    dw = g.new_empty((vocab, dim), dtype=dtype)
    ws_bytes = lib.mt_embedding_bwd_workspace_bytes(n, vocab, dim)
    ws = g.new_empty((ws_bytes,), dtype=torch.uint8) if ws_bytes else None
    st = _lib.call(
        lib.mt_embedding_bwd, dev, ids.data_ptr(), 1 if ids.dtype is torch.int64 else 0, n, g.data_ptr(),
        _lib.dtype_code(g.dtype), vocab, dim, scale, padding_idx, dw.data_ptr(), _lib.dtype_code(dtype),
        ws.data_ptr() if ws_bytes else None, ws_bytes, _lib.status_ptr(dev, op), _lib.stream_ptr(dev),
    )
    if st:
        _lib.check(st, op + " backward")
    return dw


class _EmbeddingGradient(torch.autograd.Function):
    """The gradient as a (linear) function of the output's gradient, for ``create_graph=True`` and
    forward-mode tangents: its own gradient is the lookup again, with the padded places left out."""

    @staticmethod
    def forward(ctx, grad_output, ids, args):
        ctx.save_for_backward(ids)
        ctx.save_for_forward(ids)
        ctx.args, ctx.dtype = args, grad_output.dtype
        return _gradient(grad_output, ids, *args)

    @staticmethod
    def jvp(ctx, grad_tangent, *_):
        return _gradient(grad_tangent, ctx.saved_tensors[0], *ctx.args)

    @staticmethod
    def backward(ctx, grad_table):
        (ids,) = ctx.saved_tensors
        scale, padding_idx = ctx.args[:2]
        out = scaled_embedding(ids, grad_table, scale=scale, out_dtype=ctx.dtype)
        if padding_idx >= 0:
            out = out.masked_fill((ids == padding_idx).unsqueeze(-1), 0.0)  # whatever the padding row holds
        return out, None, None


def scaled_embedding(ids: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0, padding_idx: int | None = None,
                     out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``scale * weight[ids]`` in ``out_dtype`` (the weight's by default), differentiable in ``weight``
    (any order, forward mode too).

    ``ids``: int32 or int64 of any shape; ``weight``: [vocab, dim] fp32, bf16 or fp16; the result has
    shape ``[*ids.shape, dim]``.  Places holding ``padding_idx`` (which may count from the end) look up
    their row but add to no gradient.  An id outside ``[0, vocab)`` gives a row of zeros, adds to no
    gradient and sets the device status word (:func:`mega_trading_b200._lib.check_status`)."""
    op = "scaled_embedding"
    if weight.dim() != 2 or weight.shape[0] == 0 or weight.shape[1] == 0:
        raise ValueError("weight must have shape [vocab, dim] with at least one row and column")
    if ids.dtype not in (torch.int32, torch.int64):
        raise ValueError("ids must be an int32 or int64 tensor")
    out_dtype = out_dtype or weight.dtype
    if weight.dtype not in _FLOATS or out_dtype not in _FLOATS:
        raise RuntimeError(f"{op} takes and writes float32, bfloat16 or float16")
    pad = -1
    if padding_idx is not None:
        if not -weight.shape[0] <= padding_idx < weight.shape[0]:
            raise ValueError("padding_idx must be within the vocabulary")
        pad = int(padding_idx) % weight.shape[0]
    _lib.require_one_device(op, weight, ids)
    if not (weight.requires_grad and torch.is_grad_enabled() or _lib.has_tangent(weight)):
        return _lookup(weight, ids, float(scale), out_dtype)[1]
    return _ScaledEmbedding.apply(weight, ids, float(scale), pad, out_dtype)
