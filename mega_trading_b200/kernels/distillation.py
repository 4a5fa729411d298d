"""Distillation loss of the output projection against a teacher's top logits, on sm_100a.

Beside the fused linear + cross-entropy (``fused_ce.py``): the same projection
``hidden @ weight.T`` whose logits never reach HBM, trained against the few
largest logits of a teacher per row instead of one label.  With ``p`` the
softmax of a row's listed teacher logits and ``q`` the student's softmax over
the whole vocabulary, both at ``temperature``, the loss is
``temperature**2 * mean_rows KL(p || q)`` (the factor keeps gradients comparable
across temperatures).  The reference (duoan/mega-trading) has no distillation.
"""

from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable

from .. import _lib

__all__ = ["fused_linear_distillation"]

MAX_TOP = 256  # listed teacher entries per row
_COMPUTE = (torch.bfloat16, torch.float16)
_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


class _FusedLinearDistillation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, ids, logits, temperature, ignore_index, compute_weight):
        lib = _lib.load()
        cdtype = hidden.dtype if hidden.dtype in _COMPUTE else torch.bfloat16
        h = _aligned(hidden.detach().to(cdtype))
        w = _aligned((weight if compute_weight is None else compute_weight).detach().to(cdtype))
        ids, logits = ids.contiguous(), logits.detach().contiguous()
        n, k = h.shape
        v, top = w.shape[0], ids.shape[1]
        dev = h.device
        loss = torch.empty((), device=dev, dtype=torch.float32)
        list_ids = torch.empty((n, top), device=dev, dtype=torch.int32)
        probs, z = torch.empty((2, n, top), device=dev, dtype=torch.float32).unbind(0)
        stats = torch.empty((n + 3,), device=dev, dtype=torch.float32)
        ws = torch.empty((int(lib.mt_distill_workspace_bytes(n, v)),), device=dev, dtype=torch.uint8)
        with _lib.on_device(dev):
            st = lib.mt_distill_fwd(
                h.data_ptr(), w.data_ptr(), _lib.dtype_code(cdtype), ids.data_ptr(),
                1 if ids.dtype == torch.int64 else 0, ignore_index, logits.data_ptr(), _lib.dtype_code(logits.dtype),
                n, v, k, top, temperature, loss.data_ptr(), list_ids.data_ptr(), probs.data_ptr(), z.data_ptr(),
                stats.data_ptr(), ws.data_ptr(), ws.numel(), _lib.status_ptr(dev, "fused_linear_distillation"),
                _lib.stream_ptr(dev),
            )
        _lib.check(st, "fused_linear_distillation forward")
        ctx.save_for_backward(h, w, list_ids, probs, z, stats)
        ctx.temperature = temperature
        ctx.dtypes = (hidden.dtype, weight.dtype)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        need_h, need_w = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        if not (need_h or need_w):
            return (None,) * 7
        lib = _lib.load()
        h, w, list_ids, probs, z, stats = ctx.saved_tensors
        n, k = h.shape
        v, top = w.shape[0], list_ids.shape[1]
        dev = h.device
        dh = torch.empty((n, k), device=dev, dtype=ctx.dtypes[0]) if need_h else None
        dw = torch.empty((v, k), device=dev, dtype=ctx.dtypes[1]) if need_w else None
        go = grad_output.detach().to(device=dev, dtype=torch.float32).reshape(1).contiguous()
        ws = torch.empty((int(lib.mt_distill_bwd_workspace_bytes(n, v, k)),), device=dev, dtype=torch.uint8)
        with _lib.on_device(dev):
            st = lib.mt_distill_bwd(
                h.data_ptr(), w.data_ptr(), _lib.dtype_code(h.dtype), n, v, k, top, ctx.temperature,
                list_ids.data_ptr(), probs.data_ptr(), z.data_ptr(), stats.data_ptr(), go.data_ptr(),
                dh.data_ptr() if dh is not None else None, _lib.dtype_code(ctx.dtypes[0]),
                dw.data_ptr() if dw is not None else None, _lib.dtype_code(ctx.dtypes[1]), ws.data_ptr(), ws.numel(),
                _lib.status_ptr(dev, "fused_linear_distillation"), _lib.stream_ptr(dev),
            )
        _lib.check(st, "fused_linear_distillation backward")
        return dh, dw, None, None, None, None, None


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """Contiguous and 16-byte aligned (a view at an odd offset is copied)."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def fused_linear_distillation(hidden: torch.Tensor, weight: torch.Tensor, teacher_ids: torch.Tensor,
                              teacher_logits: torch.Tensor, *, temperature: float = 1.0, ignore_index: int = -100,
                              compute_weight: torch.Tensor | None = None) -> torch.Tensor:
    """``temperature**2 * mean_rows KL(softmax(teacher_logits / T) || softmax(hidden @ weight.T / T))`` (fp32 scalar).

    ``hidden`` [rows, hidden_dim] and ``weight`` [vocab, hidden_dim]; ``teacher_ids`` (int32 / int64) and
    ``teacher_logits`` (fp32 / bf16 / fp16) [rows, top], ``top`` at most 256, in any order.  The teacher's
    distribution is normalised over a row's listed entries; entries whose id is ``ignore_index`` are left
    out (their logits may hold anything), an id listed twice counts with the sum of its probabilities.  Rows
    without an entry (padding) add neither loss nor gradient.  A teacher id outside the vocabulary is left
    out and sets the device status word.  Gradients go to ``hidden`` and ``weight`` in their own dtypes, not
    to the teacher; 16-bit products with fp32 sums (an fp32 ``hidden`` or ``weight`` is rounded to bf16).

    ``compute_weight``: an optional 16-bit copy of ``weight`` that the kernels read instead of casting it,
    as in :func:`~mega_trading_b200.kernels.fused_ce.fused_linear_cross_entropy`."""
    op = "fused_linear_distillation"
    if hidden.ndim != 2:
        raise ValueError("hidden must have shape [rows, hidden_dim]")
    if weight.ndim != 2 or weight.shape[1] != hidden.shape[1] or weight.shape[0] == 0:
        raise ValueError("weight must have shape [vocab, hidden_dim] matching hidden's last dim")
    if teacher_ids.ndim != 2 or teacher_ids.shape[0] != hidden.shape[0]:
        raise ValueError("teacher_ids must have shape [rows, top] with one row per hidden row")
    if teacher_logits.shape != teacher_ids.shape:
        raise ValueError("teacher_logits must have the shape of teacher_ids")
    if not 1 <= teacher_ids.shape[1] <= MAX_TOP:
        raise ValueError(f"{op} takes 1 to {MAX_TOP} teacher entries per row")
    if teacher_ids.dtype not in (torch.int32, torch.int64):
        raise ValueError("teacher_ids must be an integer tensor")
    if teacher_logits.dtype not in _FLOATS or hidden.dtype not in _FLOATS or weight.dtype not in _FLOATS:
        raise RuntimeError(f"{op} takes float32, bfloat16 or float16 tensors")
    temperature = float(temperature)
    if not (temperature > 0.0 and math.isfinite(temperature)):
        raise ValueError("temperature must be positive and finite")
    if hidden.shape[1] == 0 or hidden.shape[1] % 8 != 0:
        raise ValueError("hidden_dim must be a multiple of 8")
    if compute_weight is not None and compute_weight.shape != weight.shape:
        raise ValueError("compute_weight must have the weight's shape")
    _lib.require_one_device(op, hidden, weight, teacher_ids, teacher_logits)
    if compute_weight is not None:
        _lib.require_one_device(op, hidden, compute_weight)
    return _FusedLinearDistillation.apply(hidden, weight, teacher_ids, teacher_logits, temperature,
                                          int(ignore_index), compute_weight)
