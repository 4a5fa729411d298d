"""Distillation loss of the output projection against a teacher's top logits, on sm_100a.

Beside the fused linear + cross-entropy (``fused_ce.py``): the same projection
``hidden @ weight.T`` whose logits never reach HBM, trained against the few
largest logits of a teacher per row instead of one label.  With ``p`` the
softmax of a row's listed teacher logits and ``q`` the student's softmax over
the whole vocabulary, both at ``temperature``, the loss is
``temperature**2 * mean_rows sum_j p_j (log p_j - log q[id_j])`` over the listed
entries: ``KL(p || q)`` when a row's ids are distinct (the factor keeps gradients
comparable across temperatures).  The reference (duoan/mega-trading) has no
distillation.
"""

from __future__ import annotations

import math

import torch

from .. import _lib

__all__ = ["fused_linear_distillation"]

MAX_TOP = 256  # listed teacher entries per row
_COMPUTE = (torch.bfloat16, torch.float16)
_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


class _FusedLinearDistillation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, ids, logits, temperature, ignore_index, compute_weight):
        lib = _lib.load()
        op = "fused_linear_distillation"
        cdtype = hidden.dtype if hidden.dtype in _COMPUTE else torch.bfloat16
        h = _aligned(hidden, cdtype)
        w = _aligned(weight if compute_weight is None else compute_weight, cdtype)
        ids, logits = ids.contiguous(), logits.contiguous()
        n, k = h.shape
        v, top = w.shape[0], ids.shape[1]
        dev = h.device
        loss = h.new_empty((), dtype=torch.float32)
        # what the backward needs of the lists: ids, probabilities, logits [n, top] and the row statistics [n + 3]
        kept = h.new_empty((3 * n * top + n + 3,), dtype=torch.float32)
        list_ids = kept.data_ptr()
        probs, z, stats = (list_ids + 4 * n * top * i for i in (1, 2, 3))
        ws = h.new_empty((lib.mt_distill_workspace_bytes(n, v),), dtype=torch.uint8)
        st = _lib.call(
            lib.mt_distill_fwd, dev, h.data_ptr(), w.data_ptr(), _lib.dtype_code(cdtype), ids.data_ptr(),
            1 if ids.dtype is torch.int64 else 0, ignore_index, logits.data_ptr(), _lib.dtype_code(logits.dtype), n, v,
            k, top, temperature, loss.data_ptr(), list_ids, probs, z, stats, ws.data_ptr(), ws.numel(),
            _lib.status_ptr(dev, op), _lib.stream_ptr(dev),
        )
        if st:
            _lib.check(st, op + " forward")
        ctx.save_for_backward(h, w, kept)
        ctx.args = (temperature, top, hidden.dtype, weight.dtype)
        return loss

    @staticmethod
    def backward(ctx, grad_output):
        need_h, need_w = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        if not (need_h or need_w):
            return (None,) * 7
        lib = _lib.load()
        op = "fused_linear_distillation"
        _lib.refuse_second_derivative(op)
        _lib.refuse_tangent(op, grad_output)
        h, w, kept = ctx.saved_tensors
        temperature, top, h_dtype, w_dtype = ctx.args
        n, k = h.shape
        v = w.shape[0]
        dev = h.device
        dh = h.new_empty((n, k), dtype=h_dtype) if need_h else None
        dw = w.new_empty((v, k), dtype=w_dtype) if need_w else None
        go = grad_output if grad_output.dtype is torch.float32 else grad_output.float()
        list_ids = kept.data_ptr()
        probs, z, stats = (list_ids + 4 * n * top * i for i in (1, 2, 3))
        ws = h.new_empty((lib.mt_distill_bwd_workspace_bytes(n, v, k),), dtype=torch.uint8)
        st = _lib.call(
            lib.mt_distill_bwd, dev, h.data_ptr(), w.data_ptr(), _lib.dtype_code(h.dtype), n, v, k, top, temperature,
            list_ids, probs, z, stats, go.data_ptr(), None if dh is None else dh.data_ptr(), _lib.dtype_code(h_dtype),
            None if dw is None else dw.data_ptr(), _lib.dtype_code(w_dtype), ws.data_ptr(), ws.numel(),
            _lib.status_ptr(dev, op), _lib.stream_ptr(dev),
        )
        if st:
            _lib.check(st, op + " backward")
        return dh, dw, None, None, None, None, None


def _aligned(t: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """``t`` in ``dtype``, contiguous and 16-byte aligned (a view at an odd offset is copied)."""
    t = (t if t.dtype is dtype else t.to(dtype)).contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def fused_linear_distillation(hidden: torch.Tensor, weight: torch.Tensor, teacher_ids: torch.Tensor,
                              teacher_logits: torch.Tensor, *, temperature: float = 1.0, ignore_index: int = -100,
                              compute_weight: torch.Tensor | None = None) -> torch.Tensor:
    """``temperature**2 * mean_rows sum_j p_j (log p_j - log q[teacher_ids_j])`` (fp32 scalar) with
    ``p = softmax(teacher_logits / T)`` and ``q = softmax(hidden @ weight.T / T)``.

    ``hidden`` [rows, hidden_dim] and ``weight`` [vocab, hidden_dim]; ``teacher_ids`` (int32 / int64) and
    ``teacher_logits`` (fp32 / bf16 / fp16) [rows, top], ``top`` at most 256, in any order.  The teacher's
    distribution is normalised over a row's listed entries; entries whose id is ``ignore_index`` are left
    out (their logits may hold anything).  With distinct ids a row's sum is ``KL(p || q)``.  An id listed
    several times counts once per entry: the gradients are those of the KL divergence from the merged list,
    the loss is lower than it by the entropy of the split (which the student does not change) and may be
    negative.  Rows without an entry (padding) add neither loss nor gradient, whatever their hidden states
    hold.  A teacher id outside the vocabulary is left out and sets the device status word.  Gradients go to
    ``hidden`` and ``weight`` in their own dtypes, not to the teacher.  Products of 16-bit operands with fp32
    sums: in ``hidden``'s type when it is 16 bits wide, else bf16, to which the other operand is rounded; the
    backward rounds ``q - p`` to that type once (not for one or two rows).

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
