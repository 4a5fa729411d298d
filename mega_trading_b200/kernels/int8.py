"""8-bit inference operators on sm_100a: quantising norms and the 8-bit product.

A projection run in 8 bits takes its input as int8 rows with one fp32 scale per
token and its weight as int8 rows with one fp32 scale per output channel:

* :func:`add_rms_norm_int8` / :func:`rms_norm_int8` -- the block's (residual add
  and) RMSNorm, whose output leaves as int8 plus scales;
* :func:`quantize_rows_int8` -- the same for inputs that no norm produces (the
  attention output, the SwiGLU gate's output) and for weights (a row of the
  weight is an output channel);
* :func:`int8_linear` -- the product on the tensor cores (``kind::i8``), exact
  in int32, scaled in fp32 and rounded once.

Inference only: none of them has a gradient, and a call that would need one is
refused.  The reference (duoan/mega-trading) runs every projection in bf16
(``src/mega_trading/model.py:218-256``); it has no counterpart of these.
"""

from __future__ import annotations

import torch

from .. import _lib

__all__ = ["rms_norm_int8", "add_rms_norm_int8", "quantize_rows_int8", "int8_linear"]

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)
MAX_DIM = 32768      # widest row of the quantising operators
MAX_K = 131056       # longest exact int32 dot product of 8-bit values (a multiple of 16)


def _check(op: str, first: torch.Tensor, *others: torch.Tensor) -> None:
    """One CUDA device for all tensors, and no gradient (of either mode) asked of a forward-only operator."""
    _lib.require_one_device(op, first, *others)
    if torch.is_grad_enabled() and (first.requires_grad or any(t.requires_grad for t in others)):
        raise RuntimeError(f"{op} has no gradient; call it under torch.no_grad()")
    _lib.refuse_tangent(op, first, *others)


def _rows(op: str, x: torch.Tensor) -> tuple[int, int]:
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"{op} needs rows of at least one element")
    if x.dtype not in _FLOATS:
        raise RuntimeError(f"{op} takes float32, bfloat16 or float16 tensors")
    dim = x.shape[-1]
    if dim > MAX_DIM:
        raise ValueError(f"{op} takes rows of at most {MAX_DIM} elements")
    return x.numel() // dim, dim


def _norm(op: str, hidden, residual, weight, eps: float):
    if residual is None:
        _check(op, hidden, weight)
    else:
        _check(op, hidden, weight, residual)
    rows, dim = _rows(op, hidden)
    act, wdt = hidden.dtype, weight.dtype
    if weight.dim() != 1 or weight.shape[0] != dim:
        raise ValueError("weight must have one entry per hidden feature")
    if wdt is not torch.float32 and wdt is not act:
        raise RuntimeError(f"{op} takes a float32 weight or one in the hidden dtype")
    x, w = hidden.contiguous(), weight.contiguous()
    code = rcode = _lib.dtype_code(act)
    new, r_ptr, new_ptr = None, None, None
    if residual is not None:
        if residual.shape != hidden.shape:
            raise ValueError("hidden and residual must have the same shape")
        if residual.dtype is not torch.float32 and residual.dtype is not act:
            raise RuntimeError(f"{op} takes a float32 residual or one in the hidden dtype")
        r = residual.contiguous()
        new = torch.empty_like(r)
        rcode, r_ptr, new_ptr = _lib.dtype_code(r.dtype), r.data_ptr(), new.data_ptr()
    q = torch.empty_like(x, dtype=torch.int8)
    scale = x.new_empty(x.shape[:-1], dtype=torch.float32)
    dev = x.device
    st = _lib.call(_lib.load().mt_rms_norm_int8, dev, x.data_ptr(), code, r_ptr, rcode, w.data_ptr(),
                   _lib.dtype_code(wdt), new_ptr, q.data_ptr(), scale.data_ptr(), rows, dim, eps, _lib.stream_ptr(dev))
    if st:
        _lib.check(st, op)
    return new, q, scale


def rms_norm_int8(hidden: torch.Tensor, weight: torch.Tensor, *, eps: float) -> tuple[torch.Tensor, torch.Tensor]:
    """``(q, scale)`` with ``q * scale[..., None]`` = RMSNorm of ``hidden`` to half an 8-bit step.

    ``q`` int8 has hidden's shape, ``scale`` fp32 its leading dimensions.  With ``v = hidden * weight``
    and ``a = max |v|`` of a row, ``q = rint(v * (127 / a))`` (fp32, ties to even) and
    ``scale = a / 127 * rsqrt(mean(hidden^2) + eps)``.  Rows with ``a < 2**-119`` give zeros; a row with
    an infinity or NaN gives a NaN scale."""
    _, q, scale = _norm("rms_norm_int8", hidden, None, weight, eps)
    return q, scale


def add_rms_norm_int8(hidden: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, *,
                      eps: float) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(new_residual, q, scale)``: :func:`rms_norm_int8` of ``new_residual = hidden + residual``.

    ``new_residual`` is rounded to the residual's dtype (the hidden dtype or fp32) and the norm reads
    the rounded values, as :func:`~mega_trading_b200.kernels.triton_ops.add_rms_norm` does."""
    return _norm("add_rms_norm_int8", hidden, residual, weight, eps)


def quantize_rows_int8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``(q, scale)`` with ``scale = max |row| / 127`` and ``q = rint(x * (127 / max |row|))``.

    Rows are the last dimension; zero and non-finite rows as in :func:`rms_norm_int8`."""
    op = "quantize_rows_int8"
    _check(op, x)
    rows, dim = _rows(op, x)
    xc = x.contiguous()
    q = torch.empty_like(xc, dtype=torch.int8)
    scale = xc.new_empty(xc.shape[:-1], dtype=torch.float32)
    dev = x.device
    st = _lib.call(_lib.load().mt_quantize_rows_int8, dev, xc.data_ptr(), _lib.dtype_code(x.dtype), q.data_ptr(),
                   scale.data_ptr(), rows, dim, _lib.stream_ptr(dev))
    if st:
        _lib.check(st, op)
    return q, scale


def int8_linear(x: torch.Tensor, x_scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, *,
                out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``(x @ weight.T) * x_scale[..., None] * weight_scale`` of int8 ``x`` [..., K] and ``weight`` [N, K].

    The dot products are exact (int32); the scales (fp32, one per row of ``x`` and of ``weight``) are
    applied in fp32 and the result is rounded once to ``out_dtype`` (bf16, fp16 or fp32).  ``K`` must be
    a multiple of 16 and at most 131,056."""
    op = "int8_linear"
    _check(op, x, x_scale, weight, weight_scale)
    if x.dtype is not torch.int8 or weight.dtype is not torch.int8:
        raise RuntimeError("int8_linear takes int8 x and weight")
    if x.dim() < 1 or weight.dim() != 2 or weight.shape[1] != x.shape[-1]:
        raise ValueError("weight must have shape [out, in] matching x's last dimension")
    if x_scale.dtype is not torch.float32 or weight_scale.dtype is not torch.float32:
        raise RuntimeError("int8_linear takes float32 scales")
    if x_scale.shape != x.shape[:-1]:
        raise ValueError("x_scale must have one entry per row of x")
    if weight_scale.shape != weight.shape[:1]:
        raise ValueError("weight_scale must have one entry per row of weight")
    if out_dtype not in _FLOATS:
        raise RuntimeError("int8_linear writes float32, bfloat16 or float16")
    n, k = weight.shape
    if k == 0 or k % 16 != 0 or k > MAX_K or n == 0:
        raise ValueError(f"int8_linear needs at least one output and an inner dimension that is a multiple of 16 "
                         f"and at most {MAX_K}")
    y = x.new_empty((*x.shape[:-1], n), dtype=out_dtype)
    xc, w, ws = _aligned(x), _aligned(weight), _aligned(weight_scale)
    xs = x_scale.contiguous()
    dev = x.device
    st = _lib.call(_lib.load().mt_int8_gemm, dev, xc.data_ptr(), xs.data_ptr(), w.data_ptr(), ws.data_ptr(),
                   y.data_ptr(), _lib.dtype_code(out_dtype), x.numel() // k, n, k, _lib.status_ptr(dev, op),
                   _lib.stream_ptr(dev))
    if st:
        _lib.check(st, op)
    return y


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """Contiguous and 16-byte aligned (a view at an odd offset is copied)."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()
