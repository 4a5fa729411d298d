"""What the operators refuse before any GPU is touched: the C entry points'
argument checks and the Python wrappers' errors on CPU tensors."""

from __future__ import annotations

import ctypes

import pytest
import torch

FAKE = ctypes.c_void_p(4096)
ODD = ctypes.c_void_p(4104)


def test_int8_entry_points_reject_invalid_arguments():
    from mega_trading_b200 import _lib

    lib = _lib.load()
    f32, f16, bf16 = _lib.MT_F32, _lib.MT_F16, _lib.MT_BF16
    norm = lib.mt_rms_norm_int8
    assert norm(FAKE, bf16, None, bf16, FAKE, f32, None, FAKE, FAKE, 4, 0, 1e-5, None) == 1       # no columns
    assert norm(FAKE, bf16, None, bf16, FAKE, f32, None, FAKE, FAKE, -1, 8, 1e-5, None) == 1      # negative rows
    assert norm(FAKE, bf16, None, bf16, FAKE, f32, None, FAKE, FAKE, 4, 32769, 1e-5, None) == 1   # too wide
    assert norm(FAKE, bf16, FAKE, f16, FAKE, f32, FAKE, FAKE, FAKE, 4, 8, 1e-5, None) == 2        # residual dtype
    assert norm(FAKE, bf16, None, bf16, FAKE, f16, None, FAKE, FAKE, 4, 8, 1e-5, None) == 2       # weight dtype
    assert norm(FAKE, 7, None, 7, FAKE, f32, None, FAKE, FAKE, 4, 8, 1e-5, None) == 2             # unknown dtype
    assert norm(FAKE, bf16, FAKE, bf16, FAKE, f32, None, FAKE, FAKE, 4, 8, 1e-5, None) == 1       # no new_residual
    assert norm(None, bf16, None, bf16, None, f32, None, None, None, 0, 8, 1e-5, None) == 0       # nothing to do
    rows = lib.mt_quantize_rows_int8
    assert rows(FAKE, 9, FAKE, FAKE, 4, 8, None) == 2
    assert rows(None, bf16, FAKE, FAKE, 4, 8, None) == 1
    assert rows(None, bf16, None, None, 0, 8, None) == 0
    gemm = lib.mt_int8_gemm
    assert gemm(FAKE, FAKE, FAKE, FAKE, FAKE, bf16, 4, 8, 24, FAKE, None) == 3       # K % 16
    assert gemm(FAKE, FAKE, FAKE, FAKE, FAKE, bf16, 4, 8, 131072, FAKE, None) == 1   # the int32 sum could overflow
    assert gemm(FAKE, FAKE, FAKE, FAKE, FAKE, 9, 4, 8, 16, FAKE, None) == 2
    assert gemm(ODD, FAKE, FAKE, FAKE, FAKE, bf16, 4, 8, 16, FAKE, None) == 3        # 16-byte operands
    assert gemm(FAKE, FAKE, FAKE, FAKE, FAKE, bf16, 4, 8, 16, None, None) == 1       # status word
    assert gemm(None, None, None, None, None, bf16, 0, 8, 16, None, None) == 0


def test_int8_wrappers_refuse_cpu_tensors():
    from mega_trading_b200.kernels import int8

    x = torch.randn(2, 16)
    q = torch.zeros(2, 16, dtype=torch.int8)
    with pytest.raises(RuntimeError, match="CUDA"):
        int8.rms_norm_int8(x, torch.ones(16), eps=1e-5)
    with pytest.raises(RuntimeError, match="CUDA"):
        int8.add_rms_norm_int8(x, x, torch.ones(16), eps=1e-5)
    with pytest.raises(RuntimeError, match="CUDA"):
        int8.quantize_rows_int8(x)
    with pytest.raises(RuntimeError, match="CUDA"):
        int8.int8_linear(q, torch.ones(2), q, torch.ones(2))
