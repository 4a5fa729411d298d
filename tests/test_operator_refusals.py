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


def test_embedding_refusals():
    from mega_trading_b200 import _lib
    from mega_trading_b200.kernels.embedding import scaled_embedding

    lib = _lib.load()
    f32 = _lib.MT_F32
    fwd, bwd = lib.mt_embedding_fwd, lib.mt_embedding_bwd
    assert fwd(FAKE, 1, -1, FAKE, f32, 10, 8, 1.0, FAKE, f32, FAKE, None) == 1
    assert fwd(FAKE, 1, 4, FAKE, f32, 0, 8, 1.0, FAKE, f32, FAKE, None) == 1
    assert fwd(FAKE, 1, 4, FAKE, 5, 10, 8, 1.0, FAKE, f32, FAKE, None) == 2
    assert fwd(FAKE, 1, 4, FAKE, f32, 10, 8, 1.0, FAKE, f32, None, None) == 1
    assert fwd(FAKE, 1, 2 ** 31, FAKE, f32, 10, 8, 1.0, FAKE, f32, FAKE, None) == 1
    assert fwd(None, 1, 0, None, f32, 10, 8, 1.0, None, f32, None, None) == 0
    need = lib.mt_embedding_bwd_workspace_bytes(5000, 300, 64)
    assert need >= 2 * 5000 * 8
    assert bwd(FAKE, 1, 5000, FAKE, f32, 300, 64, 1.0, -1, FAKE, f32, FAKE, need - 1, FAKE, None) == 7
    assert bwd(FAKE, 1, 5000, FAKE, f32, 300, 64, 1.0, -1, FAKE, f32, ODD, need, FAKE, None) == 7
    assert bwd(FAKE, 1, 5000, FAKE, f32, 300, 64, 1.0, 300, FAKE, f32, FAKE, need, FAKE, None) == 1
    assert bwd(FAKE, 1, 5000, FAKE, f32, 300, 64, 1.0, -1, None, f32, FAKE, need, FAKE, None) == 1
    ids, w = torch.zeros(3, dtype=torch.long), torch.zeros(4, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        scaled_embedding(ids, w)
    with pytest.raises(ValueError, match="ids must be"):
        scaled_embedding(ids.float(), w)
    with pytest.raises(ValueError, match="weight must have shape"):
        scaled_embedding(ids, w[0])
    with pytest.raises(ValueError, match="padding_idx"):
        scaled_embedding(ids, w, padding_idx=4)
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        scaled_embedding(ids, w, out_dtype=torch.float64)


def test_distillation_refusals():
    from mega_trading_b200 import _lib
    from mega_trading_b200.kernels.distillation import fused_linear_distillation

    lib = _lib.load()
    f32, bf16 = _lib.MT_F32, _lib.MT_BF16
    fwd, bwd = lib.mt_distill_fwd, lib.mt_distill_bwd

    def call(hidden=FAKE, dtype=bf16, ldt=f32, n=100, v=500, k=64, top=8, temp=1.0, ws=FAKE, nbytes=1 << 30,
             status=FAKE):
        return fwd(hidden, FAKE, dtype, FAKE, 1, -100, FAKE, ldt, n, v, k, top, temp, FAKE, FAKE, FAKE, FAKE, FAKE,
                   ws, nbytes, status, None)

    assert call(dtype=f32) == 2 and call(ldt=5) == 2
    assert call(top=0) == 1 and call(top=257) == 1 and call(v=0) == 1 and call(n=-1) == 1
    assert call(temp=0.0) == 1 and call(temp=-1.0) == 1 and call(temp=float("nan")) == 1
    assert call(temp=float("inf")) == 1
    assert call(k=12) == 3 and call(hidden=ODD) == 3
    assert call(ws=None) == 7 and call(ws=ODD) == 7 and call(nbytes=lib.mt_distill_workspace_bytes(100, 500) - 1) == 7
    assert call(status=None) == 1

    def back(n=100, top=8, ws=FAKE, nbytes=1 << 40, dhd=bf16, dh=FAKE, go=FAKE):
        return bwd(FAKE, FAKE, bf16, n, 500, 64, top, 1.0, FAKE, FAKE, FAKE, FAKE, go, dh, dhd, FAKE, bf16, ws, nbytes,
                   FAKE, None)

    assert back(top=300) == 1 and back(dhd=6) == 2 and back(dh=ODD) == 3 and back(go=None) == 1
    assert back(ws=None) == 7 and back(nbytes=lib.mt_distill_bwd_workspace_bytes(100, 500, 64) - 1) == 7
    # the backward's workspace is bounded whatever the batch
    assert lib.mt_distill_bwd_workspace_bytes(1 << 20, 21504, 768) < 800 << 20

    h, w = torch.randn(4, 8), torch.randn(11, 8)
    ids, lg = torch.zeros(4, 3, dtype=torch.long), torch.zeros(4, 3)
    with pytest.raises(RuntimeError, match="CUDA"):
        fused_linear_distillation(h, w, ids, lg)
    with pytest.raises(ValueError, match="hidden must have shape"):
        fused_linear_distillation(h[None], w, ids, lg)
    with pytest.raises(ValueError, match="weight must have shape"):
        fused_linear_distillation(h, w[:, :4], ids, lg)
    with pytest.raises(ValueError, match="one row per hidden row"):
        fused_linear_distillation(h, w, ids[:2], lg[:2])
    with pytest.raises(ValueError, match="shape of teacher_ids"):
        fused_linear_distillation(h, w, ids, lg[:, :2])
    with pytest.raises(ValueError, match="1 to 256"):
        fused_linear_distillation(h, w, ids[:, :0], lg[:, :0])
    with pytest.raises(ValueError, match="integer tensor"):
        fused_linear_distillation(h, w, ids.float(), lg)
    with pytest.raises(ValueError, match="temperature"):
        fused_linear_distillation(h, w, ids, lg, temperature=0.0)
    with pytest.raises(ValueError, match="multiple of 8"):
        fused_linear_distillation(h[:, :4], w[:, :4], ids, lg)
    with pytest.raises(ValueError, match="compute_weight"):
        fused_linear_distillation(h, w, ids, lg, compute_weight=w[:3])


def test_token_table_on_the_host_still_looks_up():
    from mega_trading_b200.model import ModelConfig, TradingModelB200

    m = TradingModelB200(ModelConfig(vocab_size=50, block_size=16, hidden_dim=32, layers=1, attention_heads=4,
                                     kv_heads=2, intermediate_dim=48))
    ids = torch.tensor([[1, 2, 3]])
    assert torch.equal(m.token_embedding(ids), m.token_embedding.weight[ids])


def test_distillation_workspace_holds_what_the_call_uses():
    """No room for partial sums of dW where one product writes dW itself (one chunk of rows, one split);
    room for them where chunks of rows add up."""
    from mega_trading_b200 import _lib

    size = _lib.load().mt_distill_bwd_workspace_bytes
    # dz, the chunk's hidden states and at most 64 splits of dh in fp32
    for n, v, k in ((256, 300_000, 1024), (8, 1_200_000, 1024), (200, 21_504, 256)):
        assert size(n, v, k) <= 2 * n * (v + 8) + 2 * n * k + 64 * 256 * k * 4 + 4 * 256
    assert size(20_000, 21_504, 768) >= 21_504 * 768 * 4
