"""The token table, the distillation loss and the 8-bit operators run together:
a frozen 8-bit teacher's top logits train a smaller student.

Bounds.  An 8-bit operand is off by at most half a step of max/127; for values
spread like a normal distribution (max about 4 standard deviations in a row of
several hundred) that is about 0.9 % of a row's norm, so a product of two such
operands is off by about 1.3 % of its norm.  A model of 2 layers has 8 products
in a chain of residual adds and one for the logits: 4 % if every error
reached the logits undamped; the test allows 10 %."""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

from oracle import ops as O

pytestmark = pytest.mark.gpu

TEACHER = dict(block_size=512, hidden_dim=1024, layers=2, attention_heads=16, kv_heads=4, intermediate_dim=2816)
STUDENT = dict(block_size=512, hidden_dim=256, layers=2, attention_heads=8, kv_heads=2, intermediate_dim=688)


def _model(dev, seed, **kw):
    from mega_trading_b200.model import ModelConfig, TradingModelB200

    torch.manual_seed(seed)
    return TradingModelB200(ModelConfig(**kw)).to(dev)


@pytest.mark.parametrize("kw,batch,seq", [(TEACHER, 2, 200), (STUDENT, 3, 77), (STUDENT, 1, 1)])
def test_int8_model_follows_the_bf16_model(cuda_device, kw, batch, seq):
    from mega_trading_b200 import _lib
    from mega_trading_b200.data import composite_tokens
    from mega_trading_b200.int8_model import Int8TradingModel

    m = _model(cuda_device, 0, **kw)
    q = Int8TradingModel(m)
    ids = composite_tokens(batch, seq, seed=3, device=cuda_device)
    with torch.no_grad():
        want = m(ids)
    got = q(ids)
    assert got.shape == want.shape == (batch, seq, 21504) and got.dtype == torch.float32
    err = float((got - want).norm() / want.norm())
    assert err <= 0.10, err
    top_ids, top = q.top_logits(ids, 16)
    assert top_ids.shape == top.shape == (batch, seq, 16)
    assert torch.equal(top, got.topk(16, dim=-1).values) and torch.equal(top, got.gather(-1, top_ids))
    with torch.no_grad():
        w_ids, w_top = m.top_logits(ids, 16)
    assert torch.equal(w_top.float(), want.gather(-1, w_ids))
    assert _lib.read_status(cuda_device) == 0


def test_distillation_step_gradients(cuda_device):
    """Gradients of the whole student (both ends of the tied table among them) against the same loss
    formed by torch from the student's logits."""
    from mega_trading_b200.data import composite_tokens
    from mega_trading_b200.int8_model import Int8TradingModel

    teacher = Int8TradingModel(_model(cuda_device, 1, **TEACHER))
    student = _model(cuda_device, 2, **STUDENT)
    ids = composite_tokens(2, 150, seed=4, device=cuda_device)
    t_ids, t_logits = teacher.top_logits(ids, 24)
    t_ids[0, 140:] = -100  # padding
    temp = 2.0
    loss = student(ids, teacher=(t_ids, t_logits), temperature=temp)
    loss.backward()
    ours = {k: p.grad.clone() for k, p in student.named_parameters()}
    student.zero_grad()
    # the plain form over materialised logits (bf16 products, fp32 loss)
    x = student.hidden_states(ids)
    logq = F.log_softmax(F.linear(x.float(), student.output.weight.bfloat16().float()) / temp, -1)
    hit = t_ids != -100
    p = torch.softmax(t_logits / temp, -1)
    rows = (p * (p.log() - logq.gather(-1, t_ids.clamp(min=0)))).sum(-1)
    keep = hit.all(-1)
    ref = temp * temp * rows[keep].mean()
    assert abs(float(loss.detach()) - float(ref.detach())) <= 1e-4 * abs(float(ref.detach()))
    ref.backward()
    for name, q in student.named_parameters():
        err = O.max_rel_error(ours[name], q.grad)
        # dz and each gradient of the chain are rounded to bf16 on both sides at different places
        assert err <= 5e-2, f"{name}: {err:.3e}"


def test_distill_step_updates_the_student(cuda_device):
    from mega_trading_b200.data import composite_tokens
    from mega_trading_b200.int8_model import Int8TradingModel
    from mega_trading_b200.model import ModelConfig
    from mega_trading_b200.train import Trainer

    teacher = Int8TradingModel(_model(cuda_device, 1, **TEACHER))
    tr = Trainer(ModelConfig(**STUDENT), micro_batch=2, device=cuda_device, lr=1e-3)
    ids = composite_tokens(4, 128, seed=5, device=cuda_device)
    t_ids, t_logits = teacher.top_logits(ids, 8)
    before = tr.model.token_embedding.weight.detach().clone()
    with torch.no_grad():
        want = tr.model.forward_with_distillation(ids, t_ids, t_logits, temperature=1.5)
    got = tr.distill_step(ids, t_ids, t_logits, temperature=1.5)
    # two micro-batches of equal size: their mean is the batch's, up to fp32 rounding
    assert abs(float(got) - float(want)) <= 1e-5 * abs(float(want))
    tr.check_status()
    after = tr.model.token_embedding.weight.detach()
    assert bool(after.isfinite().all()) and not torch.equal(after, before)
    # label and distillation steps mix
    assert torch.isfinite(tr.step(ids[:, :-1], ids[:, 1:]))
    with pytest.raises(ValueError, match="not both"):
        tr.model(ids, ids, teacher=(t_ids, t_logits))
    with pytest.raises(ValueError, match="matching input_ids"):
        tr.model(ids[:, :5], teacher=(t_ids, t_logits))


def test_int8_model_refuses_odd_widths(cuda_device):
    from mega_trading_b200.int8_model import Int8TradingModel

    m = _model(cuda_device, 0, block_size=32, hidden_dim=256, layers=1, attention_heads=8, kv_heads=2,
               intermediate_dim=344)
    with pytest.raises(ValueError, match="multiples of 16"):
        Int8TradingModel(m)
    q = Int8TradingModel(_model(cuda_device, 0, **STUDENT))
    with pytest.raises(ValueError, match="block_size"):
        q(torch.zeros(1, 513, dtype=torch.long, device=cuda_device))
    with pytest.raises(ValueError, match="shape"):
        q(torch.zeros(5, dtype=torch.long, device=cuda_device))


def test_distill_step_of_a_padded_batch_is_the_batch_mean(cuda_device):
    """Padding spread unevenly over the micro-batches: the loss is that of the whole batch in one piece."""
    from mega_trading_b200.data import composite_tokens
    from mega_trading_b200.int8_model import Int8TradingModel
    from mega_trading_b200.model import ModelConfig
    from mega_trading_b200.train import Trainer

    teacher = Int8TradingModel(_model(cuda_device, 1, **TEACHER))
    tr = Trainer(ModelConfig(**STUDENT), micro_batch=2, device=cuda_device, lr=1e-3)
    ids = composite_tokens(5, 96, seed=6, device=cuda_device)
    t_ids, t_logits = teacher.top_logits(ids, 8)
    t_ids[0, 10:], t_ids[1, 30:], t_ids[4] = -100, -100, -100
    t_logits[2, :40] = -float("inf")
    with torch.no_grad():
        want = tr.model.forward_with_distillation(ids, t_ids, t_logits, temperature=1.5)
    got = tr.distill_step(ids, t_ids, t_logits, temperature=1.5)
    # fp32 means of the same rows' losses
    assert abs(float(got) - float(want)) <= 1e-5 * abs(float(want))
    tr.check_status()
