"""Trainer.distill_step on the CPU: the batch's mean does not depend on how its padded positions fall
into micro-batches, and two gloo ranks average their means.

The model is a stand-in (an embedding and a projection) whose loss is the distillation loss written
out in 64 bits, so sums in another order differ by 1e-12 at most; the micro-batch weights are fp32
quotients, off by 2^-24 each, which the comparisons allow eight times over."""

from __future__ import annotations

import os
import socket

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

VOCAB, TOP = 23, 4
TOL = 8 * 2.0 ** -24


class _Student(torch.nn.Module):
    def __init__(self):
        super().__init__()
        g = torch.Generator().manual_seed(3)
        self.w = torch.nn.Parameter(torch.randn(VOCAB, 6, generator=g).double())

    def forward(self, ids, *, teacher, temperature):
        t_ids, t_logits = (t.flatten(0, 1) for t in teacher)
        logq = torch.log_softmax(self.w[ids].flatten(0, 1) @ self.w.t() / temperature, -1)
        hit = t_ids != -100
        a = torch.where(hit, t_logits.double() / temperature, -float("inf"))
        alive = (a > -float("inf")).any(1)
        a = torch.where(alive[:, None], a, torch.zeros_like(a))
        p = torch.softmax(a, 1) * (hit & alive[:, None])
        logp = torch.where(p > 0, torch.log_softmax(a, 1), torch.zeros_like(a))
        rows = (p * (logp - logq.gather(1, t_ids.clamp(min=0)))).sum(1)
        return temperature ** 2 * rows.sum() / alive.sum().clamp(min=1)


def _batch(seqs=5, time=7):
    g = torch.Generator().manual_seed(4)
    ids = torch.randint(0, VOCAB, (seqs, time), generator=g)
    t_ids = torch.randint(0, VOCAB, (seqs, time, TOP), generator=g)
    t_logits = torch.randn(seqs, time, TOP, generator=g)
    t_ids[0, 2:] = -100                      # a short sequence
    t_ids[2] = -100                          # nothing but padding
    t_ids[3, 1, 1:] = -100                   # one entry left
    t_logits[1, 3] = -float("inf")           # entries without weight
    t_logits[t_ids == -100] = float("nan")   # masked entries may hold anything
    return ids, t_ids, t_logits


def _step(ids, t_ids, t_logits, micro):
    """(loss, gradient) of one step."""
    from mega_trading_b200.train import Trainer

    tr = Trainer(None, micro_batch=micro, device=torch.device("cpu"), model=_Student())
    seen = []
    tr.opt.step = lambda: seen.append(tr.model.w.grad.clone() if tr.world == 1 else tr.engine.module.w.grad.clone())
    loss = tr.distill_step(ids, t_ids, t_logits, temperature=1.5)
    return loss.double(), seen[0]


@pytest.mark.parametrize("micro", [1, 2, 3, 4])
def test_distill_step_does_not_depend_on_the_micro_batch(micro):
    ids, t_ids, t_logits = _batch()
    student = _Student()
    want = student(ids, teacher=(t_ids, t_logits), temperature=1.5)
    want.backward()
    loss, grad = _step(ids, t_ids, t_logits, micro)
    assert abs(float(loss) - float(want.detach())) <= TOL * float(want.detach())
    assert bool(((grad - student.w.grad).abs() <= TOL * student.w.grad.abs().max()).all())


def test_distill_step_without_any_entry():
    ids, t_ids, t_logits = _batch()
    loss, grad = _step(ids, torch.full_like(t_ids, -100), t_logits, 2)
    assert float(loss) == 0.0 and bool((grad == 0).all())


def _worker(rank, world, port, outdir):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE=str(world),
                      LOCAL_RANK=str(rank))
    from mega_trading_b200.train import init_distributed

    init_distributed("gloo", timeout_s=60)
    part = [t[rank * 2:rank * 2 + 2] for t in _batch(4)]
    torch.save(_step(*part, 1), os.path.join(outdir, f"rank{rank}.pt"))
    dist.barrier()
    dist.destroy_process_group()


def test_two_ranks_average_their_means(tmp_path):
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    procs = [ctx.Process(target=_worker, args=(r, 2, port, str(tmp_path))) for r in range(2)]
    for p in procs:
        p.start()
    for p in procs:
        p.join(timeout=240)
        assert p.exitcode == 0
    got = [torch.load(tmp_path / f"rank{r}.pt") for r in range(2)]
    want = [_step(*(t[r * 2:r * 2 + 2] for t in _batch(4)), 2) for r in range(2)]
    mean = (want[0][1] + want[1][1]) / 2
    for r in range(2):
        assert abs(float(got[r][0]) - float(want[r][0])) <= TOL * float(want[r][0])
        assert bool(((got[r][1] - mean).abs() <= TOL * mean.abs().max()).all())
