"""Distillation loss and its gradients against the definition in 64 bits.

Bounds (u = half a step of the 16-bit type, relative): a logit is an fp32 sum
of K products, off by at most (K / 16 + 4) 2^-23 |h| |w| (the tensor core adds
16 products a step, truncating); a probability q is off by a relative
e = 2 err(z) / T + 1e-4 (the exponential's 2^-22, and the sum of V terms kept
as running sums of at most a few hundred additions).  dz = q - p is rounded
once, u |dz|.  The products add (n / 16 + 4) 2^-23 of the sum of magnitudes and
the output its own half step.  The loss is off by T^2 (2 err(z) / T + 1e-4).
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
IGN = -100


def _definition(h, w, ids, logits, temp):
    """(loss, dz, rows) in 64 bits; h and w in double."""
    v = w.shape[0]
    hit = (ids != IGN) & (ids >= 0) & (ids < v)
    a = torch.where(hit, logits.double() / temp, -float("inf"))
    alive = (a > -float("inf")).any(1)
    a = torch.where(alive[:, None], a, torch.zeros_like(a))
    p = torch.softmax(a, 1) * hit * alive[:, None]
    logp = torch.where(p > 0, torch.log_softmax(a, 1), torch.zeros_like(a))
    idx = torch.where(hit, ids, torch.zeros_like(ids)).long()
    logq = torch.log_softmax((h @ w.t()) / temp, 1)
    rows = (p * (logp - logq.gather(1, idx))).sum(1)
    n = max(int(alive.sum()), 1)
    loss = temp * temp * torch.where(alive, rows, torch.zeros_like(rows)).sum() / n
    dense = torch.zeros_like(logq).scatter_add(1, idx, p)
    dz = torch.where(alive[:, None], logq.exp() - dense, torch.zeros_like(logq))
    q = torch.where(alive[:, None], logq.exp(), torch.zeros_like(logq))
    return loss, dz, q, n


def _run(dev, h, w, ids, logits, temp, dtype, gscale=1.0, compute_weight=None):
    from mega_trading_b200 import _lib
    from mega_trading_b200.kernels.distillation import fused_linear_distillation

    hd, wd = h.clone().requires_grad_(), w.clone().requires_grad_()
    loss = fused_linear_distillation(hd, wd, ids, logits, temperature=temp, ignore_index=IGN,
                                     compute_weight=compute_weight)
    assert loss.dtype == F32 and loss.shape == ()
    dh, dw = torch.autograd.grad(loss, (hd, wd), torch.tensor(gscale, device=dev))
    assert dh.dtype == h.dtype and dw.dtype == w.dtype
    assert _lib.read_status(dev) == 0
    return loss.detach(), dh, dw


def _check(h, w, ids, logits, temp, cdtype, gscale, loss, dh, dw):
    hc, wc = h.to(cdtype).double(), w.to(cdtype).double()
    ref, dz, q, n = _definition(hc, wc, ids, logits, temp)
    k, v = hc.shape[1], wc.shape[0]
    err_z = (k / 16 + 4) * 2.0 ** -23 * float(hc.norm(dim=1).max() * wc.norm(dim=1).max())
    e = 2 * err_z / temp + 1e-4
    assert abs(float(loss) - float(ref)) <= temp * temp * e, (float(loss), float(ref))
    u = torch.finfo(cdtype).eps / 2
    g = temp * gscale / n
    dz_err = u * dz.abs() + e * q + 2.0 ** -40

    def close(got, want, mag, mag_err, terms):
        uo = torch.finfo(got.dtype).eps / 2
        tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
        tol = abs(g) * (mag_err + (terms / 16 + 4) * 2.0 ** -23 * mag) * (1 + 2 * uo) + uo * want.abs() + tiny
        bad = (got.double() - want).abs() > tol * 1.0001
        assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[:4].tolist(),
                                     float(((got.double() - want).abs() / tol).max()))

    close(dh, g * (dz @ wc), dz.abs() @ wc.abs(), dz_err @ wc.abs(), v)
    close(dw, g * (dz.t() @ hc), dz.abs().t() @ hc.abs(), dz_err.t() @ hc.abs(), h.shape[0])


def _teacher(n, v, top, seed, dev, masked=0.0, empty=0.0):
    g = torch.Generator(device=dev).manual_seed(seed + 1000)
    ids = torch.stack([torch.randperm(v, device=dev, generator=g)[:top] for _ in range(min(n, 64))])
    ids = ids.repeat((n + ids.shape[0] - 1) // ids.shape[0], 1)[:n]
    ids = (ids + torch.randint(0, v, (n, 1), device=dev, generator=g)) % v
    logits = torch.randn(n, ids.shape[1], device=dev, generator=g) * 3
    if masked or empty:
        gone = torch.rand(ids.shape, device=dev, generator=g) < masked
        gone |= torch.rand(n, 1, device=dev, generator=g) < empty
        ids[gone] = IGN
        logits[gone] = float("nan")
    return ids, logits


@pytest.mark.parametrize("n,v,k,top,temp,dtype,masked,seed", [
    (1, 21504, 768, 8, 1.0, BF16, 0.0, 1),        # one token
    (1, 500, 1032, 1, 0.7, F16, 0.0, 13),
    (2, 1001, 64, 4, 1.0, BF16, 0.3, 14),
    (2, 21504, 768, 32, 2.0, F16, 0.2, 15),       # the most rows without tiles
    (2, 97, 2048, 9, 1.0, BF16, 0.2, 16),         # and the widest
    (2, 300, 2056, 5, 1.0, BF16, 0.0, 17),        # too wide for them
    (1, 70000, 1024, 3, 1.0, BF16, 0.0, 20),      # too large a weight
    (3, 2000, 256, 8, 1.0, BF16, 0.1, 18),        # the fewest rows in tiles
    (16, 21504, 768, 32, 2.0, F16, 0.2, 19),
    (300, 17, 64, 5, 2.0, BF16, 0.2, 2),          # a small vocabulary
    (77, 1000, 8, 1, 1.0, F16, 0.0, 3),           # the narrowest projection, one listed entry
    (130, 129, 104, 128, 0.5, BF16, 0.1, 4),
    (257, 1001, 256, 256, 1.5, F16, 0.3, 5),      # the longest lists, odd vocabulary
    (509, 21504, 256, 8, 1.0, BF16, 0.2, 6),
    (700, 21504, 768, 32, 2.0, BF16, 0.0, 7),
    (640, 21504, 1024, 64, 4.0, F16, 0.1, 8),
    (6500, 1500, 768, 16, 1.0, BF16, 0.1, 9),     # two chunks of rows
    (5000, 2000, 1032, 16, 2.0, F16, 0.1, 10),    # two chunks, five column tiles
    (20000, 300, 256, 33, 1.0, BF16, 0.1, 11),    # two chunks of a narrow student
    (64, 120000, 128, 20, 1.0, BF16, 0.0, 12),    # a large vocabulary
])
def test_distillation_matches_definition(cuda_device, n, v, k, top, temp, dtype, masked, seed):
    g = torch.Generator(device=cuda_device).manual_seed(seed)
    h = torch.randn(n, k, device=cuda_device, generator=g).to(dtype)
    w = (torch.randn(v, k, device=cuda_device, generator=g) * 0.05).to(dtype)
    ids, logits = _teacher(n, v, top, seed, cuda_device, masked, masked / 2)
    gscale = float(n)  # loss scaling: fp16 gradients of a mean stay in range
    out = _run(cuda_device, h, w, ids, logits, temp, dtype, gscale)
    _check(h, w, ids, logits, temp, dtype, gscale, *out)
    again = _run(cuda_device, h, w, ids, logits, temp, dtype, gscale)
    assert all(torch.equal(a, b) for a, b in zip(out, again))


def test_distillation_gradient_of_a_close_student(cuda_device):
    """A peaked student near its teacher: q and p nearly cancel where the mass is, and the
    gradient must be as exact as the difference, not as its parts."""
    g = torch.Generator(device=cuda_device).manual_seed(1)
    n, v, k = 200, 900, 64
    h = (torch.randn(n, k, device=cuda_device, generator=g)).to(BF16)
    w = (torch.randn(v, k, device=cuda_device, generator=g) * 0.8).to(BF16)
    z = h.double() @ w.double().t()
    logits, ids = z.topk(100, dim=1)
    logits = (logits + 0.01 * torch.randn(logits.shape, device=cuda_device, generator=g)).float()
    out = _run(cuda_device, h, w, ids, logits, 1.0, BF16)
    _check(h, w, ids, logits, 1.0, BF16, 1.0, *out)


def test_distillation_gradients_against_differences(cuda_device):
    g = torch.Generator(device=cuda_device).manual_seed(2)
    n, v, k, temp = 40, 60, 32, 1.7
    h = torch.randn(n, k, device=cuda_device, generator=g).to(BF16)
    w = (torch.randn(v, k, device=cuda_device, generator=g) * 0.3).to(BF16)
    ids, logits = _teacher(n, v, 7, 2, cuda_device, 0.2, 0.1)
    _, dh, dw = _run(cuda_device, h, w, ids, logits, temp, BF16)
    for leaf, grad in ((0, dh), (1, dw)):
        x = [h.double(), w.double()]
        d = torch.randn(x[leaf].shape, device=cuda_device, generator=g).double()
        step = 1e-4
        ends = []
        for sign in (1, -1):
            y = list(x)
            y[leaf] = y[leaf] + sign * step * d
            ends.append(float(_definition(y[0], y[1], ids, logits, temp)[0]))
        want = (ends[0] - ends[1]) / (2 * step)
        got = float((grad.double() * d).sum())
        # dz and the output each carry at most a relative 2^-8; the magnitudes bound the sum
        _, dz, _, rows = _definition(x[0], x[1], ids, logits, temp)
        m = (dz.abs() @ x[1].abs()) if leaf == 0 else (dz.abs().t() @ x[0].abs())
        assert abs(got - want) <= temp / rows * float((m * d.abs()).sum()) * (2.0 ** -7 + 1e-3) + 1e-6


def test_distillation_lists_in_any_order_with_repeats(cuda_device):
    g = torch.Generator(device=cuda_device).manual_seed(3)
    n, v, k, top = 90, 500, 64, 40
    h = torch.randn(n, k, device=cuda_device, generator=g).to(BF16)
    w = (torch.randn(v, k, device=cuda_device, generator=g) * 0.1).to(BF16)
    ids = torch.randint(0, 25, (n, top), device=cuda_device, generator=g)  # every id about twice
    ids[0] = 7                                                             # one id only
    logits = torch.randn(n, top, device=cuda_device, generator=g) * 2
    out = _run(cuda_device, h, w, ids, logits, 1.0, BF16)
    _check(h, w, ids, logits, 1.0, BF16, 1.0, *out)
    # int32 ids and 16-bit logits are the same lists
    l16 = logits.to(BF16)
    a = _run(cuda_device, h, w, ids.int(), l16, 1.0, BF16)
    b = _run(cuda_device, h, w, ids, l16.float(), 1.0, BF16)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    # strided lists
    wide_i, wide_l = ids.repeat_interleave(2, 1), logits.repeat_interleave(2, 1)
    c = _run(cuda_device, h, w, wide_i[:, ::2], wide_l[:, ::2], 1.0, BF16)
    assert all(torch.equal(x, y) for x, y in zip(out, c))


def test_distillation_of_one_entry_is_cross_entropy(cuda_device):
    from mega_trading_b200.kernels.fused_ce import fused_linear_cross_entropy

    g = torch.Generator(device=cuda_device).manual_seed(4)
    h = torch.randn(300, 128, device=cuda_device, generator=g).to(BF16)
    w = (torch.randn(2000, 128, device=cuda_device, generator=g) * 0.1).to(BF16)
    labels = torch.randint(0, 2000, (300,), device=cuda_device, generator=g)
    labels[::9] = IGN
    loss, dh, dw = _run(cuda_device, h, w, labels[:, None], torch.zeros(300, 1, device=cuda_device), 1.0, BF16)
    hd, wd = h.clone().requires_grad_(), w.clone().requires_grad_()
    ce = fused_linear_cross_entropy(hd, wd, labels, ignore_index=IGN)
    ce.backward()
    assert abs(float(loss) - float(ce.detach())) <= 1e-4
    for a, b in ((dh, hd.grad), (dw, wd.grad)):
        # both round dz once, at different scales: two half steps of it, and two of the output
        assert float((a.float() - b.float()).norm() / b.float().norm()) <= 4 * 2.0 ** -8


def test_distillation_masked_rows_and_lists(cuda_device):
    g = torch.Generator(device=cuda_device).manual_seed(5)
    n, v, k, top = 140, 300, 64, 6
    h = torch.randn(n, k, device=cuda_device, generator=g).to(BF16)
    w = (torch.randn(v, k, device=cuda_device, generator=g) * 0.1).to(BF16)
    ids, logits = _teacher(n, v, top, 5, cuda_device)
    logits[0] = -float("inf")                     # no mass at all
    logits[1, 1:] = -float("inf")                 # all mass on one entry
    logits[2] = torch.finfo(F32).min              # equal logits, the lowest finite value
    logits[3, 0] = torch.finfo(F32).max
    ids[4], logits[4] = IGN, float("inf")         # masked entries may hold anything
    ids[5, :5] = IGN
    logits[5, :5] = float("nan")
    out = _run(cuda_device, h, w, ids, logits, 2.0, BF16)
    assert all(bool(t.isfinite().all()) for t in out)
    _check(h, w, ids, logits, 2.0, BF16, 1.0, *out)
    assert bool((out[1][0] == 0).all()) and bool((out[1][4] == 0).all())
    # a row without an entry contributes nothing, whatever its logits would be
    big = h.clone()
    big[4] = 3e38
    other = _run(cuda_device, big, w, ids, logits, 2.0, BF16)
    assert torch.equal(other[0], out[0]) and torch.equal(other[1], out[1])
    # nothing listed anywhere
    loss, dh, dw = _run(cuda_device, h, w, torch.full_like(ids, IGN), logits, 2.0, BF16)
    assert float(loss) == 0.0 and bool((dh == 0).all()) and bool((dw == 0).all())


def test_distillation_nan_in_a_listed_logit_reaches_the_loss(cuda_device):
    h = torch.ones(3, 16, device=cuda_device, dtype=BF16)
    w = torch.ones(20, 16, device=cuda_device, dtype=BF16)
    ids = torch.tensor([[1, 2], [3, 4], [5, 6]], device=cuda_device)
    logits = torch.zeros(3, 2, device=cuda_device)
    logits[1, 0] = float("nan")
    loss, dh, _ = _run(cuda_device, h, w, ids, logits, 1.0, BF16)
    assert bool(loss.isnan()) and bool(dh[1].isnan().any()) and bool(dh[0].isfinite().all())


def test_distillation_out_of_range_ids_set_the_status_word(cuda_device):
    from mega_trading_b200 import _lib
    from mega_trading_b200.kernels.distillation import fused_linear_distillation

    g = torch.Generator(device=cuda_device).manual_seed(6)
    h = torch.randn(50, 64, device=cuda_device, generator=g).to(BF16)
    w = (torch.randn(40, 64, device=cuda_device, generator=g) * 0.1).to(BF16)
    ids, logits = _teacher(50, 40, 5, 6, cuda_device)
    clean = ids.clone()
    ids[3, 2], ids[9, 0], ids[10] = 40, -5, 2 ** 40
    clean[3, 2] = clean[9, 0] = IGN
    clean[10] = IGN
    assert _lib.read_status(cuda_device) == 0
    hd = h.clone().requires_grad_()
    loss = fused_linear_distillation(hd, w, ids, logits)
    loss.backward()
    code = _lib.read_status(cuda_device)
    assert code == (8 << 16) | 0xEEEE and "teacher id is out of range" in _lib.describe_status(code)
    want, dh, _ = _run(cuda_device, h, w, clean, logits, 1.0, BF16)
    assert torch.equal(loss.detach(), want) and torch.equal(hd.grad, dh)


def test_distillation_fp32_master_weight(cuda_device):
    """fp32 hidden and weight: the kernels read their bf16 roundings, gradients come back in fp32."""
    g = torch.Generator(device=cuda_device).manual_seed(7)
    h = torch.randn(150, 72, device=cuda_device, generator=g)
    w = torch.randn(700, 72, device=cuda_device, generator=g) * 0.1
    ids, logits = _teacher(150, 700, 9, 7, cuda_device)
    out = _run(cuda_device, h, w, ids, logits, 1.0, BF16)
    _check(h, w, ids, logits, 1.0, BF16, 1.0, *out)
    assert bool((out[2] != out[2].to(BF16).float()).any())
    copy = _run(cuda_device, h, w, ids, logits, 1.0, BF16, compute_weight=w.to(BF16))
    assert all(torch.equal(a, b) for a, b in zip(out, copy))
    # several chunks of rows into an fp32 gradient
    h2 = torch.randn(9000, 776, device=cuda_device, generator=g)
    w2 = torch.randn(600, 776, device=cuda_device, generator=g) * 0.05
    ids, logits = _teacher(9000, 600, 9, 8, cuda_device)
    out = _run(cuda_device, h2, w2, ids, logits, 1.0, BF16)
    _check(h2, w2, ids, logits, 1.0, BF16, 1.0, *out)


def test_distillation_partial_gradients_and_empty_batch(cuda_device):
    from mega_trading_b200.kernels.distillation import fused_linear_distillation

    g = torch.Generator(device=cuda_device).manual_seed(8)
    h = torch.randn(70, 64, device=cuda_device, generator=g).to(BF16)
    w = (torch.randn(90, 64, device=cuda_device, generator=g) * 0.1).to(BF16)
    ids, logits = _teacher(70, 90, 4, 8, cuda_device)
    _, dh, dw = _run(cuda_device, h, w, ids, logits, 1.0, BF16)
    hd = h.clone().requires_grad_()
    fused_linear_distillation(hd, w, ids, logits.requires_grad_()).backward()
    assert torch.equal(hd.grad, dh) and logits.grad is None
    wd = w.clone().requires_grad_()
    fused_linear_distillation(h, wd, ids, logits.detach()).backward()
    assert torch.equal(wd.grad, dw)
    with torch.no_grad():
        assert not fused_linear_distillation(h, w, ids, logits).requires_grad
    hd, wd = h[:0].clone().requires_grad_(), w.clone().requires_grad_()
    loss = fused_linear_distillation(hd, wd, ids[:0], logits[:0].detach())
    loss.backward()
    assert float(loss.detach()) == 0.0 and bool((wd.grad == 0).all()) and hd.grad.shape == (0, 64)


def test_distillation_in_a_graph_and_on_another_stream(cuda_device):
    from mega_trading_b200.kernels.distillation import fused_linear_distillation

    g = torch.Generator(device=cuda_device).manual_seed(9)
    h = torch.randn(900, 128, device=cuda_device, generator=g).to(BF16).requires_grad_()
    w = (torch.randn(1500, 128, device=cuda_device, generator=g) * 0.1).to(BF16).requires_grad_()
    ids, logits = _teacher(900, 1500, 12, 9, cuda_device)

    def step():
        loss = fused_linear_distillation(h, w, ids, logits, temperature=2.0)
        return loss.detach(), *torch.autograd.grad(loss, (h, w))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want))
    with torch.no_grad():
        h.copy_(torch.randn(900, 128, device=cuda_device, generator=g))
        logits.copy_(logits.flip(1))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_distillation_refuses_second_derivatives(cuda_device):
    from mega_trading_b200.kernels.distillation import fused_linear_distillation

    h = torch.randn(4, 16, device=cuda_device, dtype=BF16, requires_grad=True)
    w = torch.randn(20, 16, device=cuda_device, dtype=BF16)
    loss = fused_linear_distillation(h, w, torch.zeros(4, 1, dtype=torch.long, device=cuda_device),
                                     torch.zeros(4, 1, device=cuda_device))
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(loss, h, create_graph=True)


def test_distillation_vocabulary_of_one(cuda_device):
    """q is 1 everywhere: the loss and both gradients are zero."""
    g = torch.Generator(device=cuda_device).manual_seed(10)
    h = torch.randn(5, 8, device=cuda_device, generator=g).to(BF16)
    w = torch.randn(1, 8, device=cuda_device, generator=g).to(BF16)
    ids = torch.zeros(5, 3, dtype=torch.long, device=cuda_device)
    logits = torch.zeros(5, 3, device=cuda_device)
    # three equal entries of one id: p = 1 after merging, each entry counts its own log(1/3)
    loss, dh, dw = _run(cuda_device, h, w, ids, logits, 1.0, BF16)
    _check(h, w, ids, logits, 1.0, BF16, 1.0, loss, dh, dw)
    loss, dh, dw = _run(cuda_device, h, w, ids[:, :1], logits[:, :1], 1.0, BF16)
    assert abs(float(loss)) <= 1e-4 and float(dh.abs().max()) <= 1e-4 and float(dw.abs().max()) <= 1e-4


def test_distillation_nan_hidden_row_reaches_the_loss(cuda_device):
    g = torch.Generator(device=cuda_device).manual_seed(11)
    h = torch.randn(6, 64, device=cuda_device, generator=g).to(BF16)
    w = (torch.randn(90, 64, device=cuda_device, generator=g) * 0.1).to(BF16)
    ids, logits = _teacher(6, 90, 4, 11, cuda_device)
    bad = h.clone()
    bad[2, 5] = float("nan")
    loss, dh, _ = _run(cuda_device, bad, w, ids, logits, 1.0, BF16)
    assert bool(loss.isnan()) and bool(dh[2].isnan().all()) and bool(dh[[0, 1, 3, 4, 5]].isfinite().all())


def test_distillation_calls_on_two_streams_do_not_mix(cuda_device):
    g = torch.Generator(device=cuda_device).manual_seed(12)
    w = (torch.randn(3000, 256, device=cuda_device, generator=g) * 0.1).to(BF16)
    cases = []
    for i in range(4):
        h = torch.randn(700 + 300 * i, 256, device=cuda_device, generator=g).to(BF16)
        cases.append((h, *_teacher(h.shape[0], 3000, 10, 20 + i, cuda_device)))
    want = [_run(cuda_device, h, w, ids, lg, 1.5, BF16) for h, ids, lg in cases]
    torch.cuda.synchronize()
    from mega_trading_b200.kernels.distillation import fused_linear_distillation

    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for s, (h, ids, lg) in zip(streams, cases):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            hd, wd = h.clone().requires_grad_(), w.clone().requires_grad_()
            loss = fused_linear_distillation(hd, wd, ids, lg, temperature=1.5)
            got.append((loss.detach(), *torch.autograd.grad(loss, (hd, wd))))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("n", [1, 2])
def test_distillation_of_few_rows_keeps_dz_in_fp32(cuda_device, n):
    """No 16-bit rounding of dz: fp32 gradients within the sums' own rounding of the definition."""
    g = torch.Generator(device=cuda_device).manual_seed(n)
    h = torch.randn(n, 128, device=cuda_device, generator=g).to(BF16).float()
    w = (torch.randn(700, 128, device=cuda_device, generator=g) * 0.1).to(BF16).float()
    ids, logits = _teacher(n, 700, 6, n, cuda_device)
    _, dh, dw = _run(cuda_device, h, w, ids, logits, 1.5, BF16)
    _, dz, q, rows = _definition(h.double(), w.double(), ids, logits, 1.5)
    for got, want, mag in ((dh, dz @ w.double(), dz.abs() @ w.double().abs()),
                           (dw, dz.t() @ h.double(), dz.abs().t() @ h.double().abs())):
        # q carries the error of its logit and of the row's sum, 1e-5 relative and more than covered by 1e-4
        assert bool(((got.double() - 1.5 / rows * want).abs() <= 1.5 / rows * 1e-4 * (mag + 1e-6)).all())


@pytest.mark.parametrize("lo,n", [(0, 5), (64, 5), (384, 300), (0, 1)])
def test_distillation_nan_weight_rows_reach_the_loss(cuda_device, lo, n):
    """32 neighbouring NaN rows of the weight: every logit of the first step a thread looks at."""
    g = torch.Generator(device=cuda_device).manual_seed(13)
    h = torch.randn(n, 64, device=cuda_device, generator=g).to(BF16)
    w = (torch.randn(900, 64, device=cuda_device, generator=g) * 0.1).to(BF16)
    w[lo:lo + 32] = float("nan")
    ids = torch.tensor([[800, 700]], device=cuda_device).expand(n, 2)
    loss, _, _ = _run(cuda_device, h, w, ids, torch.zeros(n, 2, device=cuda_device), 1.0, BF16)
    assert bool(loss.isnan())


def test_distillation_entries_of_no_probability_leave_the_loss(cuda_device):
    """Vocabulary entries whose logits are -inf, whole steps and pieces of them, are entries with q = 0."""
    g = torch.Generator(device=cuda_device).manual_seed(14)
    h = (torch.rand(5, 64, device=cuda_device, generator=g) + 0.5).to(BF16)
    w = (torch.randn(900, 64, device=cuda_device, generator=g) * 0.1).to(BF16)
    w[0:64] = w[300:600] = -float("inf")
    ids = torch.tensor([[800, 700]], device=cuda_device).expand(5, 2)
    logits = torch.zeros(5, 2, device=cuda_device)
    loss, _, _ = _run(cuda_device, h, w, ids, logits, 1.0, BF16)
    ref = _definition(h.double(), w.double(), ids, logits, 1.0)[0]
    # the module's bound; |h| |w| <= 12 for the finite rows
    assert abs(float(loss) - float(ref)) <= 2 * (64 / 16 + 4) * 2.0 ** -23 * 12 + 1e-4


@pytest.mark.parametrize("n,k,dtype,wdt", [
    (2, 64, BF16, BF16),       # without tiles
    (3, 64, BF16, BF16),
    (140, 2056, F16, F16),
    (6500, 768, BF16, BF16),   # two chunks of rows, the empty rows in both
    (6500, 768, BF16, F32),    # the same into an fp32 gradient
    (20000, 40, F16, F16),
])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_distillation_empty_rows_may_hold_anything(cuda_device, n, k, dtype, wdt, bad):
    """Rows without an entry, and with -inf for every listed logit, add to no gradient whatever
    their hidden states hold: the same bits as with zeros there."""
    g = torch.Generator(device=cuda_device).manual_seed(15)
    h = torch.randn(n, k, device=cuda_device, generator=g).to(dtype)
    w = (torch.randn(700, k, device=cuda_device, generator=g) * 0.1).to(wdt)
    ids, logits = _teacher(n, 700, 6, 15, cuda_device)
    ids[n // 2], logits[n - 1] = IGN, -float("inf")
    h[[n // 2, n - 1]] = 0
    want = _run(cuda_device, h, w, ids, logits, 2.0, dtype)
    h[[n // 2, n - 1]] = bad
    got = _run(cuda_device, h, w, ids, logits, 2.0, dtype)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_distillation_refuses_forward_mode_tangents(cuda_device):
    import torch.autograd.forward_ad as fw

    from mega_trading_b200.kernels.distillation import fused_linear_distillation

    g = torch.Generator(device=cuda_device).manual_seed(16)
    h = torch.randn(4, 16, device=cuda_device, generator=g)
    w = torch.randn(20, 16, device=cuda_device, generator=g)
    ids, logits = _teacher(4, 20, 2, 16, cuda_device)
    with fw.dual_level():
        for at in range(3):
            args = [h, w, logits]
            args[at] = fw.make_dual(args[at], torch.ones_like(args[at]))
            with pytest.raises(RuntimeError, match="forward mode"):  # NotImplementedError is one
                fused_linear_distillation(args[0], args[1], ids, args[2])
        hd = h.clone().requires_grad_()
        loss = fused_linear_distillation(hd, w, ids, logits)
        with pytest.raises(RuntimeError, match="no forward-mode gradient"):
            torch.autograd.grad(loss, hd, fw.make_dual(torch.ones_like(loss), torch.ones_like(loss)))


def test_distillation_of_repeated_ids_against_the_merged_list(cuda_device):
    """Each listing of an id is an entry of its own: the gradients are those of the merged list, the loss
    is lower by the entropy of the split."""
    g = torch.Generator(device=cuda_device).manual_seed(17)
    n, v, k, temp = 60, 300, 64, 1.5
    h = torch.randn(n, k, device=cuda_device, generator=g)
    w = torch.randn(v, k, device=cuda_device, generator=g) * 0.1
    ids = torch.randperm(v, device=cuda_device, generator=g)[:3].expand(n, 3)
    logits = torch.randn(n, 6, device=cuda_device, generator=g) * 2
    split = _run(cuda_device, h, w, ids.repeat(1, 2), logits, temp, BF16)
    merged = torch.logsumexp(logits.view(n, 2, 3).double() / temp, 1) * temp
    whole = _run(cuda_device, h, w, ids, merged.float(), temp, BF16)
    p, big = torch.softmax(logits.double() / temp, 1), torch.softmax(merged / temp, 1)
    gap = temp ** 2 * float((torch.special.xlogy(big, big).sum(1) - torch.special.xlogy(p, p).sum(1)).mean())
    assert gap > 0.1
    # the module's bound of a loss, twice (|z| errors below 1e-5 here)
    assert abs(float(whole[0]) - float(split[0]) - gap) <= 2 * temp ** 2 * 2e-4
    for a, b in zip(split[1:], whole[1:]):
        # fp32 outputs of dz rounded to bf16: a probability that lands on the other side of a rounding border
        # moves its entry by one step, 2^-8 of it
        assert float((a - b).abs().max()) <= 2.0 ** -7 * float(b.abs().max())
