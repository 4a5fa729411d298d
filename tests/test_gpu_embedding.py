"""Token embedding and its gradient against the definition in 64 bits.

Forward: one fp32 product and one rounding (half a step of the output type).
Gradient: fp32 sums.  A run of up to 64 rows is added in sequence and the
partial sums of a longer run again in sequence, so with c tokens on a row the
sum of its terms carries at most (min(c, 64) + c / 32 + 10) roundings of 2^-24
of the sum of magnitudes; the scale adds one and the output type half a step.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _ids(n, vocab, kind, g):
    if kind == "same":
        return torch.full((n,), vocab // 2, dtype=torch.long)
    if kind == "skewed":
        return (torch.rand(n, generator=g).pow(4) * vocab).long().clamp_(max=vocab - 1)
    if kind == "ordered":
        return torch.arange(n) % vocab
    return torch.randint(0, vocab, (n,), generator=g)


def _check_grad(dw, ids, grad, vocab, scale, pad):
    """dw against the 64-bit sums, with the bound of the module docstring."""
    g = grad.double()
    keep = torch.ones_like(ids, dtype=torch.bool) if pad is None else ids != pad
    keep &= (ids >= 0) & (ids < vocab)
    g = g * keep.unsqueeze(1)
    idx = ids.clamp(0, vocab - 1)
    zero = torch.zeros(vocab, g.shape[1], device=g.device, dtype=torch.float64)
    ref = zero.index_add(0, idx, g) * scale
    mag = zero.index_add(0, idx, g.abs()) * abs(scale)
    c = torch.bincount(idx[keep], minlength=vocab).double().unsqueeze(1)
    half = torch.finfo(dw.dtype).eps / 2
    tol = (c.clamp(max=64) + c / 32 + 11) * 2.0 ** -24 * mag + half * ref.abs() \
        + torch.finfo(dw.dtype).smallest_normal * torch.finfo(dw.dtype).eps
    bad = (dw.double() - ref).abs() > tol * 1.0001
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[:4].tolist())
    assert bool((dw[c[:, 0] == 0] == 0).all())


@pytest.mark.parametrize("n,vocab,dim,kind,wt,ot,scale,pad,seed", [
    (1, 21504, 768, "uniform", F32, F32, 1.0, None, 1),
    (16, 21504, 768, "uniform", F32, BF16, 27.7, None, 2),
    (256, 21504, 768, "same", F32, F32, 2.0, None, 18),       # the most tokens that take one launch
    (200, 30, 509, "skewed", BF16, F32, 1.0, 4, 19),
    (255, 1001, 1032, "skewed", F16, F16, 1.0, 1000, 20),
    (257, 21504, 64, "uniform", F32, F32, 1.0, None, 21),
    (2048, 21504, 256, "skewed", F32, F32, 1.0, None, 22),    # the largest single-block sort
    (2049, 21504, 256, "skewed", F32, F32, 1.0, None, 23),    # the smallest tiled sort
    (4096, 21504, 256, "skewed", F32, F32, 1.0, None, 3),
    (4097, 21504, 256, "skewed", F32, F32, 1.0, None, 4),
    (20000, 21504, 768, "skewed", F32, F32, 1.0, 0, 5),
    (30011, 1000, 1000, "uniform", BF16, BF16, 31.6, 999, 6),
    (5000, 300, 509, "uniform", F16, F16, 0.5, None, 7),      # odd width: single-element accesses
    (5000, 300, 510, "skewed", F32, F16, 2.0, 17, 8),
    (70000, 70000, 16, "uniform", F32, F32, 1.0, None, 9),    # three radix passes
    (9000, 1, 40, "same", F32, F32, 1.0, None, 10),           # one row
    (9000, 2, 8, "uniform", BF16, F32, 1.0, 1, 11),
    (50000, 21504, 64, "same", F32, F32, 1.0, None, 12),      # one token takes the whole stream
    (3000, 255, 12, "same", F32, BF16, -1.5, None, 13),
    (21504, 21504, 32, "ordered", F32, F32, 1.0, None, 14),   # every id once
    (1100000, 21504, 8, "skewed", F32, F32, 1.0, 3, 15),      # tiles of several sub-tiles
    (33, 7, 1, "uniform", F16, F32, 1.0, None, 16),
    (40000, 5, 2050, "uniform", BF16, BF16, 1.0, None, 17),   # long runs, many slabs
])
def test_embedding_matches_definition(cuda_device, n, vocab, dim, kind, wt, ot, scale, pad, seed):
    from mega_trading_b200 import _lib
    from mega_trading_b200.kernels.embedding import scaled_embedding

    g = torch.Generator().manual_seed(seed)
    ids = _ids(n, vocab, kind, g).to(cuda_device)
    w = (torch.randn(vocab, dim, generator=g) * 0.5).to(cuda_device, wt).requires_grad_()
    grad = torch.randn(n, dim, generator=g).to(cuda_device, ot)
    y = scaled_embedding(ids, w, scale=scale, padding_idx=pad, out_dtype=ot)
    assert y.dtype == ot and y.shape == (n, dim)
    # one product in fp32, one rounding: torch's elementwise operations give the same bits
    assert torch.equal(y, (w.detach()[ids].float() * scale).to(ot))
    y.backward(grad)
    assert w.grad.dtype == wt
    _check_grad(w.grad, ids, grad, vocab, scale, pad)
    dw = w.grad.clone()
    w.grad = None
    scaled_embedding(ids, w, scale=scale, padding_idx=pad, out_dtype=ot).backward(grad)
    assert torch.equal(w.grad, dw)  # fixed order of the sums
    assert _lib.read_status(cuda_device) == 0


def test_embedding_gradient_against_differences(cuda_device):
    """The loss is linear in the table, so a finite difference along a direction is the
    gradient's inner product with it, up to rounding."""
    from mega_trading_b200.kernels.embedding import scaled_embedding

    g = torch.Generator(device=cuda_device).manual_seed(5)
    ids = torch.randint(0, 50, (700,), device=cuda_device, generator=g)
    w = torch.randn(50, 24, device=cuda_device, generator=g).requires_grad_()
    r = torch.randn(700, 24, device=cuda_device, generator=g)
    d = torch.randn(50, 24, device=cuda_device, generator=g)
    scaled_embedding(ids, w, scale=3.0).backward(r)
    with torch.no_grad():
        hi = (scaled_embedding(ids, w + d, scale=3.0).double() * r.double()).sum()
        lo = (scaled_embedding(ids, w - d, scale=3.0).double() * r.double()).sum()
    want = float((hi - lo) / 2)
    got = float((w.grad.double() * d.double()).sum())
    # 700 * 24 terms of magnitude ~3, each with relative rounding below 2^-22
    assert abs(got - want) <= 700 * 24 * 30 * 2.0 ** -22


def test_embedding_shapes_and_layouts(cuda_device):
    from mega_trading_b200.kernels.embedding import scaled_embedding

    g = torch.Generator(device=cuda_device).manual_seed(2)
    w = torch.randn(40, 64, device=cuda_device, generator=g)
    ids = torch.randint(0, 40, (3, 5, 7), device=cuda_device, generator=g)
    want = w[ids]
    assert torch.equal(scaled_embedding(ids, w), want)
    assert torch.equal(scaled_embedding(ids.int(), w), want)
    assert torch.equal(scaled_embedding(ids.transpose(0, 2), w), w[ids.transpose(0, 2)])
    assert torch.equal(scaled_embedding(ids[0, 0, 0], w), w[ids[0, 0, 0]])  # a single id without dimensions
    big = torch.randn(40, 131, device=cuda_device, generator=g)
    view = big[:, 3:67]
    assert torch.equal(scaled_embedding(ids, view), view[ids])
    off = torch.randn(40 * 64 + 1, device=cuda_device, generator=g)[1:].view(40, 64)  # off the 16-byte grid
    assert torch.equal(scaled_embedding(ids, off), off[ids])
    # gradients that arrive expanded (a sum) or transposed
    wl = w.clone().requires_grad_()
    scaled_embedding(ids, wl, padding_idx=-40).sum().backward()
    counts = torch.bincount(ids.flatten(), minlength=40).float()
    counts[0] = 0
    assert torch.equal(wl.grad, counts[:, None].expand(40, 64))
    wl.grad = None
    y = scaled_embedding(ids, wl)
    gr = torch.randn(64, 7, 5, 3, device=cuda_device, generator=g).permute(3, 2, 1, 0)
    y.backward(gr)
    _check_grad(wl.grad, ids.flatten(), gr.reshape(-1, 64), 40, 1.0, None)


def test_embedding_empty(cuda_device):
    from mega_trading_b200.kernels.embedding import scaled_embedding

    w = torch.randn(11, 8, device=cuda_device, requires_grad=True)
    y = scaled_embedding(torch.empty(0, 3, dtype=torch.long, device=cuda_device), w)
    assert y.shape == (0, 3, 8)
    y.sum().backward()
    assert bool((w.grad == 0).all())


def test_embedding_out_of_range_ids_set_the_status_word(cuda_device):
    from mega_trading_b200 import _lib
    from mega_trading_b200.kernels.embedding import scaled_embedding

    for n in (100, 6000):
        g = torch.Generator(device=cuda_device).manual_seed(n)
        ids = torch.randint(0, 30, (n,), device=cuda_device, generator=g)
        ids[3], ids[50], ids[99] = 30, -1, 2 ** 40
        w = torch.randn(30, 16, device=cuda_device, generator=g).requires_grad_()
        assert _lib.read_status(cuda_device) == 0
        y = scaled_embedding(ids, w)
        code = _lib.read_status(cuda_device)
        assert code == (7 << 16) | 0xEEEE and "token id is out of range" in _lib.describe_status(code)
        assert bool((y[[3, 50, 99]] == 0).all())
        grad = torch.randn(n, 16, device=cuda_device, generator=g)
        y.backward(grad)
        assert _lib.read_status(cuda_device) == (7 << 16) | 0xEEEE
        _check_grad(w.grad, ids, grad, 30, 1.0, None)
        with pytest.raises(_lib.B200KernelError, match="token id"):
            scaled_embedding(ids, w)
            _lib.check_status(cuda_device)


def test_embedding_infinities_stay_in_their_rows(cuda_device):
    from mega_trading_b200.kernels.embedding import scaled_embedding

    ids = torch.tensor([1, 2, 1, 3, 9], device=cuda_device)
    w = torch.zeros(10, 8, device=cuda_device, requires_grad=True)
    grad = torch.ones(5, 8, device=cuda_device)
    grad[1] = float("inf")
    grad[4] = float("nan")
    scaled_embedding(ids, w, padding_idx=9).backward(grad)
    assert bool((w.grad[1] == 2).all()) and bool(w.grad[2].isinf().all()) and bool((w.grad[3] == 1).all())
    assert bool((w.grad[9] == 0).all()) and bool((w.grad[0] == 0).all())  # a NaN at a padded place is not read


def test_embedding_in_a_graph_and_on_another_stream(cuda_device):
    from mega_trading_b200.kernels.embedding import scaled_embedding

    g = torch.Generator(device=cuda_device).manual_seed(4)
    ids = torch.randint(0, 500, (6000,), device=cuda_device, generator=g)
    w = torch.randn(500, 72, device=cuda_device, generator=g).requires_grad_()
    grad = torch.randn(6000, 72, device=cuda_device, generator=g)

    def step():
        y = scaled_embedding(ids, w, scale=2.0)
        return y.detach(), torch.autograd.grad(y, w, grad)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            y1, d1 = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y2, d2 = step()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y1, y2) and torch.equal(d1, d2)
    ids.copy_(torch.randint(0, 500, (6000,), device=cuda_device, generator=g))
    graph.replay()
    torch.cuda.synchronize()
    y3, d3 = step()
    assert torch.equal(y2, y3) and torch.equal(d2, d3) and not torch.equal(d2, d1)


def test_embedding_second_derivative(cuda_device):
    """The gradient is linear in the output's gradient; differentiating it gives the lookup back."""
    from mega_trading_b200.kernels.embedding import scaled_embedding

    gen = torch.Generator(device=cuda_device).manual_seed(1)
    ids = torch.tensor([1, 2, 1, 5, 9], device=cuda_device)
    w = torch.randn(10, 8, device=cuda_device, generator=gen, requires_grad=True)
    g = torch.randn(5, 8, device=cuda_device, generator=gen, requires_grad=True)
    u = torch.randn(10, 8, device=cuda_device, generator=gen, requires_grad=True)
    y = scaled_embedding(ids, w, scale=2.0, padding_idx=9)
    (dw,) = torch.autograd.grad(y, w, g, create_graph=True)
    dg, du = torch.autograd.grad((dw * u).sum(), (g, u), create_graph=True)
    want = 2.0 * u.detach()[ids]
    want[4] = 0
    assert torch.equal(dg.detach(), want) and torch.equal(du.detach(), dw.detach())
    (again,) = torch.autograd.grad((dg * g.detach()).sum(), u)
    assert torch.equal(again, dw.detach())
    # create_graph without a differentiable gradient is the plain gradient
    (plain,) = torch.autograd.grad(scaled_embedding(ids, w, scale=2.0, padding_idx=9), w, g.detach(), create_graph=True)
    assert torch.equal(plain, dw.detach())


@pytest.mark.parametrize("n", [90, 700])
def test_embedding_gradient_off_the_vector_grid(cuda_device, n):
    """A contiguous output gradient whose base is not 16-byte aligned."""
    from mega_trading_b200.kernels.embedding import scaled_embedding

    gen = torch.Generator(device=cuda_device).manual_seed(n)
    ids = torch.randint(0, 60, (n,), device=cuda_device, generator=gen)
    w = torch.randn(60, 64, device=cuda_device, generator=gen, requires_grad=True)
    g = torch.randn(n * 64 + 1, device=cuda_device, generator=gen)[1:].view(n, 64)
    (dw,) = torch.autograd.grad(scaled_embedding(ids, w), w, g)
    _check_grad(dw, ids, g, 60, 1.0, None)


def test_embedding_calls_on_two_streams_do_not_mix(cuda_device):
    from mega_trading_b200.kernels.embedding import scaled_embedding

    gen = torch.Generator(device=cuda_device).manual_seed(8)
    cases = [(torch.randint(0, 4000, (n,), device=cuda_device, generator=gen),
              torch.randn(4000, 96, device=cuda_device, generator=gen, requires_grad=True),
              torch.randn(n, 96, device=cuda_device, generator=gen)) for n in (100, 1500, 9000, 80000)]
    want = [torch.autograd.grad(scaled_embedding(i, w), w, g)[0] for i, w, g in cases]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in cases], []
    for s, (i, w, g) in zip(streams, cases):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            leaf = w.detach().requires_grad_()
            got.append(torch.autograd.grad(scaled_embedding(i, leaf), leaf, g)[0])
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("n,dim,ot,share", [
    (9000, 1024, F32, 0.7),    # four rows to a stage of the gather ring: most stages hold no row
    (30000, 96, BF16, 0.5),    # 32 rows to a stage
    (3000, 2048, BF16, 1.0),   # no row anywhere
])
def test_embedding_gradient_with_ranges_of_padding_only(cuda_device, n, dim, ot, share):
    """Padded places sort last: whole ranges of the sorted order without a row to add.  What the
    ring held before must not reach the sums, every time."""
    from mega_trading_b200.kernels.embedding import scaled_embedding

    g = torch.Generator(device=cuda_device).manual_seed(n)
    vocab, pad = 700, 13
    ids = torch.randint(0, vocab, (n,), device=cuda_device, generator=g)
    gone = torch.rand(n, device=cuda_device, generator=g) < share
    ids[gone] = pad
    ids[~gone & (ids == pad)] = pad + 1
    w = torch.randn(vocab, dim, device=cuda_device, generator=g).to(ot).requires_grad_()
    grad = torch.randn(n, dim, device=cuda_device, generator=g).to(ot)
    (first,) = torch.autograd.grad(scaled_embedding(ids, w, padding_idx=pad), w, grad)
    _check_grad(first, ids, grad, vocab, 1.0, pad)
    grad[gone] = float("nan")
    for _ in range(8):
        (again,) = torch.autograd.grad(scaled_embedding(ids, w, padding_idx=pad), w, grad)
        assert torch.equal(again, first)


@pytest.mark.parametrize("n", [5, 900])
def test_embedding_carries_forward_mode_tangents(cuda_device, n):
    """Tangents of the table (a parameter, a plain tensor, under no_grad) and of the output's gradient."""
    import torch.autograd.forward_ad as fw

    from mega_trading_b200.kernels.embedding import scaled_embedding

    g = torch.Generator(device=cuda_device).manual_seed(n)
    ids = torch.randint(0, 10, (n,), device=cuda_device, generator=g)
    w = torch.randn(10, 8, device=cuda_device, generator=g)
    t = torch.randn(10, 8, device=cuda_device, generator=g)
    with fw.dual_level():
        for leaf, grad_mode in ((w, True), (w, False), (w.clone().requires_grad_(), True),
                                (w.clone().requires_grad_(), False)):
            with torch.set_grad_enabled(grad_mode):
                y = scaled_embedding(ids, fw.make_dual(leaf, t), scale=2.0, padding_idx=3, out_dtype=BF16)
            value, tangent = fw.unpack_dual(y)
            assert torch.equal(value.detach(), (2.0 * w[ids]).to(BF16))
            assert torch.equal(tangent.detach(), (2.0 * t[ids]).to(BF16))
        # forward over reverse: the gradient of sum(y^2) / 2 has the tangent of y's own gradient
        leaf = w.clone().requires_grad_()
        (dw,) = torch.autograd.grad(scaled_embedding(ids, fw.make_dual(leaf, t), padding_idx=3).square().sum() / 2,
                                    leaf)
        value, tangent = fw.unpack_dual(dw)
        _check_grad(value, ids, w[ids], 10, 1.0, 3)
        _check_grad(tangent, ids, t[ids], 10, 1.0, 3)


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_embedding_second_derivative_leaves_the_padding_row_out(cuda_device, bad):
    """Padded places add to no gradient, so the direction's padding row reaches nothing, whatever it holds."""
    from mega_trading_b200.kernels.embedding import scaled_embedding

    gen = torch.Generator(device=cuda_device).manual_seed(2)
    ids = torch.tensor([1, 2, 1, 5, 9], device=cuda_device)
    w = torch.randn(10, 8, device=cuda_device, generator=gen, requires_grad=True)
    g = torch.randn(5, 8, device=cuda_device, generator=gen, requires_grad=True)
    u = torch.randn(10, 8, device=cuda_device, generator=gen)
    u[9] = bad
    (dw,) = torch.autograd.grad(scaled_embedding(ids, w, padding_idx=9), w, g, create_graph=True)
    (dg,) = torch.autograd.grad(dw, g, u)
    assert bool((dg[4] == 0).all()) and torch.equal(dg[:4], u[ids[:4]])


@pytest.mark.parametrize("options", [dict(max_norm=0.5), dict(max_norm=1.0, norm_type=1.0), dict(sparse=True),
                                     dict(scale_grad_by_freq=True), dict(dtype=torch.float64), dict(padding_idx=2), {}])
def test_token_table_keeps_the_options_it_inherits(cuda_device, options):
    from mega_trading_b200.model import TokenEmbedding

    torch.manual_seed(0)
    ours = TokenEmbedding(20, 8, device=cuda_device, **options)
    plain = torch.nn.Embedding(20, 8, device=cuda_device, **options)
    plain.load_state_dict(ours.state_dict())
    ids = torch.tensor([[1, 2, 2], [3, 1, 2]], device=cuda_device)
    out = [m(ids) for m in (ours, plain)]
    for y in out:
        (y.square().sum() / 4).backward()  # every product and sum of three terms is within a rounding or two
    a, b = ours.weight.grad, plain.weight.grad
    assert torch.equal(out[0], out[1]) and torch.equal(ours.weight, plain.weight)
    assert a.is_sparse == b.is_sparse and a.dtype == b.dtype
    tol = 4 * torch.finfo(a.dtype).eps * b.to_dense().abs().max()
    assert bool(((a.to_dense() - b.to_dense()).abs() <= tol).all())


@pytest.mark.parametrize("n,dim,run,ot", [
    (262144, 64, 800, F32),
    (262144, 96, 800, BF16),
    (262144, 1024, 900, F32),    # four rows to a stage of the gather ring
    (1100000, 8, 3000, F32),
    (60000, 510, 800, F32),      # not on the bulk path: chunks of 64
    (30000, 40, 150, F16),
])
def test_embedding_long_runs_keep_the_bound(cuda_device, n, dim, run, ot):
    """Every row of a run but its first is too small to change the first's sum by itself: one rounding
    per row would lose them all, the bound of the module docstring allows some of them."""
    from mega_trading_b200.kernels.embedding import scaled_embedding

    vocab = n // run + 1
    ids = torch.arange(n, device=cuda_device) // run
    big = 2.0 ** 11 if ot is F16 else 2.0 ** 24
    grad = torch.full((n, dim), 0.875 * big * 2.0 ** -24, device=cuda_device, dtype=F32)
    grad[::run] = big
    grad = grad.to(ot)
    w = torch.zeros(vocab, dim, device=cuda_device, requires_grad=True)
    (dw,) = torch.autograd.grad(scaled_embedding(ids, w, out_dtype=ot), w, grad)
    _check_grad(dw, ids, grad, vocab, 1.0, None)
