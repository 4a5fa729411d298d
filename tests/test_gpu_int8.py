"""8-bit inference operators against their definitions in 64 bits.

Quantised rows: the integers are defined by fp32 products, an exact maximum and
one fp32 product per element, all of which torch's CPU fp32 arithmetic (IEEE,
no contraction across operators) reproduces, so they must be equal.  Scales:
``a / 127 * rsqrt(mean + eps)`` takes a sum of at most 32,768 squares held in
fp32 by several threads (relative error below 4 sqrt(dim) * 2^-24 for random
signs; 1e-5 covers it) and three more fp32 operations.

Products: the integer sum is exact, float(sum) and the two scale products round
three times in fp32 (3 * 2^-24), the output once (2^-8 bf16, 2^-11 fp16 as half
steps of eps / 2, plus half a subnormal step in fp16).
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

TINY = 2.0 ** -119


def _quant_ref(v: torch.Tensor):
    amax = v.abs().amax(-1, keepdim=True)
    some = amax >= TINY
    inv = torch.where(some, torch.full_like(amax, 127.0).div(torch.where(some, amax, torch.ones_like(amax))),
                      torch.zeros_like(amax))
    return torch.round(v * inv).to(torch.int8), torch.where(some, amax, torch.zeros_like(amax))[..., 0]


def _norm_ref(x, r, w, eps):
    s = x.float() if r is None else (x.float() + r.float()).to(r.dtype).float()
    q, amax = _quant_ref(s * w.float())
    rstd = (s.double().pow(2).mean(-1) + eps).rsqrt()
    return s, q, amax.double() * rstd / 127.0


def _close(a, b, rtol):
    a, b = a.double().cpu(), b.double().cpu()
    assert a.shape == b.shape
    assert bool(((a - b).abs() <= rtol * b.abs()).all()), float(((a - b).abs() / b.abs().clamp(min=1e-300)).max())


@pytest.mark.parametrize("rows,dim,act,res,wdt,seed", [
    (1, 768, torch.bfloat16, torch.float32, torch.float32, 1),      # decoding, the training residual stream
    (5, 1024, torch.bfloat16, torch.bfloat16, torch.bfloat16, 2),
    (37, 768, torch.float16, torch.float32, torch.float32, 3),
    (64, 256, torch.float32, torch.float32, torch.float32, 4),
    (9, 2816, torch.bfloat16, torch.float32, torch.float32, 5),     # 128 threads per row
    (3, 5000, torch.float16, torch.float16, torch.float16, 6),      # 256 threads per row
    (2, 32768, torch.bfloat16, torch.float32, torch.float32, 7),    # widest
    (33, 1, torch.float32, torch.float32, torch.float32, 8),        # one element: q is +-127
    (7, 17, torch.bfloat16, torch.float32, torch.float32, 9),       # single-element accesses
    (130, 1023, torch.float16, torch.float16, torch.float32, 10),
    (4, 9001, torch.bfloat16, torch.bfloat16, torch.float32, 11),
    (1, 8, torch.bfloat16, torch.float32, torch.float32, 12),
    (700, 768, torch.bfloat16, torch.float32, torch.float32, 13),   # enough rows for one warp each
    (601, 1001, torch.float16, torch.float32, torch.float32, 14),
    (3, 4096, torch.bfloat16, torch.float32, torch.float32, 15),
])
def test_norm_int8_matches_definition(cuda_device, rows, dim, act, res, wdt, seed):
    from mega_trading_b200.kernels import int8

    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, dim, generator=g).to(act)
    r = (torch.randn(rows, dim, generator=g) * 2).to(res)
    w = (1 + 0.2 * torch.randn(dim, generator=g)).to(wdt)
    xd, rd, wd = x.to(cuda_device), r.to(cuda_device), w.to(cuda_device)
    new, q, scale = int8.add_rms_norm_int8(xd, rd, wd, eps=1e-5)
    s, qr, sr = _norm_ref(x, r, w, 1e-5)
    assert new.dtype == res and torch.equal(new.cpu().float(), s)
    assert q.dtype == torch.int8 and torch.equal(q.cpu(), qr)
    _close(scale, sr, 1e-5)
    assert torch.equal(rd.cpu(), r) and torch.equal(xd.cpu(), x)  # inputs untouched
    q2, scale2 = int8.rms_norm_int8(xd, wd, eps=1e-5)
    _, qr2, sr2 = _norm_ref(x, None, w, 1e-5)
    assert torch.equal(q2.cpu(), qr2)
    _close(scale2, sr2, 1e-5)
    q3, scale3 = int8.quantize_rows_int8(xd)
    qr3, amax = _quant_ref(x.float())
    assert torch.equal(q3.cpu(), qr3)
    _close(scale3, amax.double() / 127.0, 3 * 2.0 ** -24)


def test_norm_int8_layouts(cuda_device):
    """Leading dimensions, strided inputs and bases off the 16-byte grid."""
    from mega_trading_b200.kernels import int8

    g = torch.Generator(device=cuda_device).manual_seed(3)
    base = torch.randn(3, 5, 2 * 64 + 1, device=cuda_device, generator=g).bfloat16()
    w = torch.rand(64, device=cuda_device, generator=g) + 0.5
    for x in (base[..., 1:65], base[..., ::2][..., :64], base[:, :, 65:].transpose(0, 1)):
        q, scale = int8.rms_norm_int8(x, w, eps=1e-6)
        qc, sc = int8.rms_norm_int8(x.contiguous().clone(), w, eps=1e-6)
        assert q.shape == x.shape and scale.shape == x.shape[:-1]
        assert torch.equal(q, qc) and torch.equal(scale, sc)
    # contiguous views whose first element is not on a 16-byte boundary
    flat = torch.randn(10 * 64 + 3, device=cuda_device, generator=g).bfloat16()
    off = flat[3:].view(10, 64)
    woff = torch.cat([w.new_zeros(1), w])[1:]
    qo, so = int8.rms_norm_int8(off, woff, eps=1e-6)
    qc, sc = int8.rms_norm_int8(off.clone(), w, eps=1e-6)
    assert torch.equal(qo, qc)
    _close(so, sc, 1e-5)  # the two access widths sum the squares in another order
    q, s = int8.quantize_rows_int8(off)
    qc, sc = int8.quantize_rows_int8(off.clone())
    assert torch.equal(q, qc) and torch.equal(s, sc)


def test_norm_int8_special_rows(cuda_device):
    """Zero rows, rows of subnormals, the largest finite values, infinities and NaN."""
    from mega_trading_b200.kernels import int8

    x = torch.ones(8, 40)
    x[1] = 0
    x[2] = 1e-40                 # below 2^-119
    x[3, 7] = float("inf")
    x[4, 0] = float("nan")
    x[5] = torch.finfo(torch.float32).max
    x[6, 3] = float("-inf")
    w = torch.ones(40)
    q, s = int8.quantize_rows_int8(x.to(cuda_device))
    q, s = q.cpu(), s.cpu()
    assert bool((q[0] == 127).all()) and float(s[0]) == pytest.approx(1 / 127, rel=1e-6)
    for row in (1, 2):
        assert bool((q[row] == 0).all()) and float(s[row]) == 0.0
    for row in (3, 4, 6):
        assert bool(s[row].isnan())
    assert bool((q[5] == 127).all()) and bool(s[5].isfinite())
    assert bool((q[7] == 127).all())  # a neighbour of bad rows is untouched
    qn, sn = int8.rms_norm_int8(x.to(cuda_device), w.to(cuda_device), eps=1e-5)
    qn, sn = qn.cpu(), sn.cpu()
    assert bool((qn[1] == 0).all()) and float(sn[1]) == 0.0
    for row in (3, 4, 6):
        assert bool(sn[row].isnan())
    # a NaN in the weight reaches every row
    w[2] = float("nan")
    _, sw = int8.rms_norm_int8(x[:1].to(cuda_device), w.to(cuda_device), eps=1e-5)
    assert bool(sw.isnan().all())


def test_int8_empty_and_refusals(cuda_device):
    from mega_trading_b200.kernels import int8

    d = cuda_device
    q, s = int8.quantize_rows_int8(torch.empty(0, 64, device=d))
    assert q.shape == (0, 64) and s.shape == (0,)
    y = int8.int8_linear(q, s, torch.zeros(5, 64, dtype=torch.int8, device=d), torch.ones(5, device=d))
    assert y.shape == (0, 5) and y.dtype == torch.bfloat16
    x = torch.randn(4, 64, device=d)
    with pytest.raises(RuntimeError, match="no gradient"):
        int8.rms_norm_int8(x.clone().requires_grad_(), torch.ones(64, device=d), eps=1e-5)
    with pytest.raises(ValueError, match="one entry per hidden feature"):
        int8.rms_norm_int8(x, torch.ones(32, device=d), eps=1e-5)
    with pytest.raises(ValueError, match="same shape"):
        int8.add_rms_norm_int8(x, x[:2], torch.ones(64, device=d), eps=1e-5)
    with pytest.raises(RuntimeError, match="residual"):
        int8.add_rms_norm_int8(x, x.bfloat16(), torch.ones(64, device=d), eps=1e-5)
    with pytest.raises(ValueError, match="at most"):
        int8.quantize_rows_int8(torch.zeros(1, 40000, device=d))
    xq = torch.zeros(4, 64, dtype=torch.int8, device=d)
    wq, ones4, ones5 = torch.zeros(5, 64, dtype=torch.int8, device=d), torch.ones(4, device=d), torch.ones(5, device=d)
    with pytest.raises(ValueError, match="x_scale"):
        int8.int8_linear(xq, ones5, wq, ones5)
    with pytest.raises(ValueError, match="weight_scale"):
        int8.int8_linear(xq, ones4, wq, ones4)
    with pytest.raises(RuntimeError, match="float32 scales"):
        int8.int8_linear(xq, ones4.bfloat16(), wq, ones5)
    with pytest.raises(ValueError, match="multiple of 16"):
        int8.int8_linear(xq[:, :40].contiguous(), ones4, wq[:, :40].contiguous(), ones5)
    with pytest.raises(RuntimeError, match="int8 x and weight"):
        int8.int8_linear(xq.float(), ones4, wq, ones5)


def _product(dev, m, k, n, out, seed, extreme=False):
    from mega_trading_b200 import _lib
    from mega_trading_b200.kernels import int8

    g = torch.Generator().manual_seed(seed)
    x = torch.randint(-128, 128, (m, k), generator=g, dtype=torch.int8)
    w = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int8)
    if extreme:
        x.fill_(-128)
        w.fill_(-128)
    xs = torch.rand(m, generator=g) * 0.02 + 1e-3
    ws = torch.rand(n, generator=g) * 2e-4 + 1e-5
    y = int8.int8_linear(x.to(dev), xs.to(dev), w.to(dev), ws.to(dev), out_dtype=out)
    assert _lib.read_status(dev) == 0
    assert y.shape == (m, n) and y.dtype == out
    xd, wd = x.to(dev).double(), w.to(dev).double()
    ref = (xd @ wd.t()) * torch.outer(xs.to(dev).double(), ws.to(dev).double())
    half = torch.finfo(out).eps / 2
    tol = (half + 4 * 2.0 ** -24) * ref.abs() + torch.finfo(out).smallest_normal * torch.finfo(out).eps
    bad = (y.double() - ref).abs() > tol
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[:4].tolist())


@pytest.mark.parametrize("m,k,n,out,seed", [
    (1, 768, 21504, torch.bfloat16, 1),
    (2, 16, 1, torch.float32, 2),
    (3, 1024, 1280, torch.float16, 3),
    (8, 2816, 1024, torch.bfloat16, 4),
    (16, 400, 333, torch.float32, 5),
    (9, 768, 768, torch.bfloat16, 16),        # first tensor-core size
    (17, 768, 768, torch.bfloat16, 6),
    (100, 16, 64, torch.float32, 7),          # one K stage, mostly zero fill
    (129, 144, 130, torch.bfloat16, 8),       # ragged in every dimension, rows off the 16-byte grid
    (200, 4112, 257, torch.float16, 9),
    (300, 768, 7, torch.float32, 10),
    (1000, 1024, 4096, torch.bfloat16, 11),   # below the pairs' size
    (2000, 1024, 4096, torch.bfloat16, 14),   # CTA pairs, ragged rows
    (4097, 256, 2310, torch.float32, 12),     # CTA pairs, fp32, ragged columns
    (5000, 2816, 1023, torch.float16, 13),    # plain stores
    (8000, 272, 1023, torch.bfloat16, 15),    # CTA pairs, plain stores
])
def test_int8_linear_matches_definition(cuda_device, m, k, n, out, seed):
    _product(cuda_device, m, k, n, out, seed)


def test_int8_linear_extreme_sums_do_not_wrap(cuda_device):
    """Every element -128 at the longest inner dimension: 128 * 128 * 131,056 = 2,147,221,504 < 2^31."""
    _product(cuda_device, 3, 131056, 5, torch.float32, 0, extreme=True)
    _product(cuda_device, 40, 131056, 70, torch.float32, 0, extreme=True)


def test_int8_linear_reads_strided_and_offset_operands(cuda_device):
    from mega_trading_b200.kernels import int8

    g = torch.Generator(device=cuda_device).manual_seed(5)
    big = torch.randint(-127, 128, (64, 3 * 128 + 5), generator=g, device=cuda_device, dtype=torch.int8)
    x, w = big[:40, 5:133], big[3:60, 133:261]
    xs = torch.rand(41, device=cuda_device, generator=g)[1:]
    ws = torch.rand(58, device=cuda_device, generator=g)[1:]
    y = int8.int8_linear(x, xs, w, ws, out_dtype=torch.float32)
    ref = int8.int8_linear(x.contiguous().clone(), xs.clone(), w.contiguous().clone(), ws.clone(),
                           out_dtype=torch.float32)
    assert torch.equal(y, ref)
    y3 = int8.int8_linear(x.reshape(5, 8, 128), xs.reshape(5, 8), w, ws, out_dtype=torch.float32)
    assert torch.equal(y3.reshape(40, -1), ref)


def test_int8_linear_on_another_stream_and_in_a_graph(cuda_device):
    from mega_trading_b200.kernels import int8

    g = torch.Generator(device=cuda_device).manual_seed(6)
    h = torch.randn(300, 768, device=cuda_device, generator=g).bfloat16()
    wn = torch.rand(768, device=cuda_device, generator=g) + 0.5
    wq, ws = int8.quantize_rows_int8(torch.randn(512, 768, device=cuda_device, generator=g) * 0.02)

    def step():
        q, s = int8.rms_norm_int8(h, wn, eps=1e-5)
        return int8.int8_linear(q, s, wq, ws)

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    h.copy_(torch.randn(300, 768, device=cuda_device, generator=g))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, step())
    assert not torch.equal(out, want)


def test_int8_nan_scale_reaches_the_product(cuda_device):
    """A row with an infinity or NaN quantises to a NaN scale, and its products are NaN, alone."""
    from mega_trading_b200.kernels import int8

    gen = torch.Generator(device=cuda_device).manual_seed(7)
    wq, ws = int8.quantize_rows_int8(torch.randn(300, 64, device=cuda_device, generator=gen))
    for rows in (5, 140):
        x = torch.randn(rows, 64, device=cuda_device, generator=gen)
        x[1, 3], x[3, 0] = float("inf"), float("nan")
        q, s = int8.quantize_rows_int8(x)
        y = int8.int8_linear(q, s, wq, ws)
        assert bool(y[[1, 3]].isnan().all())
        keep = torch.ones(rows, dtype=torch.bool, device=cuda_device)
        keep[[1, 3]] = False
        assert bool(y[keep].isfinite().all())


def test_int8_operators_refuse_forward_mode_tangents(cuda_device):
    import torch.autograd.forward_ad as fw

    from mega_trading_b200.kernels import int8

    x, w = torch.randn(4, 16, device=cuda_device), torch.ones(16, device=cuda_device)
    q, s = int8.quantize_rows_int8(x)
    with fw.dual_level(), torch.no_grad():
        xd, wd, sd = (fw.make_dual(t, torch.ones_like(t)) for t in (x, w, s))
        for call in (lambda: int8.quantize_rows_int8(xd), lambda: int8.rms_norm_int8(xd, w, eps=1e-5),
                     lambda: int8.rms_norm_int8(x, wd, eps=1e-5),
                     lambda: int8.add_rms_norm_int8(x, xd, w, eps=1e-5),
                     lambda: int8.int8_linear(q, sd, q, s), lambda: int8.int8_linear(q, s, q, sd)):
            with pytest.raises(RuntimeError, match="no forward-mode gradient"):
                call()
        assert torch.equal(int8.quantize_rows_int8(x)[0], q)  # without a tangent nothing is refused


@pytest.mark.parametrize("dim", [40, 41, 768, 1024, 1500, 5000, 9001, 32768])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_norm_int8_of_rows_whose_squares_leave_fp32(cuda_device, dim, dtype):
    """Rows of the type's lowest and largest values, of 1e25, one such value alone, and (without eps) of
    1e-30: the scale is the definition's although the sum of squares is outside fp32's range."""
    from mega_trading_b200.kernels import int8

    g = torch.Generator().manual_seed(dim)
    x = torch.randn(8, dim, generator=g)
    x[0] = torch.finfo(dtype).min
    x[1] = torch.finfo(dtype).max * torch.rand(dim, generator=g)
    x[2] *= 1e25
    x[3, dim // 2] = 3e38
    x[4] *= 1e-30
    x[5] *= 1e-20
    x[6] = 0
    x = x.to(dtype)
    w = 0.2 + 0.5 * torch.rand(dim, generator=g)
    r = torch.zeros(8, dim, dtype=dtype)
    for eps in (1e-5, 0.0):
        if eps == 0.0:
            x[7, 0] = 1.0
        s, q, amax = x.float(), *_quant_ref(x.float() * w)
        want = amax.double() / 127 * (s.double().pow(2).mean(-1) + eps).rsqrt()
        want[6] = 0.0
        got = int8.rms_norm_int8(x.to(cuda_device), w.to(cuda_device), eps=eps)
        new = int8.add_rms_norm_int8(x.to(cuda_device), r.to(cuda_device), w.to(cuda_device), eps=eps)
        assert torch.equal(new[0].cpu(), x)
        for qq, scale in (got, new[1:]):
            assert torch.equal(qq.cpu(), q)
            _close(scale, want, 1e-5)
