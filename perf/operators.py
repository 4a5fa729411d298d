"""Measured cases of the token-table, distillation and 8-bit inference operators.

Five operators: the token embedding lookup with its gradient by sorted tokens,
the distillation loss of a student's output projection against a teacher's top
logits, (residual add +) RMSNorm with an 8-bit output, 8-bit row quantisation,
and the 8-bit matrix product with a scale per token and per channel.

``own`` selects the side: False runs each operator in its plain form
(elementary torch operations in 32 bits, one rounding per output), True calls
the library.  Both sides take the same ``prepare``d state.
"""

import math

import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}

VOCAB = 21504  # 2 actions x 2 sides x 21 depths x 16 volumes x 16 interarrival times
_IGNORE = -100
_TINY = 2.0 ** -119  # rows whose largest magnitude is below this quantise to zero


def listed():
    return [
        # one decoding step of 16 order-flow streams: a handful of rows of the 768-wide table
        dict(name="embed_step", op="embed", tokens=16, vocab=VOCAB, dim=768, table="fp32", out="fp32", scale=1.0,
             pad=False, train=False),
        # a ragged fine-tuning batch on a 16-bit table with padded tails and the sqrt(dim) input scale
        dict(name="embed_ragged", op="embed", tokens=30011, vocab=VOCAB, dim=1000, table="bf16", out="bf16",
             scale=math.sqrt(1000.0), pad=True, train=True),
        # the training micro-batch of the 12-layer model: 128 sequences of 2048 tokens, fp32 residual stream
        dict(name="embed_train", op="embed", tokens=128 * 2048, vocab=VOCAB, dim=768, table="fp32", out="fp32",
             scale=1.0, pad=False, train=True),
        # one short sequence against a narrow student (256 wide): the latency end of a distillation step
        dict(name="distill_small", op="distill", rows=509, vocab=VOCAB, dim=256, top=8, temp=1.0, type="bf16",
             masked=True),
        # a quarter of a micro-batch of the 12-layer student, teacher's top 32 at temperature 2
        dict(name="distill_step", op="distill", rows=16 * 2048, vocab=VOCAB, dim=768, top=32, temp=2.0, type="bf16",
             masked=False),
        # the 24-layer model's width as the student, teacher's top 64, half precision, padded sequences
        dict(name="distill_wide", op="distill", rows=4 * 4096, vocab=VOCAB, dim=1024, top=64, temp=1.5, type="fp16",
             masked=True),
        # decoding: the norm before a projection on 16 tokens
        dict(name="norm8_step", op="norm8", rows=16, dim=768, act="bf16", res="fp32", add=True),
        # prompt pass of the 24-layer teacher: branch in bf16, residual stream in fp32
        dict(name="norm8_prompt", op="norm8", rows=32 * 4096, dim=1024, act="bf16", res="fp32", add=True),
        # the gate's output (2816 wide) quantised before the down projection, an odd number of tokens
        dict(name="rows8_gate", op="rows8", rows=30011, dim=2816, act="bf16"),
        # attention outputs of 8 tokens while decoding
        dict(name="rows8_step", op="rows8", rows=8, dim=1024, act="bf16"),
        # decoding: the output projection of 4 tokens over the whole vocabulary
        dict(name="linear8_step", op="linear8", rows=4, k=768, n=VOCAB, out="bf16"),
        # prompt pass: the gate/up projection of the 24-layer teacher
        dict(name="linear8_prompt", op="linear8", rows=16 * 4096 + 1, k=1024, n=2 * 2816, out="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embed", "distill", "norm8", "rows8", "linear8"])
    if op == "embed":
        dim = rng.choice([_log(rng, 8, 1024), 8 * _log(rng, 4, 128)])
        return dict(op=op, tokens=_log(rng, 1, 128 * 2048), vocab=_log(rng, 17, 32768), dim=dim,
                    table=rng.choice(["fp32", "bf16", "fp16"]), out=rng.choice(["fp32", "bf16", "fp16"]),
                    scale=round(rng.uniform(0.5, 32.0), 3), pad=rng.random() < 0.5, train=rng.random() < 0.7)
    if op == "distill":
        rows, vocab, dim = _log(rng, 1, 16 * 2048), _log(rng, 100, 32768), 8 * _log(rng, 8, 128)
        rows = max(1, min(rows, 16 * 2048 * VOCAB * 768 // (vocab * dim)))
        return dict(op=op, rows=rows, vocab=vocab, dim=dim, top=_log(rng, 1, 64),
                    temp=round(rng.uniform(0.5, 4.0), 2), type=rng.choice(["bf16", "fp16"]),
                    masked=rng.random() < 0.5)
    if op == "norm8":
        dim = _log(rng, 16, 4096)
        rows = min(_log(rng, 1, 32 * 4096), 32 * 4096 * 1024 // dim)
        act, add = rng.choice(["fp32", "bf16", "fp16"]), rng.random() < 0.7
        return dict(op=op, rows=rows, dim=dim, act=act, res=rng.choice([act, "fp32"]) if add else act, add=add)
    if op == "rows8":
        dim = _log(rng, 16, 8192)
        rows = min(_log(rng, 1, 32 * 4096), 30011 * 2816 // dim)
        return dict(op=op, rows=rows, dim=dim, act=rng.choice(["fp32", "bf16", "fp16"]))
    k, n = 16 * _log(rng, 2, 256), _log(rng, 1, VOCAB)
    rows = max(1, min(_log(rng, 1, 16 * 4096), 16 * 4096 * 1024 * 5632 // (k * n)))
    return dict(op=op, rows=rows, k=k, n=n, out=rng.choice(["fp32", "bf16", "fp16"]))


def work(case):
    c = case
    if c["op"] == "embed":
        elems, ts, os_ = c["tokens"] * c["dim"], _SIZE[c["table"]], _SIZE[c["out"]]
        b = 8 * c["tokens"] + min(c["tokens"], c["vocab"]) * c["dim"] * ts + elems * os_
        f = elems
        if c["train"]:
            b += elems * os_ + c["vocab"] * c["dim"] * ts
            f += 2 * elems
        return {"bytes": b, "flops": f}
    if c["op"] == "distill":
        n, v, k = c["rows"], c["vocab"], c["dim"]
        return {"bytes": 2 * 2 * (n * k + v * k) + n * c["top"] * (8 + 4) + 4, "flops": 6.0 * n * v * k}
    if c["op"] == "norm8":
        a, r = _SIZE[c["act"]], _SIZE[c["res"]]
        per = a + 1 + (2 * r if c["add"] else 0)
        return {"bytes": c["rows"] * (c["dim"] * per + 4) + 4 * c["dim"], "flops": 6 * c["rows"] * c["dim"]}
    if c["op"] == "rows8":
        return {"bytes": c["rows"] * (c["dim"] * (_SIZE[c["act"]] + 1) + 4), "flops": 3 * c["rows"] * c["dim"]}
    m, k, n = c["rows"], c["k"], c["n"]
    return {"bytes": m * k + n * k + 4 * (m + n) + m * n * _SIZE[c["out"]], "flops": 2.0 * m * n * k}


def _tokens(n, vocab, g):
    """Skewed ids: a few tokens take a large part of the stream, as order-flow tokens do."""
    u = torch.rand(n, device="cuda", generator=g)
    ids = (u.pow(3.0) * vocab).long().clamp_(max=vocab - 1)
    return (ids * 7919 + 13) % vocab


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    if c["op"] == "embed":
        s = {"ids": _tokens(c["tokens"], c["vocab"], g),
             "weight": (normal(c["vocab"], c["dim"]) * 0.02).to(_TYPES[c["table"]])}
        pad = c["vocab"] - 1 if c["pad"] else None
        if pad is not None:
            s["ids"][c["tokens"] - c["tokens"] // 5:] = pad
        if c["train"]:
            s["grad"] = normal(c["tokens"], c["dim"]).to(_TYPES[c["out"]])
        s["pad"] = pad
    elif c["op"] == "distill":
        n, v, t = c["rows"], c["vocab"], _TYPES[c["type"]]
        top = min(c["top"], v)
        # a teacher's top logits: distinct ids, falling logits
        steps = torch.randint(1, v // top + 1, (n, top), device="cuda", generator=g)
        start = torch.randint(0, v, (n, 1), device="cuda", generator=g)
        ids = (start + steps.cumsum(1) - 1) % v
        ids = ids[:, torch.randperm(top, device="cuda", generator=g)].contiguous()
        logits = (normal(n, top).abs() * 3.0).sort(dim=1, descending=True).values.contiguous()
        if c["masked"]:
            gone = torch.rand(n, top, device="cuda", generator=g) < 0.1
            gone |= torch.rand(n, 1, device="cuda", generator=g) < 0.1  # whole rows: padding
            ids[gone] = _IGNORE
            logits[gone] = float("nan")
        s = {"hidden": normal(n, c["dim"]).to(t), "weight": (normal(v, c["dim"]) * 0.05).to(t),
             "ids": ids, "logits": logits,
             # loss scaling of 16-bit training: keeps the gradients of a mean over many rows in range
             "loss_scale": torch.tensor(float(n), device="cuda")}
    elif c["op"] == "norm8":
        s = {"hidden": normal(c["rows"], c["dim"]).to(_TYPES[c["act"]]),
             "weight": 1.0 + 0.2 * normal(c["dim"])}
        if c["add"]:
            s["residual"] = (normal(c["rows"], c["dim"]) * 2.0).to(_TYPES[c["res"]])
    elif c["op"] == "rows8":
        s = {"x": (normal(c["rows"], c["dim"]) * normal(c["rows"], 1).exp()).to(_TYPES[c["act"]])}
    else:
        def whole(*shape):
            return torch.randint(-127, 128, shape, device="cuda", generator=g, dtype=torch.int8)
        s = {"x": whole(c["rows"], c["k"]), "xs": normal(c["rows"]).abs() * 0.02 + 1e-3,
             "w": whole(c["n"], c["k"]), "ws": normal(c["n"]).abs() * 2e-4 + 1e-5}
    s["case"] = dict(c)
    return s


# ---------------------------------------------------------------------------
# the library's calls
# ---------------------------------------------------------------------------
def _own(s):
    c = s["case"]
    if c["op"] == "embed":
        from mega_trading_b200.kernels.embedding import scaled_embedding

        w = s["weight"].detach().requires_grad_(c["train"])
        y = scaled_embedding(s["ids"], w, scale=c["scale"], padding_idx=s["pad"], out_dtype=_TYPES[c["out"]])
        if not c["train"]:
            return {"out": y}
        return {"out": y.detach(), "dweight": torch.autograd.grad(y, w, s["grad"])[0]}
    if c["op"] == "distill":
        from mega_trading_b200.kernels.distillation import fused_linear_distillation

        h, w = s["hidden"].detach().requires_grad_(), s["weight"].detach().requires_grad_()
        loss = fused_linear_distillation(h, w, s["ids"], s["logits"], temperature=c["temp"], ignore_index=_IGNORE)
        dh, dw = torch.autograd.grad(loss, (h, w), s["loss_scale"])
        return {"loss": loss.detach(), "dhidden": dh, "dweight": dw}
    from mega_trading_b200.kernels import int8

    if c["op"] == "norm8":
        if c["add"]:
            new, q, scale = int8.add_rms_norm_int8(s["hidden"], s["residual"], s["weight"], eps=1e-5)
            return {"residual": new, "q": q, "scale": scale}
        q, scale = int8.rms_norm_int8(s["hidden"], s["weight"], eps=1e-5)
        return {"q": q, "scale": scale}
    if c["op"] == "rows8":
        q, scale = int8.quantize_rows_int8(s["x"])
        return {"q": q, "scale": scale}
    return {"out": int8.int8_linear(s["x"], s["xs"], s["w"], s["ws"], out_dtype=_TYPES[c["out"]])}


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _plain_embed(s):
    c = s["case"]
    out = (s["weight"][s["ids"]].float() * c["scale"]).to(_TYPES[c["out"]])
    if not c["train"]:
        return {"out": out}
    grad = s["grad"].float()
    if s["pad"] is not None:
        grad = grad * (s["ids"] != s["pad"]).unsqueeze(1)
    dw = torch.zeros(c["vocab"], c["dim"], device="cuda").index_add_(0, s["ids"], grad) * c["scale"]
    return {"out": out, "dweight": dw.to(_TYPES[c["table"]])}


def _log_sum_exp(x):
    top = x.amax(1, keepdim=True)
    return (x - top).exp().sum(1, keepdim=True).log() + top


def _plain_distill(s):
    c, t = s["case"], s["case"]["temp"]
    h, w = s["hidden"].float(), s["weight"].float()
    there = s["ids"] != _IGNORE
    ids = torch.where(there, s["ids"], 0)
    a = torch.where(there, s["logits"].float() / t, -math.inf)
    valid = there.any(1, keepdim=True)
    a = torch.where(valid, a, 0.0)
    logp = a - _log_sum_exp(a)
    p = torch.where(there, logp.exp(), 0.0)
    z = (h @ w.t()) / t
    lse = _log_sum_exp(z)
    row = (p * (torch.where(there, logp, 0.0) - (z.gather(1, ids) - lse))).sum(1)
    n = valid.sum().clamp(min=1)
    loss = t * t * torch.where(valid[:, 0], row, 0.0).sum() / n
    dz = (z - lse).exp_().scatter_add_(1, ids, -p)
    dz = dz * (valid * (t / n * s["loss_scale"]))
    return {"loss": loss, "dhidden": (dz @ w).to(s["hidden"].dtype), "dweight": (dz.t() @ h).to(s["weight"].dtype)}


def _to_int8(v):
    amax = v.abs().amax(1, keepdim=True)
    some = amax >= _TINY
    inv = torch.where(some, torch.full_like(amax, 127.0) / torch.where(some, amax, 1.0), 0.0)
    return torch.round(v * inv).to(torch.int8), torch.where(some, amax, 0.0)[:, 0]


def _plain_norm8(s):
    c = s["case"]
    x, out = s["hidden"].float(), {}
    if c["add"]:
        out["residual"] = (x + s["residual"].float()).to(_TYPES[c["res"]])
        x = out["residual"].float()
    rstd = torch.rsqrt((x * x).mean(1) + 1e-5)
    out["q"], amax = _to_int8(x * s["weight"])
    out["scale"] = amax * rstd / 127.0
    return out


def _plain_rows8(s):
    q, amax = _to_int8(s["x"].float())
    return {"q": q, "scale": amax / 127.0}


def _plain_linear8(s):
    acc = s["x"].float() @ s["w"].float().t()
    return {"out": (acc * s["xs"][:, None] * s["ws"]).to(_TYPES[s["case"]["out"]])}


_PLAIN = {"embed": _plain_embed, "distill": _plain_distill, "norm8": _plain_norm8, "rows8": _plain_rows8,
          "linear8": _plain_linear8}


def run(state):
    if own:
        return _own(state)
    return _PLAIN[state["case"]["op"]](state)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["op"] == "embed":
        # each token selects its table row; the gradient of a row is the sum over the places that chose it,
        # taken as differences of a running sum over the tokens in sorted order, a strip of columns at a time
        ids, w = s["ids"], s["weight"].double()
        out = {"out": torch.index_select(w, 0, ids).mul_(c["scale"])}
        if c["train"]:
            order = torch.argsort(ids)
            ends = torch.searchsorted(ids[order], torch.arange(c["vocab"], device="cuda"), right=True)
            dw = torch.empty(c["vocab"], c["dim"], device="cuda", dtype=torch.float64)
            for lo in range(0, c["dim"], 64):
                part = s["grad"][order, lo:lo + 64].double().cumsum(0)
                part = torch.cat([torch.zeros_like(part[:1]), part])[ends]
                dw[:, lo:lo + 64] = part - torch.cat([torch.zeros_like(part[:1]), part[:-1]])
            if s["pad"] is not None:
                dw[s["pad"]] = 0.0
            out["dweight"] = dw * c["scale"]
        return out
    if c["op"] == "distill":
        # KL(teacher || student) with the teacher's distribution over its listed entries, written densely
        t, h, w = c["temp"], s["hidden"].double(), s["weight"].double()
        total, count = 0.0, 0
        dh, dw = torch.zeros_like(h), torch.zeros_like(w)
        for lo in range(0, c["rows"], 8192):
            ids, lg = s["ids"][lo:lo + 8192], s["logits"][lo:lo + 8192].double()
            hit = ids.ge(0)
            e = torch.zeros_like(lg)
            e[hit] = lg[hit]
            e = torch.exp((e - e.amax(1, keepdim=True)) / t) * hit
            mass = e.sum(1, keepdim=True)
            alive = mass > 0
            p = e / mass.where(alive, torch.ones_like(mass))
            x = h[lo:lo + 8192]
            logq = torch.log_softmax(torch.matmul(x, w.T) / t, dim=1)
            dense = torch.zeros_like(logq).scatter_add_(1, ids.clamp(min=0), p)
            total += float(torch.special.xlogy(p, p).sum() - (dense * logq).sum())
            count += int(alive.sum())
            d = (logq.exp() - dense) * alive
            dh[lo:lo + 8192] = torch.matmul(d, w)
            dw += torch.matmul(d.T, x)
        count = max(count, 1)
        grad = t / count * c["rows"]
        return {"loss": torch.tensor(total * t * t / count, dtype=torch.float64), "dhidden": dh * grad,
                "dweight": dw * grad}
    if c["op"] == "norm8":
        x, out = s["hidden"].double(), {}
        if c["add"]:
            out["residual"] = x + s["residual"].double()
            x = out["residual"].to(_TYPES[c["res"]]).double()
        norm = torch.linalg.vector_norm(x, dim=1) / math.sqrt(c["dim"])
        out["q"] = None
        out["scale"] = (x * s["weight"].double()).abs().max(1).values / torch.hypot(
            norm, torch.full_like(norm, math.sqrt(1e-5))) / 127
        return out
    if c["op"] == "rows8":
        return {"q": None, "scale": s["x"].double().abs().max(1).values / 127}
    prod = torch.matmul(s["x"].double(), s["w"].double().T)
    return {"out": prod * torch.outer(s["xs"].double(), s["ws"].double())}
