"""Cases of the operators that train the dense parameters around the experts: RMS norm with its
backward pass (and the residual addition before it), the embedding lookup with its gradient, and the
AdamW step over many tensors with states in 32 or 8 bits."""
import math

import torch

own = False

BLOCK = 256          # a tensor's states start at a multiple of this many values; one 8-bit scale for each
E4M3_MAX = 448.0
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
DEVICE = "cuda"


def listed():
    return [
        # one token's row in front of a layer, as a model answering word by word has it
        dict(name="norm_token", kind="norm", rows=1, width=2048, dtype="bf16", wtype="bf16", residual=False,
             train=False),
        # a training batch of 4 x 2048 tokens: residual addition and norm, forward and backward
        dict(name="norm_residual", kind="norm", rows=8192, width=2048, dtype="bf16", wtype="bf16", residual=True,
             train=True),
        # the norm of the query heads: 32 heads of 128 for each of 8192 tokens
        dict(name="norm_heads", kind="norm", rows=262144, width=128, dtype="bf16", wtype="bf16", residual=False,
             train=True),
        # a wide layer's rows, weights kept in 32 bits
        dict(name="norm_wide", kind="norm", rows=4096, width=6144, dtype="bf16", wtype="fp32", residual=False,
             train=True),
        # an odd number of odd rows in 32 bits
        dict(name="norm_odd", kind="norm", rows=1021, width=771, dtype="fp32", wtype="fp32", residual=True,
             train=True),
        # the rows of a few tokens
        dict(name="embed_tokens", kind="embed", tokens=16, vocab=151936, width=2048, dtype="bf16", scale=1.0,
             padded=0.0, train=False, adds=False),
        # a training batch of 4 x 2048 tokens: lookup and a gradient of the whole table
        dict(name="embed_batch", kind="embed", tokens=8192, vocab=151936, width=2048, dtype="bf16", scale=1.0,
             padded=0.0, train=True, adds=False),
        # a long batch whose second half is padding, odd width, scaled rows, added to the gradient of
        # the micro-batch before
        dict(name="embed_padded", kind="embed", tokens=32768, vocab=32003, width=1001, dtype="fp32", scale=31.6386,
             padded=0.5, train=True, adds=True),
        # the norms and routers of eight layers in 32 bits: many small tensors
        dict(name="adamw_small", kind="adamw", layers=8, width=2048, experts=128, vocab=0, dtype="fp32",
             master=False, bits=32),
        # two layers and the embedding, 16-bit weights with 32-bit masters
        dict(name="adamw_master", kind="adamw", layers=2, width=2048, experts=128, vocab=151936, dtype="bf16",
             master=True, bits=32),
        # the same with states in 8 bits and no masters
        dict(name="adamw8_bf16", kind="adamw", layers=2, width=2048, experts=128, vocab=151936, dtype="bf16",
             master=False, bits=8),
        # odd sizes, 32-bit weights, states in 8 bits
        dict(name="adamw8_odd", kind="adamw", layers=5, width=771, experts=37, vocab=10007, dtype="fp32",
             master=False, bits=8),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(("norm", "embed", "adamw"))
    dtype = rng.choice(("fp32", "bf16", "bf16", "fp16"))
    if kind == "norm":
        width = rng.choice((_log(rng, 16, 8192), 8 * _log(rng, 8, 1024), 128))
        rows = _log(rng, 1, min(262144, 16777216 // width))
        return dict(kind=kind, rows=rows, width=width, dtype=dtype, wtype=rng.choice((dtype, "fp32")),
                    residual=rng.random() < 0.5, train=rng.random() < 0.7)
    if kind == "embed":
        width = rng.choice((_log(rng, 16, 4096), 8 * _log(rng, 8, 512)))
        vocab = _log(rng, 300, min(151936, 67108864 // width))
        return dict(kind=kind, tokens=_log(rng, 1, min(32768, 33554432 // width)), vocab=vocab, width=width,
                    dtype=dtype, scale=rng.choice((1.0, round(math.sqrt(width), 4))),
                    padded=rng.choice((0.0, round(rng.uniform(0.05, 0.9), 3))), train=rng.random() < 0.8,
                    adds=rng.random() < 0.4)
    width = rng.choice((_log(rng, 16, 4096), 8 * _log(rng, 8, 512)))
    dtype = rng.choice(("fp32", "bf16"))
    return dict(kind=kind, layers=rng.randint(1, 11), width=width, experts=_log(rng, 4, 256),
                vocab=rng.choice((0, _log(rng, 300, min(151936, 67108864 // width)))), dtype=dtype,
                master=dtype == "bf16" and rng.random() < 0.5, bits=rng.choice((8, 32)))


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    state = {"norm": _prepare_norm, "embed": _prepare_embed, "adamw": _prepare_adamw}[case["kind"]](case, g)
    state.update(case)
    return state


def run(state):
    return {"norm": _run_norm, "embed": _run_embed, "adamw": _run_adamw}[state["kind"]](state)


def work(case):
    kind, size = case["kind"], SIZE.get(case.get("dtype"))
    if kind == "norm":
        n = case["rows"] * case["width"]
        weight = case["width"] * SIZE[case["wtype"]]
        passes, flops = (4 if case["residual"] else 2), 4 * n
        total = passes * n * size + weight
        if case["train"]:
            # dy, the normed row, the gradient of the sum; dx written. The weight gradient.
            total += ((4 if case["residual"] else 3) * n) * size + 2 * weight
            flops += 10 * n
        return {"bytes": total, "flops": flops}
    if kind == "embed":
        tokens, vocab, width = case["tokens"], case["vocab"], case["width"]
        live = tokens - int(tokens * case["padded"])
        # distinct tokens of a 1/rank law: sum over ranks of 1 - (1 - p)^n, by its integral over log rank
        steps, span = 256, math.log(vocab)
        distinct = 0.0
        for i in range(steps):
            rank = math.exp((i + 0.5) * span / steps)
            distinct += rank * span / steps * -math.expm1(-live / (rank * span))
        distinct = min(distinct, live)
        total = 8 * tokens + (distinct + tokens) * width * size
        flops = tokens * width
        if case["train"]:
            total += 8 * tokens + live * width * size
            total += 2 * distinct * width * size if case["adds"] else vocab * width * size
            flops += live * width
        return {"bytes": total, "flops": flops}
    n = sum(math.prod(s) for s in _shapes(case))
    each = 3 * size + 8 * 2 if case["bits"] == 32 else 3 * size + 2 * 2 + 16 / BLOCK
    if case["master"]:
        each += 8 - size     # the master is read and written, the 16-bit weight written only
    return {"bytes": n * each, "flops": 15 * n}


# ---- RMS norm ---------------------------------------------------------------------------------------------

EPS = 1e-6


def _prepare_norm(case, g):
    rows, width, dtype = case["rows"], case["width"], TYPES[case["dtype"]]

    def rand(*shape):
        return torch.randn(*shape, device=DEVICE, generator=g)

    # hidden states: rows of unlike size, a few columns far larger than the others
    column = torch.exp(0.5 * rand(width))
    state = {"x": (rand(rows, width) * torch.exp(0.5 * rand(rows, 1)) * column).to(dtype),
             "w": (1 + 0.2 * rand(width)).to(TYPES[case["wtype"]])}
    if case["residual"]:
        state["res"] = (rand(rows, width) * column).to(dtype)
    if case["train"]:
        state["dy"] = (0.01 * rand(rows, width)).to(dtype)
        if case["residual"]:
            state["dsum"] = (0.01 * rand(rows, width)).to(dtype)
    return state


def _run_norm(s):
    if own:
        from usaf_b200 import norms
        if not s["train"]:
            if s["residual"]:
                y, total = norms.rms_norm(s["x"], s["w"], EPS, residual=s["res"])
                return {"y": y, "sum": total}
            return {"y": norms.rms_norm(s["x"], s["w"], EPS)}
        y, rstd, total = norms.rms_norm_forward(s["x"], s["w"], EPS, residual=s.get("res"))
        dx, dw = norms.rms_norm_backward(s["dy"], total, s["w"], rstd, dsum=s.get("dsum"))
        out = {"y": y, "dx": dx, "dw": dw}
        if s["residual"]:
            out["sum"] = total
        return out
    x, w = s["x"], s["w"].float()
    if s["residual"]:
        x = (x.float() + s["res"].float()).to(x.dtype)     # the sum is stored, and the norm is the stored sum's
    x32 = x.float()
    rstd = torch.rsqrt((x32 * x32).mean(-1, keepdim=True) + EPS)
    hat = x32 * rstd
    out = {"y": (hat * w).to(x.dtype)}
    if s["residual"]:
        out["sum"] = x
    if s["train"]:
        dy = s["dy"].float()
        dg = dy * w
        dx = rstd * (dg - hat * (dg * hat).mean(-1, keepdim=True))
        if s["residual"]:
            dx = dx + s["dsum"].float()
        out["dx"] = dx.to(x.dtype)
        out["dw"] = (dy * hat).sum(0).to(s["w"].dtype)
    return out


def _exact_norm(s):
    v = s["x"].double()
    if s["residual"]:
        v = v + s["res"].double()
        total, v = v, v.to(s["x"].dtype).double()
    n = v.shape[1]
    norm = (v.pow(2).sum(1) / n + EPS).sqrt()[:, None]
    unit = v / norm
    out = {"y": unit * s["w"].double()}
    if s["residual"]:
        out["sum"] = total
    if s["train"]:
        up = s["dy"].double()
        out["dw"] = torch.einsum("rc,rc->c", up, unit)
        up = up * s["w"].double()
        along = torch.einsum("rc,rc->r", up, unit)[:, None] / n
        out["dx"] = (up - along * unit) / norm + (s["dsum"].double() if s["residual"] else 0.0)
    return out


# ---- embedding --------------------------------------------------------------------------------------------

def _padding(s):
    """The padding's id: the table's last row."""
    return s["vocab"] - 1 if s["padded"] else None


def _prepare_embed(case, g):
    tokens, vocab, width, dtype = case["tokens"], case["vocab"], case["width"], TYPES[case["dtype"]]
    # ids by a 1/rank law, as tokens of text come; the padded tail has the padding's id
    u = torch.rand(tokens, device=DEVICE, generator=g, dtype=torch.float64)
    ids = (float(vocab) ** u).floor().long().clamp_(1, vocab) - 1
    pad = int(tokens * case["padded"])
    if pad:
        ids[tokens - pad:] = _padding(case)
    state = {"ids": ids, "table": torch.empty(vocab, width, device=DEVICE, dtype=dtype).normal_(0, 0.02, generator=g)}
    if case["train"]:
        state["dy"] = torch.empty(tokens, width, device=DEVICE, dtype=dtype).normal_(0, 0.01, generator=g)
        if case["adds"]:
            state["grad"] = torch.empty(vocab, width, device=DEVICE, dtype=dtype).normal_(0, 0.01, generator=g)
    return state


def _run_embed(s):
    pad = _padding(s)
    if own:
        from usaf_b200 import embedding
        out = {"y": embedding.embedding(s["ids"], s["table"], s["scale"])}
        if s["train"]:
            out["grad"] = embedding.embedding_backward(s["dy"], s["ids"], s["vocab"], s["scale"], padding_idx=pad,
                                                       grad=s.get("grad"))
        return out
    out = {"y": (s["table"][s["ids"]].float() * s["scale"]).to(s["table"].dtype)}
    if s["train"]:
        dy = s["dy"].float() * s["scale"]
        if pad is not None:
            dy = dy * (s["ids"] != pad).unsqueeze(1)
        total = torch.zeros(s["vocab"], s["width"], device=dy.device)
        total.index_add_(0, s["ids"], dy)
        if s["adds"]:
            s["grad"].copy_(s["grad"].float() + total)
            out["grad"] = s["grad"]
        else:
            out["grad"] = total.to(s["dy"].dtype)
    return out


def _exact_embed(s):
    out = {"y": s["table"].index_select(0, s["ids"]).double() * s["scale"]}
    if s["train"]:
        grad = s["grad"].double() if s["adds"] else torch.zeros(s["vocab"], s["width"], device=DEVICE,
                                                                 dtype=torch.float64)
        keep = torch.arange(s["tokens"], device=DEVICE)
        if s["padded"]:
            keep = keep[s["ids"] != s["vocab"] - 1]
        # equal tokens next to one another, their rows' running sums taken apart at the ends
        order = keep[torch.argsort(s["ids"][keep], stable=True)]
        names, counts = torch.unique_consecutive(s["ids"][order], return_counts=True)
        ends = counts.cumsum(0)
        sums = s["dy"][order].double().cumsum(0)
        first = torch.cat([torch.zeros_like(sums[:1]), sums[ends[:-1] - 1]])[:names.numel()]
        grad[names] += s["scale"] * (sums[ends - 1] - first)
        out["grad"] = grad
    return out


# ---- AdamW ------------------------------------------------------------------------------------------------

STEP, LR, BETA1, BETA2, ADAM_EPS, DECAY, DIV = 7, 1e-3, 0.9, 0.999, 1e-8, 0.01, 3.0


def _shapes(case):
    width, head = case["width"], 128
    layer = [(case["experts"], width), (width,), (width,), (head,), (head,)]   # router, two norms, two head norms
    return layer * case["layers"] + [(width,)] + ([(case["vocab"], width)] if case["vocab"] else [])


def _places(shapes):
    """Where each tensor's states start, and how many values all have."""
    starts, at = [], 0
    for s in shapes:
        starts.append(at)
        at += -(-math.prod(s) // BLOCK) * BLOCK
    return starts, at


def _pack(x, least):
    """`x` (whole blocks) as e4m3 values and a scale for each block; `least`: what is above zero stays above it."""
    b = x.view(-1, BLOCK)
    top = b.abs().amax(1, keepdim=True)
    live = top >= 1e-30
    by = torch.where(live, top.reciprocal() * E4M3_MAX, 0.0)
    q = (b * by).to(torch.float8_e4m3fn)
    if least:
        q = torch.where((q.float() == 0) & (b > 0) & live, 2.0 ** -9, q.float()).to(torch.float8_e4m3fn)
    return q.view(-1), torch.where(live, top * (1.0 / E4M3_MAX), 0.0).view(-1)


def _unpack(q, scale):
    return (q.view(-1, BLOCK).float() * scale.view(-1, 1)).view(-1)


def _prepare_adamw(case, g):
    shapes, dtype = _shapes(case), TYPES[case["dtype"]]
    starts, total = _places(shapes)

    def flat(scale):
        return torch.empty(total, device=DEVICE).normal_(0, scale, generator=g)

    # the padding between tensors holds zeros
    real = torch.zeros(total, dtype=torch.bool, device=DEVICE)
    for s, a in zip(shapes, starts):
        real[a:a + math.prod(s)] = True
    master, m, v = flat(0.02) * real, flat(1e-3) * real, (flat(2e-3) * real).square_()
    state = {"params": [], "grads": []}
    for s, a in zip(shapes, starts):
        n = math.prod(s)
        state["params"].append(master[a:a + n].to(dtype, copy=True).view(s))
        # gradients of unlike rows, as rare and frequent tokens have them
        size = 3e-3 * torch.exp(torch.randn(s[0], device=DEVICE, generator=g))
        grad = torch.empty(s, device=DEVICE, dtype=dtype).normal_(0, 1, generator=g)
        state["grads"].append(grad.mul_(size.to(dtype).view(-1, *[1] * (len(s) - 1))))
    state["masters"] = master if case["master"] else None
    if case["bits"] == 8:
        state["m"], state["v"] = _pack(m, False), _pack(v.sqrt_(), True)
    else:
        state["m"], state["v"] = m, v
    state["decays"] = [DECAY if len(s) > 1 else 0.0 for s in shapes]
    return state


def _run_adamw(s):
    if own:
        from usaf_b200 import dense_optim
        dense_optim.adamw_step(s["params"], s["grads"], s["m"], s["v"], step=STEP, lr=LR, betas=(BETA1, BETA2),
                               eps=ADAM_EPS, weight_decay=s["decays"], masters=s["masters"], grad_div=DIV)
    else:
        _plain_adamw(s)
    out = {"params": s["params"], "m": s["m"], "v": s["v"]}
    if s["masters"] is not None:
        out["master"] = s["masters"]
    return out


def _plain_adamw(s):
    eight = s["bits"] == 8
    starts, total = _places([p.shape for p in s["params"]])

    def together(tensors):
        """The tensors in 32 bits, one after another as their states lie."""
        parts = []
        for t in tensors:
            flat = t.reshape(-1).float()
            parts += [flat, flat.new_zeros(-flat.numel() % BLOCK)]
        return torch.cat(parts)

    g = together(s["grads"]) * (1.0 / DIV)
    p = s["masters"] if s["masters"] is not None else together(s["params"])
    keep = torch.cat([p.new_full((-(-t.numel() // BLOCK) * BLOCK,), 1.0 - LR * d)
                      for t, d in zip(s["params"], s["decays"])])
    m = _unpack(*s["m"]) if eight else s["m"]
    v = _unpack(*s["v"]) if eight else s["v"]
    if eight:
        v = v * v
    m = m * BETA1 + g * (1.0 - BETA1)
    v = v * BETA2 + (g * (1.0 - BETA2)) * g
    root = torch.sqrt(v)
    p = p * keep - (m / (root * (1.0 / math.sqrt(1.0 - BETA2 ** STEP)) + ADAM_EPS)) * (LR / (1.0 - BETA1 ** STEP))
    if s["masters"] is not None:
        s["masters"].copy_(p)
    for t, a in zip(s["params"], starts):
        t.copy_(p[a:a + t.numel()].view(t.shape))
    if eight:
        for held, new in zip(s["m"] + s["v"], _pack(m, False) + _pack(root, True)):
            held.copy_(new)
    else:
        s["m"].copy_(m)
        s["v"].copy_(v)


def _exact_adamw(s):
    """One tensor after the other, in 64 bits from the states as they are stored."""
    eight = s["bits"] == 8

    def stored(held, a, n):
        if not eight:
            return held[a:a + n].double()
        blocks = slice(a // BLOCK, a // BLOCK + -(-n // BLOCK))
        values = held[0].view(-1, BLOCK)[blocks].double() * held[1][blocks].double()[:, None]
        return values.flatten()[:n]

    def codes(x, least):
        wide = torch.zeros(-(-x.numel() // BLOCK), BLOCK, device=DEVICE, dtype=torch.float64)
        wide.view(-1)[:x.numel()] = x
        top = wide.abs().max(1).values[:, None]
        unit = wide / torch.where(top > 0, top / E4M3_MAX, 1.0)
        # e4m3: steps of an eighth of the power of two below, of 2^-9 under 2^-6
        step = torch.exp2(torch.floor(torch.log2(unit.abs().clamp_min(2.0 ** -6))) - 3)
        near = torch.round(unit / step) * step
        if least:
            near = torch.where((unit > 0) & (near == 0), 2.0 ** -9, near)
        return near.flatten(), top.flatten() / E4M3_MAX

    out = {"params": [], "m": [], "v": [], "master": []}
    at = 0
    for p, g, decay in zip(s["params"], s["grads"], s["decays"]):
        n = p.numel()
        w = s["masters"][at:at + n].double() if s["masters"] is not None else p.double().flatten()
        d = g.double().flatten() / DIV
        first, second = stored(s["m"], at, n), stored(s["v"], at, n)
        if eight:
            second = second.square()
        first = BETA1 * first + (1 - BETA1) * d
        second = BETA2 * second + (1 - BETA2) * d.square()
        move = (first / (1 - BETA1 ** STEP)) / ((second / (1 - BETA2 ** STEP)).sqrt() + ADAM_EPS)
        w = w - LR * decay * w - LR * move
        out["params"].append(w.view(p.shape))
        fill = torch.zeros(-n % BLOCK, device=DEVICE, dtype=torch.float64)
        out["master"].append(torch.cat([w, fill]))
        out["m"].append(codes(first, False) if eight else torch.cat([first, fill]))
        out["v"].append(codes(second.sqrt(), True) if eight else torch.cat([second, fill]))
        at += n + fill.numel()
    for k in ("m", "v"):
        out[k] = tuple(torch.cat(x) for x in zip(*out[k])) if eight else torch.cat(out[k])
    if s["masters"] is None:
        del out["master"]
    else:
        out["master"] = torch.cat(out["master"])
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "embed": _exact_embed, "adamw": _exact_adamw}[case["kind"]](s)
