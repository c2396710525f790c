"""Measured cases of the vocabulary-side operators of a training step.

Three operators share the vocabulary axis of one language-model step:

* ``embedding``  -- token lookup with scaling, and its gradient (a dense (V, d)
  matrix whose rows sum the output gradients of equal tokens);
* ``linear_ce``  -- softmax cross entropy of the head ``h w^T`` over a large
  vocabulary without keeping the logits, and the gradients of ``h`` and ``w``;
* ``distil``     -- Kullback-Leibler distillation from a teacher's top logits, and
  the gradient of the student's logits.

``run`` computes them in plain 32-bit torch operations, or, with ``own`` set,
through the framework's entry points.
"""

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _size(name):
    return 4 if name == "fp32" else 2


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one token for each sequence of a decode batch (the default vocabulary): latency only
        {"name": "embed decode", "op": "embedding", "n": 32, "v": 100287, "d": 1024, "dtype": "fp16",
         "scale": 32.0, "padding": False, "train": False},
        # prompts of the 7B trunk, 16 x 4095 tokens, embeddings scaled by sqrt(d)
        {"name": "embed prompts", "op": "embedding", "n": 65520, "v": 32000, "d": 4096, "dtype": "bf16",
         "scale": 64.0, "padding": False, "train": False},
        # one micro-step of the 1B trunk: 16 x 4096 padded tokens, forward and gradient
        {"name": "embed train", "op": "embedding", "n": 65536, "v": 32000, "d": 2048, "dtype": "bf16",
         "scale": 1.0, "padding": True, "train": True},
        # fp32 training with the default vocabulary and an odd width (unaligned rows)
        {"name": "embed train odd fp32", "op": "embedding", "n": 8189, "v": 100287, "d": 1001, "dtype": "fp32",
         "scale": 1.5, "padding": False, "train": True},
        # the tiny configuration's head on a short batch: launches count
        {"name": "ce train short", "op": "linear_ce", "n": 512, "v": 32000, "d": 256, "dtype": "bf16",
         "reduction": "mean", "train": True},
        # scoring sequences with the 1B head (per-token losses, no gradient)
        {"name": "ce score", "op": "linear_ce", "n": 8191, "v": 32000, "d": 2048, "dtype": "bf16",
         "reduction": "none", "train": False},
        # the 1B head in training: 4 x 4096 tokens
        {"name": "ce train", "op": "linear_ce", "n": 16384, "v": 32000, "d": 2048, "dtype": "bf16",
         "reduction": "mean", "train": True},
        # the default odd vocabulary in fp16, per-token weights (a policy-gradient step)
        {"name": "ce train weighted odd fp16", "op": "linear_ce", "n": 4093, "v": 100287, "d": 1024, "dtype": "fp16",
         "reduction": "none", "train": True},
        # a few positions against a stored teacher: latency, few rows with a long axis
        {"name": "distil short", "op": "distil", "n": 17, "v": 100287, "k": 32, "dtype": "bf16",
         "temperature": 1.0, "reduction": "none", "ragged": False, "train": False},
        # evaluation of a student, ragged teacher lists
        {"name": "distil score", "op": "distil", "n": 4095, "v": 32000, "k": 64, "dtype": "fp16",
         "temperature": 1.0, "reduction": "mean", "ragged": True, "train": False},
        # a training step, 4 x 4096 tokens of the 1B head
        {"name": "distil train", "op": "distil", "n": 16384, "v": 32000, "k": 64, "dtype": "bf16",
         "temperature": 2.0, "reduction": "mean", "ragged": True, "train": True},
        # the default odd vocabulary (unaligned rows), fp32 logits, long teacher lists
        {"name": "distil train odd fp32", "op": "distil", "n": 4093, "v": 100287, "k": 200, "dtype": "fp32",
         "temperature": 1.5, "reduction": "sum", "ragged": True, "train": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embedding", "linear_ce", "distil"])
    v = rng.choice([32000, 100287, _log_int(rng, 500, 100287)])
    train = rng.random() < 0.6
    if op == "embedding":
        c = {"op": op, "n": _log_int(rng, 1, 65536), "v": v, "d": _log_int(rng, 64, 4096),
             "dtype": rng.choice(["bf16", "fp16", "fp32"]), "scale": rng.choice([1.0, 8.0, 22.625]),
             "padding": rng.random() < 0.5, "train": train}
        if rng.random() < 0.6:
            c["d"] = max(8, c["d"] // 8 * 8)
        most = 500e6
        while work(c)["bytes"] > most:
            c["n"], c["d"] = max(1, c["n"] * 3 // 4), max(64, c["d"] * 3 // 4)
        return c
    if op == "linear_ce":
        c = {"op": op, "n": _log_int(rng, 1, 16384), "v": v, "d": _log_int(rng, 8, 512) * 8,
             "dtype": rng.choice(["bf16", "fp16"]), "reduction": rng.choice(["mean", "sum", "none"]), "train": train}
        while c["n"] * c["v"] * c["d"] > 16384 * 32000 * 2048:
            c["n"] = c["n"] * 3 // 4
        return c
    c = {"op": op, "n": _log_int(rng, 1, 16384), "v": v, "k": _log_int(rng, 1, 256),
         "dtype": rng.choice(["bf16", "fp16", "fp32"]), "temperature": rng.choice([1.0, 2.0, 3.5]),
         "reduction": rng.choice(["mean", "sum", "none"]), "ragged": rng.random() < 0.5, "train": train}
    while c["n"] * c["v"] * _size(c["dtype"]) > 1.0e9:
        c["n"] = c["n"] * 3 // 4
    return c


# ------------------------------------------------------------------ the inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _tokens(n, v, g):
    """Token ids with the 1 / rank frequencies of text, ranks spread over the vocabulary."""
    u = torch.rand(n, device="cuda", generator=g, dtype=torch.float64)
    rank = (torch.exp(u * math.log(v)) - 1.0).long().clamp_(0, v - 1)
    return torch.randperm(v, device="cuda", generator=g)[rank]


def prepare(case, seed):
    c, g = case, _gen(seed)
    n, v, t = c["n"], c["v"], _DTYPES[c["dtype"]]
    s = {"case": c}
    if c["op"] == "embedding":
        w = (0.02 * torch.randn(v, c["d"], device="cuda", generator=g)).to(t)
        ids = _tokens(n, v, g)
        s["padding"] = None
        if c["padding"]:  # a twentieth of the positions is padding at the ends of sequences
            s["padding"] = v - 1
            ids[n - n // 20:] = v - 1
        s.update(ids=ids, w=w.requires_grad_(c["train"]))
        if c["train"]:
            s["dy"] = torch.randn(n, c["d"], device="cuda", generator=g).to(t)
        return s
    if c["op"] == "linear_ce":
        d = c["d"]
        w = torch.randn(v, d, device="cuda", generator=g) * (2.0 / math.sqrt(d))
        tgt = _tokens(n, v, g)
        h = torch.randn(n, d, device="cuda", generator=g) + 1.5 * w[tgt]  # a head that has learned something
        drop = torch.rand(n, device="cuda", generator=g) < 0.1
        drop[0] = False
        tgt = torch.where(drop, torch.full_like(tgt, -100), tgt)  # prompt and padding positions
        s.update(h=h.to(t).requires_grad_(c["train"]), w=w.to(t).requires_grad_(c["train"]), targets=tgt)
        if c["train"]:
            s["g"] = (torch.randn(n, device="cuda", generator=g) if c["reduction"] == "none"
                      else torch.rand((), device="cuda", generator=g) + 0.5)
        return s
    k = min(c["k"], v)
    x = 2.0 * torch.randn(n, v, device="cuda", generator=g)
    start = torch.randint(0, v, (n, 1), device="cuda", generator=g)
    ids = (start + torch.arange(k, device="cuda") * (v // k)) % v  # k distinct tokens for each row
    teacher = (6.0 + 2.0 * torch.randn(n, k, device="cuda", generator=g)).sort(dim=1, descending=True)[0]
    x.scatter_add_(1, ids, 0.8 * teacher + torch.randn(n, k, device="cuda", generator=g))
    if c["ragged"]:  # lists cut at a probability, some rows (prompts) without a teacher
        kept = torch.randint(0, k + 1, (n, 1), device="cuda", generator=g)
        kept[0] = k
        ids = torch.where(torch.arange(k, device="cuda") < kept, ids, torch.full_like(ids, -1))
    s.update(x=x.to(t).requires_grad_(c["train"]), teacher=teacher.to(t), ids=ids)
    if c["train"]:
        s["g"] = (torch.randn(n, device="cuda", generator=g) if c["reduction"] == "none"
                  else torch.rand((), device="cuda", generator=g) + 0.5)
    return s


# ------------------------------------------------------------------ one pass
def run(state):
    c = state["case"]
    if own:
        return _OWN[c["op"]](state, c)
    with torch.no_grad():
        return _PLAIN[c["op"]](state, c)


def _own_embedding(s, c):
    from llm_research_b200 import ops

    out = ops.embedding(s["ids"], s["w"], scale=c["scale"], padding_idx=s["padding"])
    if not c["train"]:
        return {"out": out}
    dw, = torch.autograd.grad(out, (s["w"],), s["dy"])
    return {"out": out.detach(), "dw": dw}


def _plain_embedding(s, c):
    ids, w = s["ids"], s["w"]
    out = (w[ids].float() * c["scale"]).to(w.dtype)
    if not c["train"]:
        return {"out": out}
    dw = torch.zeros(w.shape, dtype=torch.float32, device=w.device)
    dw.index_add_(0, ids, s["dy"].float())
    if s["padding"] is not None:
        dw[s["padding"]] = 0.0
    return {"out": out, "dw": (dw * c["scale"]).to(w.dtype)}


def _own_linear_ce(s, c):
    from llm_research_b200 import ops

    loss = ops.piecewise_linear_cross_entropy(s["h"], s["w"], s["targets"], reduction=c["reduction"])
    if not c["train"]:
        return {"loss": loss}
    dh, dw = torch.autograd.grad(loss, (s["h"], s["w"]), s["g"])
    return {"loss": loss.detach(), "dh": dh, "dw": dw}


def _reduced(rows, counted, reduction):
    """The loss, and the factor of each row in it."""
    if reduction == "none":
        return rows, counted
    if reduction == "sum":
        return rows.sum(), counted
    n = counted.sum().clamp(min=1.0)
    return rows.sum() / n, counted / n


def _plain_linear_ce(s, c):
    h, w, t = s["h"].float(), s["w"].float(), s["targets"]
    counted = (t != -100).float()
    at = t.clamp(min=0)[:, None]
    z = h @ w.t()
    m = z.amax(dim=1, keepdim=True)
    lse = m + (z - m).exp().sum(dim=1, keepdim=True).log()
    rows = (lse - z.gather(1, at))[:, 0] * counted
    loss, factor = _reduced(rows, counted, c["reduction"])
    if not c["train"]:
        return {"loss": loss}
    z = (z - lse).exp()
    z.scatter_add_(1, at, torch.full_like(at, -1.0, dtype=torch.float32))
    z *= (s["g"] * factor)[:, None]
    return {"loss": loss, "dh": (z @ w).to(s["h"].dtype), "dw": (z.t() @ h).to(s["w"].dtype)}


def _own_distil(s, c):
    from llm_research_b200 import ops

    loss = ops.topk_distillation(s["x"], s["teacher"], s["ids"], temperature=c["temperature"],
                                 reduction=c["reduction"])
    if not c["train"]:
        return {"loss": loss}
    dx, = torch.autograd.grad(loss, (s["x"],), s["g"])
    return {"loss": loss.detach(), "dx": dx}


def _plain_distil(s, c):
    T, ids = c["temperature"], s["ids"]
    x = s["x"].float() / T
    kept = ids >= 0
    at = ids.clamp(min=0)
    y = torch.where(kept, s["teacher"].float() / T, torch.full_like(at, -1e30, dtype=torch.float32))
    y = y - y.amax(dim=1, keepdim=True)
    e = torch.where(kept, y.exp(), torch.zeros_like(y))
    total = e.sum(dim=1, keepdim=True)
    counted = (total[:, 0] > 0).float()
    p = e / total.clamp(min=1e-30)
    log_p = y - total.clamp(min=1e-30).log()
    m = x.amax(dim=1, keepdim=True)
    lse = m + (x - m).exp().sum(dim=1, keepdim=True).log()
    rows = T * T * torch.where(kept, p * (log_p - (x.gather(1, at) - lse)), torch.zeros_like(p)).sum(dim=1)
    loss, factor = _reduced(rows, counted, c["reduction"])
    if not c["train"]:
        return {"loss": loss}
    x = (x - lse).exp()
    x.scatter_add_(1, at, -p)
    x *= (T * s["g"] * factor)[:, None]
    return {"loss": loss, "dx": x.to(s["x"].dtype)}


_OWN = {"embedding": _own_embedding, "linear_ce": _own_linear_ce, "distil": _own_distil}
_PLAIN = {"embedding": _plain_embedding, "linear_ce": _plain_linear_ce, "distil": _plain_distil}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c, e = case, _size(case["dtype"])
    n, v = c["n"], c["v"]
    if c["op"] == "embedding":
        d = c["d"]
        moved = 8 * n + (min(n, v) + n) * d * e  # ids, the looked-up rows, the output
        if c["train"]:
            moved += (n + v) * d * e             # the output's gradient, the weight's gradient
        return {"bytes": moved, "flops": n * d * (2 if c["train"] else 1)}
    if c["op"] == "linear_ce":
        d = c["d"]
        moved = (n + v) * d * e * (2 if c["train"] else 1) + 12 * n
        return {"bytes": moved, "flops": (6.0 if c["train"] else 2.0) * n * v * d}
    moved = n * v * e * (2 if c["train"] else 1) + n * c["k"] * (8 + e) + 4 * n
    return {"bytes": moved, "flops": n * v * (8 if c["train"] else 4)}


# ------------------------------------------------------------------ from the definition, in 64 bits
def exact(case, seed):
    s, c = prepare(case, seed), case
    f = torch.float64
    if c["op"] == "embedding":
        w, ids = s["w"].detach().to(f), s["ids"]
        got = {"out": torch.nn.functional.embedding(ids, w) * c["scale"]}
        if c["train"]:
            dw = torch.zeros_like(w).index_put_((ids,), s["dy"].to(f) * c["scale"], accumulate=True)
            if s["padding"] is not None:
                dw[s["padding"]] = 0
            got["dw"] = dw
        return got
    blocks = range(0, c["n"], 2048)
    if c["op"] == "linear_ce":
        n = max(int((s["targets"] != -100).sum()), 1)
        w = s["w"].detach().to(f)
        losses, dh, dw = [], [], torch.zeros_like(w)
        for b in blocks:
            h, t = s["h"][b:b + 2048].detach().to(f), s["targets"][b:b + 2048]
            logq = torch.log_softmax(h @ w.t(), dim=1)
            losses.append(torch.nn.functional.nll_loss(logq, t, ignore_index=-100, reduction="none"))
            if c["train"]:
                up = s["g"].to(f)[b:b + 2048] if c["reduction"] == "none" else \
                    s["g"].to(f) / (n if c["reduction"] == "mean" else 1)
                dz = logq.exp_() - torch.nn.functional.one_hot(t.clamp(min=0), c["v"])
                dz *= (up * (t != -100)).reshape(-1, 1)
                dh.append(dz @ w)
                dw += dz.t() @ h
        loss = torch.cat(losses)
        loss = loss if c["reduction"] == "none" else loss.sum() / (n if c["reduction"] == "mean" else 1)
        return {"loss": loss, "dh": torch.cat(dh), "dw": dw} if c["train"] else {"loss": loss}
    T, losses, dx = c["temperature"], [], []
    n = max(int((s["ids"] >= 0).any(dim=1).sum()), 1)
    for b in blocks:
        with torch.enable_grad():
            x = s["x"][b:b + 2048].detach().to(f).requires_grad_(c["train"])
            ids = s["ids"][b:b + 2048]
            some = (ids >= 0).any(dim=1)
            teacher = s["teacher"][b:b + 2048].to(f).masked_fill(ids < 0, -math.inf) / T
            teacher = torch.where(some[:, None], teacher, torch.zeros_like(teacher))
            p = torch.softmax(teacher, dim=1)
            q = torch.log_softmax(x / T, dim=1).gather(1, ids.clamp(min=0))
            row = (T * T) * torch.where(ids >= 0, torch.special.xlogy(p, p) - p * q, torch.zeros_like(p)).sum(dim=1)
            losses.append(row.detach())
            if c["train"]:
                up = s["g"].to(f)[b:b + 2048] if c["reduction"] == "none" else \
                    (s["g"].to(f) / (n if c["reduction"] == "mean" else 1)).expand(row.shape)
                dx.append(torch.autograd.grad(row, x, up)[0])
    loss = torch.cat(losses)
    loss = loss if c["reduction"] == "none" else loss.sum() / (n if c["reduction"] == "mean" else 1)
    return {"loss": loss, "dx": torch.cat(dx)} if c["train"] else {"loss": loss}
