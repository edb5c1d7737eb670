"""The operators on a language model's logits, as cases that can be timed: scoring tokens
(``token_logprobs``) and learning from a teacher's top logits (``distill_loss``).

``own`` selects the framework's kernels; otherwise each operator is computed from elementary torch
operations.  A case is a dict of

    op           "score" or "distill"
    train        whether the gradient of the logits is part of the pass
    batch, length, vocab, dtype
    k            alternatives returned (score) or the teacher's slots (distill)
    shift        the logits are [:, :-1] of a [batch, length + 1, vocab] tensor, as next-token losses take them
    behind       columns behind the vocabulary (a head padded to a round width)
    masked       the share of the vocabulary that a mask has set to -inf
    padding      the share of rows that are padding (token == IGNORE)
    temperature, alpha, tail, reduction   as the operators take them
"""
import math
import random

import torch

own = False

IGNORE = -100
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}

BASE = dict(train=False, dtype="fp32", k=0, shift=False, behind=0, masked=0.0, padding=0.0, temperature=1.0)
SCORE = dict(BASE, op="score")
DISTILL = dict(BASE, op="distill", train=True, alpha=1.0, tail=False, reduction="mean")


def listed():
    return [
        # a character model's batch (64 x 256, vocabulary 65) scored after a training step: odd rows of 260 bytes
        dict(SCORE, name="score_char", batch=64, length=256, vocab=65, k=5),
        # the same batch with gradients, as a policy or a calibration loss takes them
        dict(SCORE, name="score_char_train", batch=64, length=256, vocab=65, k=4, train=True),
        # one token served: its alternatives over a large vocabulary, one row for the whole GPU
        dict(SCORE, name="score_one", batch=1, length=1, vocab=131072, dtype="bf16", k=20),
        # a served batch, constrained by a mask, from a head that is padded to a round width (odd vocabulary)
        dict(SCORE, name="score_served", batch=48, length=1, vocab=50021, behind=27, k=8, masked=0.5, temperature=0.7),
        # a teacher's pass over its training text: shifted logits, 64 alternatives for each position
        dict(SCORE, name="score_teacher", batch=8, length=512, vocab=131072, dtype="bf16", k=64, shift=True),
        # a policy-gradient step: log probabilities with an entropy bonus, padded sequences
        dict(SCORE, name="score_policy", batch=16, length=512, vocab=65536, dtype="bf16", train=True, padding=0.2),
        # a character model learning from another, hard and soft labels mixed
        dict(DISTILL, name="distill_char", batch=64, length=256, vocab=65, k=8, alpha=0.5, temperature=2.0),
        # a small batch at an odd vocabulary: latency
        dict(DISTILL, name="distill_small", batch=3, length=33, vocab=5003, k=16, tail=True, padding=0.1),
        # fp32 logits with two temperatures and an odd vocabulary
        dict(DISTILL, name="distill_mixed", batch=4, length=512, vocab=50021, k=32, alpha=0.7, temperature=2.0,
             padding=0.1),
        # the teacher's remaining mass as one bucket
        dict(DISTILL, name="distill_tail", batch=8, length=512, vocab=65536, dtype="bf16", k=50, tail=True),
        # the largest step: shifted logits of a large vocabulary
        dict(DISTILL, name="distill_large", batch=16, length=512, vocab=131072, dtype="bf16", k=64, shift=True),
        # a validation pass: each row's loss, no gradient
        dict(DISTILL, name="distill_eval", batch=8, length=512, vocab=32768, dtype="bf16", k=20, train=False,
             padding=0.3, reduction="none"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    op = rng.choice(["score", "distill"])
    c = dict(SCORE if op == "score" else DISTILL)
    c["dtype"] = rng.choice(["fp32", "bf16"])
    c["vocab"] = max(8, min(262144, _log_uniform(rng, 8, 262144) + rng.choice([0, 0, 1])))
    rows = _log_uniform(rng, 1, min(131072, max(1, 2 ** 28 // c["vocab"])))
    c["batch"] = min(rows, rng.choice([1, 2, 5, 16]))
    c["length"] = max(1, rows // c["batch"])
    c["shift"] = rng.random() < 0.3
    c["behind"] = rng.choice([0, 0, 0, 1, 27])
    c["masked"] = rng.choice([0.0, 0.0, 0.5, 0.9])
    c["padding"] = rng.choice([0.0, 0.0, 0.3])
    c["temperature"] = rng.choice([1.0, 0.7, 2.0])
    c["train"] = rng.random() < 0.6
    if op == "score":
        c["k"] = rng.choice([0, min(c["vocab"], _log_uniform(rng, 1, 128))])
    else:
        c["k"] = min(c["vocab"], _log_uniform(rng, 1, 128))
        c["alpha"] = rng.choice([1.0, 0.5, 0.9])
        c["tail"] = rng.random() < 0.4
        if c["tail"]:  # something has to be left outside the slots
            c["k"] = min(c["k"], c["vocab"] // 2)
            c["masked"] = c["masked"] if c["vocab"] >= 1024 else 0.0
        c["reduction"] = rng.choice(["mean", "mean", "sum"]) if c["train"] else rng.choice(["mean", "none"])
    return c


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = dict(generator=g, device="cuda")
    B, T, V, k = case["batch"], case["length"], case["vocab"], case["k"]
    dtype = DTYPES[case["dtype"]]
    base = torch.randn(B, T + (1 if case["shift"] else 0), V + case["behind"], dtype=dtype, **rnd).mul_(2.5)
    logits = base[:, :T, :V]
    if case["masked"] > 0:
        logits.masked_fill_(torch.rand(V, **rnd) < case["masked"], float("-inf"))
    tokens = torch.randint(0, V, (B, T), **rnd)
    state = {"case": case}
    if case["op"] == "distill":
        # distinct slots for each row, spread over the vocabulary; a teacher's log probabilities that leave some mass
        first = torch.randint(0, V, (B, T, 1), **rnd)
        state["top_index"] = (first + torch.arange(k, device="cuda") * max(1, V // k)) % V
        raw = torch.randn(B, T, k, **rnd).mul_(2.0)
        left = torch.rand(B, T, 1, **rnd).mul_(0.3).add_(0.02)
        state["top_logprob"] = raw - raw.exp().sum(-1, keepdim=True).log() + (1 - left).log()
        # the student gives those tokens most of its mass too
        logits.scatter_(-1, state["top_index"],
                        (raw + torch.randn(B, T, k, **rnd) + math.log(V) + 3.0 * case["temperature"]).to(dtype))
    if case["op"] == "score" or case["alpha"] < 1.0:
        # the given tokens are never masked
        logits.scatter_(-1, tokens[..., None], torch.randn(B, T, 1, **rnd).mul_(2.0).add_(4.0).to(dtype))
    if case["padding"] > 0:
        tokens[torch.rand(B, T, **rnd) < case["padding"]] = IGNORE
    state["logits"], state["tokens"] = logits, tokens
    if case["op"] == "score" and case["train"]:
        state["g_logprob"] = torch.randn(B, T, **rnd)
        state["g_entropy"] = torch.randn(B, T, **rnd).mul_(0.1)
        state["g_top"] = torch.randn(B, T, k, **rnd)
    return state


def _targets(case, tokens):
    """distill_loss's targets: the hard labels, or the mark of padded rows alone, or none."""
    return tokens if case["alpha"] < 1.0 or case["padding"] > 0 else None


def _parts(x):
    """max, exp(x - max) and its sum over the last dimension."""
    m = x.amax(-1, keepdim=True)
    e = (x - m).exp()
    return m, e, e.sum(-1, keepdim=True)


def _top(logits, k):
    """The k largest values' indices, largest first, equal values by index: topk of (value, -index) in one integer."""
    bits = (logits.float() + 0.0).view(torch.int32)  # -0 counts as 0
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    at = torch.arange(logits.shape[-1] - 1, -1, -1, device=logits.device)
    return logits.shape[-1] - 1 - ((order << 32) | at).topk(k, dim=-1).values.bitwise_and(0xFFFFFFFF)


def _plain_score(s):
    case, logits, tokens = s["case"], s["logits"], s["tokens"]
    tau, k = case["temperature"], case["k"]
    x = logits.float() / tau
    m, e, total = _parts(x)
    live = tokens != IGNORE
    at = torch.where(live, tokens, 0)[..., None]
    log_total = total.log()
    logprob = (x.gather(-1, at) - m - log_total)[..., 0]
    p = e / total
    log_p = torch.where(p > 0, x - m - log_total, 0.0)
    entropy = -(p * log_p).sum(-1)
    out = {"logprob": torch.where(live, logprob, 0.0), "entropy": torch.where(live, entropy, 0.0)}
    index = _top(logits, k) if k else torch.zeros(*tokens.shape, 0, dtype=torch.long, device=x.device)
    top = x.gather(-1, index) - m - log_total
    out["top_index"] = torch.where(live[..., None], index, -1)
    out["top_logprob"] = torch.where(live[..., None], top, float("-inf"))
    if case["train"]:
        g = s["g_logprob"][..., None]
        gt = s["g_top"]
        d = -p * (g + gt.sum(-1, keepdim=True) + s["g_entropy"][..., None] * (log_p + entropy[..., None]))
        d.scatter_add_(-1, at, g)
        d.scatter_add_(-1, index, gt)
        d = torch.where(live[..., None], d / tau, 0.0)
        out["grad"] = d.to(logits.dtype)
    return out


def _plain_distill(s):
    case, logits = s["case"], s["logits"]
    index, l = s["top_index"], s["top_logprob"]
    tau, alpha = case["temperature"], case["alpha"]
    targets = _targets(case, s["tokens"])
    x = logits.float() / tau
    m, e, total = _parts(x)
    p = e / total
    log_p = x.gather(-1, index) - m - total.log()
    if case["tail"]:
        q64 = l.double().exp()  # the rest of the mass is a small difference
        rest64 = (1 - q64.sum(-1, keepdim=True)).clamp(min=0)
        q, rest = q64.float(), rest64.float()
        p_rest = p.scatter(-1, index, 0.0).sum(-1, keepdim=True)
        kl = (q * (l - log_p)).sum(-1) + torch.where(rest > 0, rest * (rest.log() - p_rest.log()), 0.0)[..., 0]
    else:
        lm, le, ltotal = _parts(l)
        q = le / ltotal
        kl = (q * (l - lm - ltotal.log() - log_p)).sum(-1)
    rows = alpha * tau * tau * kl
    live = torch.ones_like(rows, dtype=torch.bool) if targets is None else targets != IGNORE
    at = None
    if alpha < 1.0:
        at = torch.where(live, targets, 0)[..., None]
        x1 = logits.float()
        m1, e1, total1 = _parts(x1)
        rows = rows - (1 - alpha) * (x1.gather(-1, at) - m1 - total1.log())[..., 0]
    rows = torch.where(live, rows, 0.0)
    count = live.sum().clamp(min=1)
    out = {"loss": rows if case["reduction"] == "none" else rows.sum() / count if case["reduction"] == "mean" else rows.sum()}
    if case["train"]:
        if case["tail"]:
            total_q = q.sum(-1, keepdim=True) + rest
            inside = p.gather(-1, index) * total_q
            d = p * (total_q - torch.where(rest > 0, rest / p_rest, 0.0))
            d.scatter_(-1, index, inside - q)
        else:
            d = p
            d.scatter_add_(-1, index, -q)
        d = d * (alpha * tau)
        if at is not None:
            d = d + (1 - alpha) * (e1 / total1)
            d.scatter_add_(-1, at, torch.full_like(at, alpha - 1, dtype=torch.float32))
        d = torch.where(live[..., None], d, 0.0)
        if case["reduction"] == "mean":
            d = d / count
        out["grad"] = d.to(logits.dtype)
    return out


def _own_score(s):
    from aiwn_b200 import token_logprobs

    case, logits = s["case"], s["logits"]
    kw = dict(top_k=case["k"], temperature=case["temperature"], ignore_index=IGNORE)
    if not case["train"]:
        r = token_logprobs(logits, s["tokens"], **kw)
        return r._asdict()
    leaf = logits.detach().requires_grad_(True)
    r = token_logprobs(leaf, s["tokens"], **kw)
    outs, gs = [r.logprob, r.entropy], [s["g_logprob"], s["g_entropy"]]
    if case["k"]:
        outs.append(r.top_logprob)
        gs.append(s["g_top"])
    (grad,) = torch.autograd.grad(outs, leaf, gs)
    return {**{n: t.detach() for n, t in r._asdict().items()}, "grad": grad}


def _own_distill(s):
    from aiwn_b200 import distill_loss

    case, logits = s["case"], s["logits"]
    kw = dict(alpha=case["alpha"], temperature=case["temperature"], tail=case["tail"], ignore_index=IGNORE,
              reduction=case["reduction"])
    targets = _targets(case, s["tokens"])
    if not case["train"]:
        return {"loss": distill_loss(logits, s["top_index"], s["top_logprob"], targets, **kw)}
    leaf = logits.detach().requires_grad_(True)
    loss = distill_loss(leaf, s["top_index"], s["top_logprob"], targets, **kw)
    (grad,) = torch.autograd.grad(loss, leaf)
    return {"loss": loss.detach(), "grad": grad}


def run(state):
    if own:
        return _own_score(state) if state["case"]["op"] == "score" else _own_distill(state)
    return _plain_score(state) if state["case"]["op"] == "score" else _plain_distill(state)


def work(case):
    rows, V, k = case["batch"] * case["length"], case["vocab"], case["k"]
    matrix = rows * V * (4 if case["dtype"] == "fp32" else 2)
    if case["op"] == "score":
        # logits, tokens; log probability, entropy and the alternatives; with gradients, those given and the logits'
        b = matrix + rows * (8 + 8 + 12 * k) + (matrix + rows * (8 + 4 * k) if case["train"] else 0)
        # a difference, an exponential, two sums with a product; three products and two sums back
        return {"bytes": b, "flops": rows * V * (5 + (6 if case["train"] else 0))}
    hard = 8 if case["alpha"] < 1.0 or case["padding"] > 0 else 0
    b = matrix + rows * (12 * k + hard) + (matrix if case["train"] else 0) + (4 * rows if case["reduction"] == "none" else 4)
    return {"bytes": b, "flops": rows * V * ((3 if case["alpha"] == 1.0 or case["temperature"] == 1.0 else 6) + (3 if case["train"] else 0))}


def exact(case, seed):
    """The definitions in 64 bits, gradients by differentiating them, some rows at a time."""
    s = prepare(case, seed)
    B, T, V, k = case["batch"], case["length"], case["vocab"], case["k"]
    tau = case["temperature"]
    tokens = s["tokens"].reshape(-1)
    rows = B * T
    z = s["logits"]
    step = max(1, 2 ** 26 // V)
    live = tokens != IGNORE
    outs = {}

    def put(name, piece):
        outs.setdefault(name, []).append(piece.detach())

    count = max(1, int(live.sum())) if case["op"] == "score" or _targets(case, s["tokens"]) is not None else rows
    for a in range(0, rows, step):
        r = torch.arange(a, min(rows, a + step), device="cuda")
        zr = z[r // T, r % T].double().requires_grad_(case["train"])
        ok, t = live[r], tokens[r].clamp(min=0)[:, None]
        logp = torch.log_softmax(zr / tau, -1)
        if case["op"] == "score":
            lp = logp.gather(1, t)[:, 0]
            finite = torch.isfinite(logp)
            safe = torch.where(finite, logp, 0.0)
            h = -(torch.where(finite, safe.exp(), 0.0) * safe).sum(-1)
            put("logprob", torch.where(ok, lp, 0.0))
            put("entropy", torch.where(ok, h, 0.0))
            order = torch.sort(zr.detach(), dim=-1, descending=True, stable=True).indices[:, :k] if k else t[:, :0]
            top = logp.gather(1, order)
            put("top_logprob", torch.where(ok[:, None], top, float("-inf")))
            if case["train"]:
                up = [s[n].reshape(rows, -1)[r].double() for n in ("g_logprob", "g_entropy", "g_top")] if k else \
                    [s[n].reshape(rows, -1)[r].double() for n in ("g_logprob", "g_entropy")]
                goal = torch.where(ok, lp * up[0][:, 0] + h * up[1][:, 0], 0.0)
                if k:
                    goal = goal + torch.where(ok[:, None], top.masked_fill(~torch.isfinite(top), 0.0) * up[2], 0.0).sum(-1)
                    # the gradient at an alternative that a mask holds at -inf: its own slot, and all of the row's mass
                    gone = torch.where(ok[:, None] & ~torch.isfinite(top), up[2], 0.0)
                put_grad = torch.autograd.grad(goal.sum(), zr)[0]
                if k:
                    put_grad = put_grad - logp.detach().exp() * gone.sum(-1, keepdim=True) / tau
                    put_grad = put_grad.scatter_add(1, order, gone / tau)
                put("grad", put_grad)
            continue
        idx, l = s["top_index"].reshape(rows, k)[r], s["top_logprob"].reshape(rows, k)[r].double()
        ps = logp.gather(1, idx)
        if case["tail"]:
            q = l.exp()
            rest = (1 - q.sum(-1)).clamp(min=0)
            others = torch.logsumexp(logp.scatter(1, idx, float("-inf")), -1)
            kl = (q * (l - ps)).sum(-1)
            kl = kl + torch.where(rest > 0, torch.special.xlogy(rest, rest) - rest * others.masked_fill(rest <= 0, 0.0), 0.0)
        else:
            lq = torch.log_softmax(l, -1)
            kl = (lq.exp() * (lq - ps)).sum(-1)
        loss = case["alpha"] * tau ** 2 * kl
        if case["alpha"] < 1.0:
            loss = loss - (1 - case["alpha"]) * torch.log_softmax(zr, -1).gather(1, t)[:, 0]
        if _targets(case, s["tokens"]) is not None:
            loss = torch.where(ok, loss, 0.0)
        if case["reduction"] == "mean":
            loss = loss / count
        put("loss", loss if case["reduction"] == "none" else loss.sum()[None])
        if case["train"]:
            put("grad", torch.autograd.grad(loss.sum(), zr)[0])
    res = {}
    for name, pieces in outs.items():
        v = torch.cat(pieces)
        if name == "loss":
            res[name] = v.reshape(B, T) if case["reduction"] == "none" else v.sum()
        else:
            res[name] = v.reshape(B, T, *v.shape[1:])
    if case["op"] == "score":
        res["top_index"] = None
    return res
