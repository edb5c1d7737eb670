"""token_logprobs and distill_loss in 64 bits, from their definitions, with the
bounds that fp32 sums of V terms and a type's rounding leave around them.

Rounding bounds.  The kernels' base-2 exponential is off by at most 2^-22 of
its value, the exponent d = (z - m) log2(e) / tau by two roundings, |d| 2^-23,
which is |d| 2^-23 ln 2 of the value; a term of the sum weighs 2^-|d|, and
|d| 2^-|d| <= 0.54.  A sum over V terms is a chain of at most V / 512 + 32
additions (rows up to 1024 logits: 32 + 5) of 2^-24 each.  Together
    sum_tol(V) = 2^-22 + 2^-23 + (V / 512 + 40) 2^-24     relative, in s,
which is the absolute error that it causes in ln s.  A single probability is
off by that, by its own exponential (2^-22) and by |d| 2^-23 ln 2; d is at most
MAX_D in the tests' inputs."""
import torch

MAX_D = 150.0
F32 = 2.0 ** -24  # half a step of a rounding to fp32
IGNORE = -100


def sum_tol(V):
    return 2.0 ** -22 + 2.0 ** -23 + (V / 512 + 40) * 2.0 ** -24


def prob_tol(V):
    return sum_tol(V) + 2.0 ** -22 + MAX_D * 0.6932 * 2.0 ** -23


def log_softmax64(z, tau):
    """ln softmax(z / tau) of fp64 rows; -inf everywhere where nothing is above -inf."""
    x = z / tau
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == float("-inf"), 0.0, m)
    s = (x - m).exp().sum(-1, keepdim=True)
    return torch.where(s == 0, float("-inf"), x - m - s.log())


def top64(z, k):
    """Indices of the k largest, largest first, equal ones by index; NaN counts as -inf."""
    y = torch.where(torch.isnan(z), float("-inf"), z)
    return torch.sort(y, dim=-1, descending=True, stable=True).indices[..., :k]


def scores64(logits, tokens, k, tau):
    """(logprob, entropy, index, top) in 64 bits."""
    z = logits.double()
    V = z.shape[-1]
    logp = log_softmax64(z, tau)
    p = logp.exp()
    h = -torch.where(p > 0, p * logp, torch.where(torch.isnan(p), p, 0.0)).sum(-1)
    index = top64(z, k)
    top = logp.gather(-1, index)
    live = tokens != IGNORE
    bad = live & ((tokens < 0) | (tokens >= V))
    lp = logp.gather(-1, torch.where(live & ~bad, tokens, 0)[..., None])[..., 0]
    lp = torch.where(bad, float("nan"), lp)
    return (torch.where(live, lp, 0.0), torch.where(live, h, 0.0), torch.where(live[..., None], index, -1),
            torch.where(live[..., None], top, float("-inf")))


def score_grad64(logits, tokens, k, tau, g, gh, gt):
    """(gradient, sum of the absolute terms that it is made of) by the formula."""
    z = logits.double()
    logp = log_softmax64(z, tau)
    p = logp.exp()
    lp0 = torch.where(p > 0, logp, 0.0)
    h = -(p * lp0).sum(-1, keepdim=True)
    live = (tokens != IGNORE)[..., None]
    at = torch.where(live[..., 0], tokens, 0)[..., None]
    index = top64(z, k)
    g, gh, gt = g.double()[..., None], gh.double()[..., None], gt.double()
    all_ = g + gt.sum(-1, keepdim=True)
    d = -p * (all_ + gh * (lp0 + h))
    size = p * (g.abs() + gt.abs().sum(-1, keepdim=True) + gh.abs() * (lp0.abs() + h))
    d.scatter_add_(-1, at, g)
    d.scatter_add_(-1, index, gt)
    size.scatter_add_(-1, at, g.abs())
    size.scatter_add_(-1, index, gt.abs())
    return torch.where(live, d / tau, 0.0), torch.where(live, size / tau, 0.0)


def distill64(logits, index, logprob, targets, alpha, tau, tail, reduction, g=1.0):
    """(loss, gradient, error that fp32 may leave in the rows' losses, absolute terms of the gradient)."""
    z = logits.double()
    V = z.shape[-1]
    logp = log_softmax64(z, tau)
    p = logp.exp()
    used = index >= 0
    at = torch.where(used, index, 0)
    l = torch.where(used, logprob.double(), float("-inf"))
    if tail:
        q = l.exp()
        rest = (1 - q.sum(-1, keepdim=True)).clamp(min=0)
        lnq = l
    else:
        m = l.amax(-1, keepdim=True) if l.shape[-1] else l.sum(-1, keepdim=True)
        m = torch.where(m == float("-inf"), 0.0, m)
        s = (l - m).exp().sum(-1, keepdim=True)
        lnq = torch.where(s > 0, l - m - s.log(), float("-inf"))
        q = lnq.exp()
        rest = torch.zeros_like(s)
    lp = logp.gather(-1, at)
    zero = torch.zeros((), dtype=torch.float64, device=z.device)
    kl = torch.where(q > 0, q * (lnq - lp), zero).sum(-1)
    size = torch.where(q > 0, q * (lnq.abs() + lp.abs()), zero).sum(-1)
    inside = torch.zeros_like(p).scatter_add_(-1, at, used.double()) > 0
    p_rest = torch.where(inside, zero, p).sum(-1, keepdim=True)
    if tail:
        kl = kl + torch.where(rest > 0, rest * (rest.log() - p_rest.log()), zero)[..., 0]
        size = size + torch.where(rest > 0, rest * (rest.log().abs() + p_rest.log().abs()), zero)[..., 0]
    live = torch.ones_like(kl, dtype=torch.bool) if targets is None else targets != IGNORE
    rows = alpha * tau ** 2 * kl
    size = alpha * tau ** 2 * size
    hard = alpha < 1.0
    if hard:
        t = torch.where(live, targets, 0)[..., None]
        logp1 = log_softmax64(z, 1.0)
        ce = -logp1.gather(-1, t)[..., 0]
        rows = rows + (1 - alpha) * ce
        size = size + (1 - alpha) * ce.abs()
    rows, size = torch.where(live, rows, zero), torch.where(live, size, zero)
    # each logarithm carries the sums' error, and a few roundings of its size
    err = torch.where(live, (alpha * tau ** 2 * 2 + 1) * sum_tol(V), zero) + 16 * F32 * size
    count = max(1, int(live.sum()))
    scale = 1.0 / count if reduction == "mean" else 1.0
    loss = rows if reduction == "none" else rows.sum() * scale
    Q = q.sum(-1, keepdim=True) + rest
    outside = torch.where(rest > 0, rest / p_rest, zero) if tail else zero
    d = torch.where(inside, p * Q, p * (Q - outside) if tail else p * Q)
    dsize = torch.where(inside, p * Q, p * (Q + outside) if tail else p * Q)
    d = (d.scatter_add(-1, at, -torch.where(used, q, zero))) * alpha * tau
    dsize = (dsize.scatter_add(-1, at, torch.where(used, q, zero))) * alpha * tau
    if hard:
        d = d + (1 - alpha) * logp1.exp()
        dsize = dsize + (1 - alpha) * logp1.exp()
        one = torch.full_like(t, 1, dtype=torch.float64) * (1 - alpha)
        d, dsize = d.scatter_add(-1, t, -one), dsize.scatter_add(-1, t, one)
    w = (g.double()[..., None] if torch.is_tensor(g) else g) * scale
    d, dsize = torch.where(live[..., None], d * w, zero), torch.where(live[..., None], (dsize * w).abs(), zero)
    if reduction != "none":
        # V-independent: the rows' sum is a chain of at most rows / 1024 + 10 additions, and two products
        err = err.sum() * scale + (rows.numel() / 1024 + 14) * F32 * rows.abs().sum() * scale
    return loss, d, err, dsize


def near(got, want, tol, what):
    """|got - want| <= tol (elementwise, 64 bits) where want is finite, else the same inf or NaN."""
    got = got.double()
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    off = (got - want).abs() - tol
    bad = ~same & ~(off <= 0)
    assert not bad.any(), (what, int(bad.sum()), "of", bad.numel(), "first",
                           [(float(a), float(b)) for a, b in zip(got[bad][:3], want[bad][:3])])
