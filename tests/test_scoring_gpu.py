"""token_logprobs and distill_loss on the GPU against their definitions in 64
bits: types, layouts, masks, ties, lengths on both sides of every kernel's
range, padding, gradients, streams, graphs and repeated calls."""
import contextlib
import itertools

import pytest
import torch

from aiwn_b200 import _lib, distill_loss, token_logprobs
from logits_oracle import (F32, IGNORE, distill64, near, prob_tol, score_grad64, scores64, sum_tol)

pytestmark = pytest.mark.gpu

DEV = "cuda"
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
LOWEST = -3.0e38


def make_logits(B, T, V, dtype, layout="plain", seed=0):
    """Rows [B, T, V] in several layouts: whole, shifted (:-1 of T + 1), behind (an odd number of columns more),
    offset (a base that is not aligned to 16 bytes), turned (batch and time exchanged)."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    behind = 5 if layout == "behind" else 0
    shape = (B, T + (layout == "shifted"), V + behind)
    n = shape[0] * shape[1] * shape[2]
    flat = torch.randn(n + 1, generator=g, device=DEV).mul_(3.0).to(dtype)
    z = (flat[1:] if layout == "offset" else flat[:-1]).view(shape)
    if layout == "shifted":
        return z[:, :-1]
    if layout == "behind":
        return z[..., :V]
    if layout == "turned":
        return z.transpose(0, 1)
    return z


def mask_(z, kind, seed=1):
    g = torch.Generator(device=DEV).manual_seed(seed)
    V = z.shape[-1]
    drop = torch.rand(V, generator=g, device=DEV) < 0.7
    drop[V // 2] = False
    if kind == "neg_inf":
        z[..., drop] = float("-inf")
    elif kind == "lowest":
        z[..., drop] = LOWEST
    elif kind == "one_left":
        z[..., torch.arange(V, device=DEV) != V // 2] = float("-inf")
    elif kind == "empty_row":
        z[0, 0] = float("-inf")
    elif kind == "all_masked":  # by finite values: what is left is an even distribution
        z[0, 0] = LOWEST
        z[-1, -1] = -1e9
    elif kind == "equal":
        z.fill_(1.5)
    elif kind == "two_values":
        z.copy_((torch.rand(z.shape, generator=g, device=DEV) < 0.5).to(z.dtype))
    elif kind == "rising":
        z.copy_(torch.linspace(-20, 20, V, device=DEV).to(z.dtype).expand(z.shape))
    elif kind == "falling":
        z.copy_(torch.linspace(20, -20, V, device=DEV).to(z.dtype).expand(z.shape))
    elif kind == "signed_zeros":
        z.copy_(torch.where(torch.rand(z.shape, generator=g, device=DEV) < 0.5, -0.0, 0.0).to(z.dtype))
    return z


def check_scores(z, tokens, k, tau, r):
    V = z.shape[-1]
    lp, h, index, top = scores64(z, tokens, k, tau)
    fin = lambda t: torch.where(torch.isfinite(t), t.abs(), 0.0)  # noqa: E731
    # ln s, the difference to the maximum and its quotient, the difference of the two
    near(r.logprob, lp, sum_tol(V) + 8 * F32 * (fin(lp) + 12), "logprob")
    near(r.top_logprob, top, sum_tol(V) + 8 * F32 * (fin(top) + 12), "top_logprob")
    # ln s and u / s, each with the sums' error; |u / s| <= ln s + H
    near(r.entropy, h, 4 * sum_tol(V) * (1 + 2 * fin(h)) + 8 * F32 * 12, "entropy")
    assert torch.equal(r.top_index, index)


SHAPES = [(2, 3, 1), (1, 2, 2), (3, 5, 31), (2, 4, 65), (1, 3, 128), (2, 2, 1000), (2, 3, 1024), (2, 3, 1025),
          (1, 3, 2049), (3, 2, 5003), (1, 2, 16391), (2, 1, 50021), (1, 1, 131072), (160, 2, 4099)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_scores(shape, dtype):
    B, T, V = shape
    for n, (layout, k, tau) in enumerate(itertools.product(["plain", "shifted", "behind", "offset", "turned"],
                                                           [0, 1, 20, 128], [1.0, 0.6])):
        if k > V or (layout != "plain" and k == 1):
            continue
        z = make_logits(B, T, V, dtype, layout, seed=n)
        tokens = torch.randint(0, V, z.shape[:2], device=DEV)
        tokens[0, 0] = IGNORE
        check_scores(z, tokens, k, tau, token_logprobs(z, tokens, k, temperature=tau))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("kind", ["neg_inf", "lowest", "one_left", "empty_row", "all_masked", "equal", "two_values", "rising",
                                  "falling", "signed_zeros"])
def test_scores_of_masked_and_tied_rows(kind, dtype):
    for B, T, V, k in [(2, 2, 65, 30), (2, 3, 1024, 128), (2, 2, 1025, 128), (3, 2, 40007, 128), (1, 1, 131072, 64),
                       (320, 1, 20011, 50), (1, 2, 6000, 5)]:
        z = mask_(make_logits(B, T, V, dtype, "behind"), kind)
        tokens = torch.randint(0, V, (B, T), device=DEV)
        check_scores(z, tokens, k, 1.0, token_logprobs(z, tokens, k))


def test_scores_of_nan_and_infinite_logits():
    for V in (50, 3001, 70001):
        for dtype in (torch.float32, torch.bfloat16):
            z = make_logits(2, 3, V, dtype)
            z[0, 1, V // 3] = float("nan")
            z[0, 2, V // 3] = float("inf")
            z[1, 0] = float("nan")
            z[1, 1, :] = float("inf")
            tokens = torch.randint(0, V, (2, 3), device=DEV)
            tokens[1, 2] = V  # outside
            r = token_logprobs(z, tokens, 10)
            nan = torch.tensor([[0, 1, 1], [1, 1, 0]], device=DEV, dtype=torch.bool)
            assert torch.equal(torch.isnan(r.entropy), nan)
            assert torch.equal(torch.isnan(r.logprob), nan | (tokens == V))
            assert torch.equal(torch.isnan(r.top_logprob).all(-1), nan)
            lp, h, index, top = scores64(z, torch.zeros_like(tokens), 10, 1.0)
            assert torch.equal(r.top_index, index)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES + [(2, 2, 70001)], ids=str)
def test_score_gradients(shape, dtype):
    B, T, V = shape
    for n, (layout, k, tau) in enumerate([("plain", 0, 1.0), ("plain", min(V, 7), 0.6), ("shifted", min(V, 128), 1.0),
                                          ("behind", min(V, 3), 2.0), ("turned", 0, 1.0), ("offset", 1, 1.0)]):
        z = make_logits(B, T, V, dtype, layout, seed=n)
        lead = z.shape[:2]
        tokens = torch.randint(0, V, lead, device=DEV)
        tokens[0, 0] = IGNORE
        g, gh, gt = torch.randn(lead, device=DEV), torch.randn(lead, device=DEV), torch.randn(*lead, k, device=DEV)
        leaf = z.detach().requires_grad_(True)
        r = token_logprobs(leaf, tokens, k, temperature=tau)
        outs, gs = [r.logprob, r.entropy, r.top_logprob], [g, gh, gt]
        outs, gs = (outs, gs) if k else (outs[:2], gs[:2])
        (got,) = torch.autograd.grad(outs, leaf, gs)
        want, size = score_grad64(z, tokens, k, tau, g, gh, gt)
        assert got.dtype == dtype and got.shape == z.shape
        # probabilities' error on every term, the sum of up to k + 1 upstream gradients, a rounding to the type
        near(got, want, (prob_tol(V) + (k + 12) * F32) * size + HALF_STEP[dtype] * want.abs() + 1e-37, (layout, k))
        check_scores(z, tokens, k, tau, type(r)(*(t.detach() for t in r)))


def test_score_gradient_of_one_result_and_of_masked_rows():
    for V in (65, 5003):
        z = mask_(make_logits(2, 3, V, torch.float32), "neg_inf")
        z[1, 2] = float("-inf")
        tokens = torch.full((2, 3), V // 2, device=DEV)
        zero = torch.zeros(2, 3, device=DEV)
        none = torch.zeros(2, 3, 0, device=DEV)
        one = torch.ones(2, 3, device=DEV)
        for pick in (0, 1):
            leaf = z.detach().requires_grad_(True)
            r = token_logprobs(leaf, tokens if pick == 0 else None)
            (got,) = torch.autograd.grad(r[pick].masked_fill(~torch.isfinite(r[pick]), 0.0).sum(), leaf)
            gs = (one.clone(), zero) if pick == 0 else (zero, one.clone())
            gs[pick][1, 2] = 0.0 if pick == 0 else 1.0
            want, size = score_grad64(z, tokens, 0, 1.0, *gs, none)
            near(got, want, (prob_tol(V) + 12 * F32) * size + F32 * want.abs(), pick)
            assert torch.equal(got[1, 2], torch.zeros_like(got[1, 2]))


def test_score_gradients_by_differences():
    V = 33
    z = make_logits(1, 2, V, torch.float32).double()
    tokens = torch.tensor([[4, 30]], device=DEV)
    w = torch.randn(3, device=DEV).double()

    def f(x):
        lp, h, _, top = scores64(x, tokens, 3, 0.8)
        return (w[0] * lp + w[1] * h + w[2] * top.sum(-1)).sum()

    leaf = z.float().requires_grad_(True)
    r = token_logprobs(leaf, tokens, 3, temperature=0.8)
    (w[0].float() * r.logprob + w[1].float() * r.entropy + w[2].float() * r.top_logprob.sum(-1)).sum().backward()
    step = 1e-5
    for t in range(2):
        for j in range(V):
            e = torch.zeros_like(z)
            e[0, t, j] = step
            diff = (f(z + e) - f(z - e)) / (2 * step)
            assert abs(float(leaf.grad[0, t, j]) - float(diff)) < 2e-5  # fp32 terms of size ~4, 1e-10 of the differences


def test_leading_dimensions_and_no_tokens():
    z = make_logits(6, 4, 300, torch.float32)
    tokens = torch.randint(0, 300, (6, 4), device=DEV)
    whole = token_logprobs(z, tokens, 5)
    r4 = token_logprobs(z.view(2, 3, 4, 300), tokens.view(2, 3, 4), 5)
    r2 = token_logprobs(z.view(24, 300), tokens.view(24), 5)
    r1 = token_logprobs(z[1, 2], tokens[1, 2], 5)
    for a, b, c, d in zip(whole, r4, r2, r1):
        assert torch.equal(a.reshape(b.shape), b) and torch.equal(a.reshape(c.shape), c) and torch.equal(a[1, 2], d)
    assert r4.top_index.shape == (2, 3, 4, 5) and r1.logprob.shape == ()
    alone = token_logprobs(z, None, 5)
    assert alone.logprob is None
    assert torch.equal(alone.entropy, whole.entropy) and torch.equal(alone.top_index, whole.top_index)
    empty = token_logprobs(z[:0], tokens[:0], 3)
    assert empty.logprob.shape == (0, 4) and empty.top_index.shape == (0, 4, 3)
    # the logits' last dimension need not be contiguous
    turned = z.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(token_logprobs(turned, tokens, 5).logprob, whole.logprob)


def test_token_views_and_repeated_calls():
    z = make_logits(4, 9, 2500, torch.bfloat16)
    both = torch.randint(0, 2500, (4, 10), device=DEV)
    r = token_logprobs(z, both[:, 1:], 3)
    again = token_logprobs(z, both[:, 1:].contiguous(), 3)
    for a, b in zip(r, again):
        assert torch.equal(a, b)
    check_scores(z, both[:, 1:], 3, 1.0, r)


# ---- distillation -------------------------------------------------------------------

def teacher(B, T, V, k, seed=0, spread=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    index = torch.rand(B, T, V, generator=g, device=DEV).topk(k, dim=-1).indices if V < 2000 else \
        (torch.randint(0, V, (B, T, 1), generator=g, device=DEV) + torch.arange(k, device=DEV) * (V // max(k, 1))) % V
    raw = torch.randn(B, T, k, generator=g, device=DEV) * 2
    left = torch.rand(B, T, 1, generator=g, device=DEV) * 0.4 + 0.01
    return index, raw - raw.exp().sum(-1, keepdim=True).log() + (1 - left).log()


def check_distill(z, index, logprob, targets, g=None, **kw):
    """Loss and gradient, upstream gradient g (None: 1)."""
    V, dtype = z.shape[-1], z.dtype
    leaf = z.detach().requires_grad_(True)
    loss = distill_loss(leaf, index, logprob, targets, **kw)
    up = torch.ones_like(loss) if g is None else g
    (got,) = torch.autograd.grad(loss, leaf, up)
    args = (kw.get("alpha", 1.0), kw.get("temperature", 1.0), kw.get("tail", False), kw.get("reduction", "mean"))
    want, d, err, size = distill64(z, index, logprob, targets, *args, g=1.0 if g is None else g)
    near(loss.detach(), want, err, "loss")
    # probabilities of two softmaxes and of the slots (k additions), a few products, a rounding to the type
    near(got, d, (2 * prob_tol(V) + (index.shape[-1] + 24) * F32) * size + HALF_STEP[dtype] * d.abs() + 1e-37, "grad")
    with torch.no_grad():
        near(distill_loss(z, index, logprob, targets, **kw), want, err, "loss alone")
    return got


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES + [(2, 2, 70001)], ids=str)
def test_distill(shape, dtype):
    B, T, V = shape
    for n, (layout, k, alpha, tau, tail, reduction) in enumerate([
            ("plain", 1, 1.0, 1.0, False, "mean"), ("shifted", 128, 0.5, 2.0, False, "mean"),
            ("behind", 20, 0.5, 1.0, True, "sum"), ("turned", 7, 0.9, 0.7, True, "none"),
            ("offset", 16, 0.0, 2.0, False, "mean"), ("plain", 33, 1.0, 3.0, True, "mean"),
            ("plain", 0, 0.4, 1.0, False, "mean")]):
        k = min(k, V // 2 if tail else V)
        if tail and k == 0:
            continue
        z = make_logits(B, T, V, dtype, layout, seed=n)
        lead = z.shape[:2]
        index, logprob = teacher(*lead, V, k, seed=n)
        targets = None
        if alpha < 1.0 or n == 0:
            targets = torch.randint(0, V, lead, device=DEV)
            targets[0, 0] = IGNORE
        g = None
        if reduction == "none":
            g = torch.randn(lead, device=DEV)
        elif n == 2:
            g = torch.tensor(-3.7, device=DEV)
        check_distill(z, index, logprob, targets, g, alpha=alpha, temperature=tau, tail=tail, reduction=reduction)


@pytest.mark.parametrize("tail", [False, True], ids=["normalised", "tail"])
@pytest.mark.parametrize("V", [65, 1024, 5003, 40007])
def test_distill_of_empty_repeated_and_masked_slots(V, tail):
    for dtype in (torch.float32, torch.bfloat16):
        z = make_logits(2, 4, V, dtype)
        index, logprob = teacher(2, 4, V, 12)
        index[0, 0, 5:] = -1           # fewer slots
        index[0, 1] = -1               # none at all
        index[0, 2, 3] = index[0, 2, 9]  # a token twice
        index[0, 3, :] = index[0, 3, :1]  # one token in every slot
        logprob[1, 0, 2] = float("-inf")
        targets = torch.randint(0, V, (2, 4), device=DEV)
        targets[1, 1] = index[1, 1, 4]  # the target among the slots
        other = torch.ones(V, dtype=torch.bool, device=DEV)
        other[index[1, 2]] = False
        other[targets[1, 2]] = False
        other[(torch.arange(6, device=DEV) * 7 + 1) % V] = False
        z[1, 2, other] = float("-inf")  # a mask that leaves the slots and a few more
        check_distill(z, index, logprob, targets, alpha=0.6, temperature=1.7, tail=tail)
        check_distill(z, index, logprob, targets, alpha=1.0, tail=tail)


def test_distill_tail_of_students_that_agree_or_disagree():
    """The student's mass outside the slots from all of it down to e^-60, where 1 - sum p has no digit left."""
    for V in (65, 5003, 40007):
        z = make_logits(1, 5, V, torch.float32)
        index, logprob = teacher(1, 5, V, 8)
        for row, add in enumerate([-40.0, 0.0, 10.0, 30.0, 60.0]):
            z[0, row].scatter_add_(0, index[0, row], torch.full((8,), add, device=DEV))
        check_distill(z, index, logprob, None, tail=True)
        check_distill(z, index, logprob, torch.zeros(1, 5, dtype=torch.long, device=DEV), tail=True, alpha=0.5,
                      temperature=0.5)


def test_distill_of_rows_without_mass():
    """p is 0 where every logit, or every logit outside the slots, is -inf."""
    for V in (50, 5003):
        z = make_logits(1, 3, V, torch.float32)
        index, logprob = teacher(1, 3, V, 4)
        z[0, 0] = float("-inf")
        keep = z[0, 1, index[0, 1]].clone()
        z[0, 1] = float("-inf")
        z[0, 1, index[0, 1]] = keep
        for tail in (False, True):
            leaf = z.detach().requires_grad_(True)
            loss = distill_loss(leaf, index, logprob, reduction="none", tail=tail)
            assert torch.isposinf(loss[0, 0]) and torch.isfinite(loss[0, 2])
            assert torch.isposinf(loss[0, 1]) if tail else torch.isfinite(loss[0, 1])
            (got,) = torch.autograd.grad(loss, leaf, torch.ones_like(loss))
            assert torch.isfinite(got).all()
            want = torch.zeros(V, device=DEV).double()
            q = logprob[0, 0].double().exp() if tail else torch.softmax(logprob[0, 0].double(), -1)
            want.scatter_add_(0, index[0, 0], -q)
            near(got[0, 0], want, 1e-6, "empty row")


def test_distill_of_invalid_entries():
    for V in (50, 5003):
        z = make_logits(1, 4, V, torch.float32)
        index, logprob = teacher(1, 4, V, 4)
        targets = torch.randint(0, V, (1, 4), device=DEV)
        index[0, 0, 2] = V
        targets[0, 1] = V + 7
        z[0, 2, 3] = float("nan")
        leaf = z.detach().requires_grad_(True)
        loss = distill_loss(leaf, index, logprob, targets, alpha=0.5, reduction="none")
        assert torch.isnan(loss[0, :3]).all() and torch.isfinite(loss[0, 3])
        (got,) = torch.autograd.grad(loss, leaf, torch.ones_like(loss))
        assert torch.isnan(got[0, :3]).all() and torch.isfinite(got[0, 3]).all()


def test_distill_of_no_rows():
    z = make_logits(2, 3, 700, torch.float32).requires_grad_(True)
    index, logprob = teacher(2, 3, 700, 4)
    none = torch.full((2, 3), IGNORE, device=DEV)
    loss = distill_loss(z, index, logprob, none)
    loss.backward()
    assert float(loss.detach()) == 0.0 and not z.grad.any()
    assert float(distill_loss(z.detach()[:0], index[:0], logprob[:0])) == 0.0
    assert distill_loss(z.detach()[:0], index[:0], logprob[:0], reduction="none").shape == (0, 3)


def test_distill_upstream_gradients_and_second_backward():
    for V in (65, 3001):
        z = make_logits(2, 3, V, torch.bfloat16).requires_grad_(True)
        index, logprob = teacher(2, 3, V, 6)
        loss = distill_loss(z, index, logprob)
        (one,) = torch.autograd.grad(loss, z, retain_graph=True)
        kept = one.clone()
        (three,) = torch.autograd.grad(loss * 3.0, z, retain_graph=True)
        (again,) = torch.autograd.grad(loss, z)
        assert torch.equal(one, kept) and torch.equal(again, kept) and one.data_ptr() != again.data_ptr()
        check_distill(z.detach(), index, logprob, None, torch.tensor(3.0, device=DEV))
        _, d, _, size = distill64(z.detach(), index, logprob, None, 1.0, 1.0, False, "mean", g=3.0)
        near(three, d, (2 * prob_tol(V) + 40 * F32) * size + 2.0 ** -8 * d.abs(), "three")
    with pytest.raises(RuntimeError):
        z2 = z.detach().requires_grad_(True)
        loss = distill_loss(z2 * 1.0, index, logprob)
        (g1,) = torch.autograd.grad(loss, z2, create_graph=True)
        g1.sum().backward()


def test_teacher_scores_feed_the_student():
    """score -> distill: the alternatives of one model, padding included, are the slots of the other."""
    for V, k in ((65, 10), (9001, 40)):
        tz, sz = make_logits(2, 6, V, torch.bfloat16, seed=3), make_logits(2, 6, V, torch.float32, seed=4)
        tokens = torch.randint(0, V, (2, 6), device=DEV)
        tokens[:, 4:] = IGNORE
        top = token_logprobs(tz, tokens, k, temperature=2.0)
        assert (top.top_index[:, 4:] == -1).all()
        got = check_distill(sz, top.top_index, top.top_logprob, tokens, alpha=0.8, temperature=2.0, tail=True)
        assert not got[:, 4:].any()
        # a student equal to its teacher has nothing to learn: KL and gradient vanish
        same = token_logprobs(sz, None, k)
        z = sz.detach().requires_grad_(True)
        loss = distill_loss(z, same.top_index, same.top_logprob, tail=True)
        loss.backward()
        assert abs(float(loss.detach())) < 4 * sum_tol(V) * 12
        assert z.grad.abs().max() < 4 * prob_tol(V)


def test_other_stream_and_captured_calls():
    V = 5003
    z = make_logits(2, 3, V, torch.float32).requires_grad_(True)
    index, logprob = teacher(2, 3, V, 6)
    tokens = torch.randint(0, V, (2, 3), device=DEV)
    tokens[1, 1] = IGNORE

    def step():
        r = token_logprobs(z, tokens, 4)
        loss = distill_loss(z, index, logprob, tokens, alpha=0.5) - r.logprob.sum() + r.entropy.sum()
        (g,) = torch.autograd.grad(loss, z)
        return loss.detach(), g, r.top_index

    want = step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    old = z.detach().clone()
    with torch.no_grad():
        z.copy_(torch.roll(old, 1, -1))
    new = step()
    for graph, out in graphs * 2:
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(new, out):
            assert torch.equal(a, b)
    with torch.no_grad():
        z.copy_(old)
    for graph, out in graphs:
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(want, out):
            assert torch.equal(a, b)


def test_kernels_of_the_library_run():
    z = make_logits(1, 2, 3000, torch.float32)
    n = _lib.kernel_launches()
    token_logprobs(z, None, 2)
    assert _lib.kernel_launches() == n + 1


def test_long_rows_beyond_32_bit_offsets():
    """Rows behind the 2^31st element of their tensor."""
    free, _ = torch.cuda.mem_get_info()
    V, T = 1 << 20, 2100
    if free < 3 * V * T * 2:
        pytest.skip("not enough memory")
    base = torch.empty(T, V, dtype=torch.bfloat16, device=DEV)
    z = base[-2:]
    z.copy_(make_logits(1, 2, V, torch.bfloat16)[0])
    every = base[None, ::2099]  # rows 0 and 2099
    every[0, 0].fill_(0.25)
    tokens = torch.tensor([[5, V - 1]], device=DEV)
    r = token_logprobs(every, tokens, 20)
    check_scores(every, tokens, 20, 1.0, r)
    index, logprob = teacher(1, 2, V, 20)
    check_distill(every, index, logprob, tokens, alpha=0.5, tail=True)


PINS = ["64,1", "64,8", "128,1", "256,1", "512,1", "128,4", "256,2", "512,16"]


@pytest.mark.parametrize("pin", PINS)
def test_every_plan(pin, monkeypatch):
    """CTAs of every size and clusters of several, whatever the plan would take: rows whose part for a CTA is less than
    a step and more than several, many rows a cluster, ties that run over a list, padding between the rows."""
    monkeypatch.setenv("AIWN_IL_LOGITS", pin)
    few = [(2, 3, 1025), (3, 2, 5003), (1, 3, 40007)]
    many = [(300, 3, 1500), (700, 2, 4099)]
    for dtype in (torch.float32, torch.bfloat16):
        for n, (B, T, V) in enumerate(few + many):
            for layout, k in (("behind", 0), ("offset", 7), ("shifted", 100)):
                z = make_logits(B, T, V, dtype, layout, seed=n)
                tokens = torch.randint(0, V, z.shape[:2], device=DEV)
                tokens[torch.rand(z.shape[:2], device=DEV) < 0.3] = IGNORE
                check_scores(z, tokens, k, 0.8, token_logprobs(z, tokens, k, temperature=0.8))
            for k, alpha, tau, tail in ((33, 0.5, 2.0, False), (20, 1.0, 1.0, True), (100, 0.9, 0.7, True)):
                index, logprob = teacher(*z.shape[:2], V, k, seed=n)
                check_distill(z, index, logprob, tokens, alpha=alpha, temperature=tau, tail=tail)
        for kind in ("neg_inf", "lowest", "all_masked", "equal", "two_values", "rising", "falling", "empty_row"):
            z = mask_(make_logits(4, 3, 9001, dtype, "behind"), kind)
            tokens = torch.randint(0, 9001, (4, 3), device=DEV)
            check_scores(z, tokens, 90, 1.0, token_logprobs(z, tokens, 90))
            if kind in ("all_masked", "equal"):  # a slot that a mask holds at -3e38 would make a loss of 3e38
                index, logprob = teacher(4, 3, 9001, 12)
                check_distill(z, index, logprob, tokens, alpha=0.5, tail=True)
                check_distill(z, index, logprob, tokens, alpha=0.5, temperature=2.0)


@pytest.mark.parametrize("V", [65, 5003, 40007])
def test_results_do_not_change_from_run_to_run(V):
    z = make_logits(6, 5, V, torch.bfloat16).requires_grad_(True)
    index, logprob = teacher(6, 5, V, 30)
    index[0, 0, 7] = index[0, 0, 3]
    tokens = torch.randint(0, V, (6, 5), device=DEV)

    def run():
        r = token_logprobs(z, tokens, 40)
        loss = distill_loss(z, index, logprob, tokens, alpha=0.5, temperature=2.0, tail=True)
        (a,) = torch.autograd.grad([r.logprob, r.entropy, r.top_logprob], z,
                                   [torch.ones_like(t) for t in (r.logprob, r.entropy, r.top_logprob)])
        (b,) = torch.autograd.grad(loss, z)
        return (*(t.detach() for t in r), loss.detach(), a, b)

    first = run()
    for _ in range(4):
        for x, y in zip(first, run()):
            assert torch.equal(x, y)


def test_two_calls_at_once():
    """Calls on two streams share nothing."""
    V = 40007
    sets = []
    for seed in range(2):
        z = make_logits(8, 4, V, torch.float32, seed=seed).requires_grad_(True)
        index, logprob = teacher(8, 4, V, 20, seed=seed)
        sets.append((z, index, logprob))

    def run(z, index, logprob):
        loss = distill_loss(z, index, logprob)
        return (loss.detach(), torch.autograd.grad(loss, z)[0], *token_logprobs(z.detach(), None, 30)[1:])

    want = [run(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        got = []
        for s, args in zip(streams, sets):
            with torch.cuda.stream(s):
                got.append([run(*args) for _ in range(3)])
        torch.cuda.synchronize()
        for w, g in zip(want, got):
            for one in g:
                for x, y in zip(w, one):
                    assert torch.equal(x, y)


def test_extreme_temperatures_and_logits():
    for V in (65, 5003):
        z = make_logits(2, 3, V, torch.float32)
        tokens = torch.randint(0, V, (2, 3), device=DEV)
        hot = token_logprobs(z, tokens, 3, temperature=1e30)
        near(hot.entropy, torch.full((2, 3), V, device=DEV).double().log(), 1e-5, "uniform")
        cold = token_logprobs(z, tokens, 3, temperature=1e-30)
        assert torch.equal(cold.top_logprob[..., 0], torch.zeros(2, 3, device=DEV))
        assert torch.equal(cold.entropy, torch.zeros(2, 3, device=DEV))
        assert torch.equal(cold.top_index, token_logprobs(z, tokens, 3).top_index)
        big = z * 1e7  # maxima beyond 2^22
        r = token_logprobs(big, tokens, 2)
        assert torch.equal(r.top_logprob[..., 0], torch.zeros(2, 3, device=DEV))
        leaf = big.requires_grad_(True)
        best = r.top_index[..., 0]
        loss = distill_loss(leaf, best[..., None], torch.zeros(2, 3, 1, device=DEV))
        loss.backward()
        assert float(loss.detach()) == 0.0 and not leaf.grad.any()


def test_logits_far_from_zero():
    """A constant added to a row changes nothing, up to where it leaves the logits no digits: fp32 logits around 7e5
    (their exponent's whole part has 20 bits) and around -3e6, beyond what is taken against a whole number."""
    for V in (65, 5003):
        for add in (7e5, -3e6):
            z = make_logits(2, 4, V, torch.float32) + add
            tokens = torch.randint(0, V, (2, 4), device=DEV)
            r = token_logprobs(z, tokens, 9)
            check_scores(z, tokens, 9, 1.0, r)
            index, logprob = teacher(2, 4, V, 12)
            for tail in (False, True):
                check_distill(z, index, logprob, tokens, alpha=0.5, temperature=2.0, tail=tail)
                check_distill(z, index, logprob, tokens, alpha=0.5, tail=tail)


def test_logits_that_are_views_of_one_row():
    """Rows of stride 0: one row's logits for every position, its gradient their sum."""
    for V in (65, 5003):
        row = make_logits(1, 1, V, torch.float32)[0, 0].requires_grad_(True)
        z = row.expand(3, 4, V)
        tokens = torch.randint(0, V, (3, 4), device=DEV)
        r = token_logprobs(z, tokens, 2)
        check_scores(z.detach(), tokens, 2, 1.0, type(r)(*(t.detach() for t in r)))
        r.logprob.sum().backward()
        want, size = score_grad64(z.detach(), tokens, 0, 1.0, *(torch.full((3, 4), v, device=DEV) for v in (1.0, 0.0)),
                                  torch.zeros(3, 4, 0, device=DEV))
        near(row.grad, want.sum((0, 1)), ((prob_tol(V) + 30 * F32) * size).sum((0, 1)) + F32 * want.abs().sum((0, 1)), V)


def test_logits_changed_before_the_backward_are_noticed():
    z = make_logits(1, 2, 70, torch.float32).requires_grad_(True)
    index, logprob = teacher(1, 2, 70, 3)
    for f in (lambda x: distill_loss(x, index, logprob), lambda x: token_logprobs(x, None).entropy.sum()):
        x = z * 1.0
        y = f(x)
        x.mul_(2.0)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            y.backward()


@pytest.mark.parametrize("V", [65, 3001])
def test_saved_tensors_that_hooks_replace(V):
    """The backward reads what the hooks unpack, not the memory that the forward read."""
    z = make_logits(2, 3, V + 7, torch.float32)[..., :V]
    index, logprob = teacher(2, 3, V, 6)
    targets = torch.randint(0, V, (3, 2), device=DEV).t()

    def gradients(hooks=None):
        x = z.detach().requires_grad_(True)
        with hooks or contextlib.nullcontext():
            y = x * 1.0
            i, l, t = index.clone(), logprob.clone(), targets.clone()
            a = distill_loss(y, i, l, t, alpha=0.3)
            b = distill_loss(y, i, l, t, alpha=0.3, tail=True, reduction="none")
            s = token_logprobs(y, t, top_k=4)
        if hooks:  # what the forward read holds other values by now
            for old in (y, i, l, t):
                old.detach().data.zero_()
        return torch.autograd.grad(2.0 * a + b.sum() + s.logprob.sum() + s.entropy.sum() + s.top_logprob.sum(), x)[0]

    def strided(t):  # the same values, those of the last dimension apart
        t = t.detach()
        return t if t.dim() == 0 else torch.stack([t, t], -1)[..., 0]

    plain = gradients()
    for hooks in (torch.autograd.graph.save_on_cpu(),
                  torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(), lambda t: t),
                  torch.autograd.graph.saved_tensors_hooks(strided, lambda t: t)):
        assert torch.equal(gradients(hooks), plain)


@pytest.mark.parametrize("V", [65, 1500, 5003])
def test_scores_of_masked_rows_at_extreme_temperatures(V):
    """Rows whose largest logit is 0 and whose mask is -inf, or about the type's lowest value: at small temperatures
    the masked logits' exponents overflow, at large ones only those of -inf do."""
    for dtype in (torch.float32, torch.bfloat16):
        for tau in (2.0 ** -120, 2.0 ** -60, 2.0 ** -28, 2.0 ** -20, 2.0 ** 66, 2.0 ** 70, 2.0 ** 100, 2.0 ** 126):
            for low in (float("-inf"), LOWEST):
                z = make_logits(2, 3, V, dtype)
                z -= z.amax(-1, keepdim=True)
                z[..., 3::2] = low
                z[..., 0], z[..., 1] = 0.0, -tau  # two that count
                tokens = torch.zeros(2, 3, dtype=torch.int64, device=DEV)
                r = token_logprobs(z, tokens, 4, temperature=tau)
                lp, h, index, _ = scores64(z, tokens, 4, tau)
                near(r.logprob, lp, sum_tol(V) + 8 * F32 * 12, "logprob")
                near(r.entropy, h, 4 * sum_tol(V) * (1 + 2 * h) + 8 * F32 * 12, "entropy")
                assert torch.equal(r.top_index, index)


@pytest.mark.parametrize("V", [65, 1500, 5003])
def test_distill_of_masked_rows_at_extreme_temperatures(V):
    """The same rows; the slots are the two tokens that count at every temperature, and an empty one."""
    for dtype in (torch.float32, torch.bfloat16):
        for tau in (2.0 ** -60, 2.0 ** -28, 2.0 ** -20, 2.0 ** 20, 2.0 ** 60):
            for low in (float("-inf"), LOWEST):
                z = make_logits(2, 3, V, dtype)
                z -= z.amax(-1, keepdim=True)
                z[..., 3::2] = low
                z[..., 0], z[..., 1] = 0.0, -min(tau, 1.0)
                index = torch.tensor([1, -1, 0], device=DEV).expand(2, 3, 3)
                logprob = torch.tensor([0.6, 0.5, 0.3], device=DEV).log().expand(2, 3, 3)
                check_distill(z, index, logprob, None, temperature=tau)
                check_distill(z, index, logprob, torch.zeros(2, 3, dtype=torch.int64, device=DEV), alpha=0.5,
                              temperature=tau)
                if tau > 1.0:
                    check_distill(z, index, logprob, None, temperature=tau, tail=True)
