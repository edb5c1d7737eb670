"""token_logprobs and distill_loss on the GPU where they once went wrong: logits whose exponents change form on the
way, saved tensors that hooks replace."""
import pytest
import torch

from aiwn_b200 import distill_loss, token_logprobs
from aiwn_b200._lib import ILError
from logits_oracle import F32, distill64, near, prob_tol
from test_scoring_gpu import DEV, check_distill, check_scores, make_logits, teacher

pytestmark = pytest.mark.gpu

# |z| log2(e) / tau is 2^22 here: below, exponents are taken to a whole number, above to the maximum
BORDER = 2.0 ** 22 * 0.6931471805599453


def _around(z, centre, order, tau=1.0):
    """z around centre, less 0 to 15 (of tau) for the rows: the border lies among each row's values, or among their
    largest; order: a row's maxima come early, late or anywhere."""
    z = z.sort(dim=-1, descending=order == "falling").values if order != "any" else z
    return z + (centre - tau * torch.arange(16, device=DEV).view(2, 8, 1))


@pytest.mark.parametrize("order", ["any", "rising", "falling"])
@pytest.mark.parametrize("sign", [1.0, -1.0], ids=["positive", "negative"])
@pytest.mark.parametrize("V", [5003, 20011, 50021])
def test_scores_where_the_exponent_changes_form(V, sign, order):
    for tau in (1.0, 0.5, 2.0, 1e-5):
        z = _around(make_logits(2, 8, V, torch.float32) * tau, sign * BORDER * tau, order, tau)
        tokens = torch.randint(0, V, (2, 8), device=DEV)
        tokens[0] = z[0].argmax(-1)
        check_scores(z, tokens, 9, tau, token_logprobs(z, tokens, 9, temperature=tau))


@pytest.mark.parametrize("order", ["any", "rising", "falling"])
@pytest.mark.parametrize("sign", [1.0, -1.0], ids=["positive", "negative"])
@pytest.mark.parametrize("V", [5003, 20011, 50021])
def test_distill_where_the_exponent_changes_form(V, sign, order):
    """At the border of the temperature, and of temperature 1 where both are taken."""
    for tau, centre in ((1.0, BORDER), (2.0, BORDER), (2.0, 2 * BORDER), (0.5, BORDER / 2)):
        z = _around(make_logits(2, 8, V, torch.float32), sign * centre, order)
        tokens = torch.randint(0, V, (2, 8), device=DEV)
        index, logprob = teacher(2, 8, V, 12)
        for tail in (False, True):
            check_distill(z, index, logprob, tokens, alpha=0.5, temperature=tau, tail=tail)
            check_distill(z, index, logprob, None, temperature=tau, tail=tail)


@pytest.mark.parametrize("unpack", [lambda t: t.cpu(), lambda t: t.double() if t.is_floating_point() else t.int(),
                                    lambda t: t[:1] if t.dim() else t], ids=["host", "types", "sizes"])
def test_saved_tensors_that_no_kernel_takes(unpack):
    """A hook's tensors on another device, of another type or size are refused before a launch."""
    z = make_logits(2, 3, 65, torch.float32).requires_grad_(True)
    tokens = torch.zeros(2, 3, dtype=torch.int64, device=DEV)
    index, logprob = teacher(2, 3, 65, 4)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        outs = [token_logprobs(z, tokens, 2).logprob.sum(), distill_loss(z, index, logprob, tokens, alpha=0.5),
                distill_loss(z, index, logprob, reduction="none").sum()]
    for out in outs:
        with pytest.raises(ILError, match="saved tensor"):
            out.backward()


@pytest.mark.parametrize("V", [65, 1024, 5003, 50021])
def test_padded_rows_count_for_nothing_whatever_they_hold(V):
    """NaN and infinite logits, slots beyond the vocabulary and upstream gradients of NaN in rows of padding."""
    z = make_logits(2, 8, V, torch.float32)
    tokens = torch.randint(0, V, (2, 8), device=DEV)
    index, logprob = teacher(2, 8, V, 5)
    pad = torch.zeros(2, 8, dtype=torch.bool, device=DEV)
    pad[0, ::3] = pad[1, 4:] = True
    tokens[pad] = -100
    plain = z.clone().requires_grad_(True)
    dirty = z.clone()
    dirty[pad] = float("nan")
    dirty[1, 5] = float("inf")
    dirty = dirty.requires_grad_(True)
    index2, logprob2 = index.clone(), logprob.clone()
    index2[pad], logprob2[pad] = V + 3, float("nan")
    up = torch.ones(2, 8, device=DEV)
    bad = up.masked_fill(pad, float("nan"))

    def run(x, idx, lp, g):
        r = token_logprobs(x, tokens, 4)
        loss = distill_loss(x, idx, lp, tokens, alpha=0.5, temperature=2.0)
        each = distill_loss(x, idx, lp, tokens, alpha=0.5, reduction="none", tail=True)
        return (*(t.detach() for t in r), loss.detach(), each.detach(),
                torch.autograd.grad([r.logprob, r.entropy, r.top_logprob], x, [g, g, g[..., None].expand(2, 8, 4)])[0],
                torch.autograd.grad(loss, x)[0], torch.autograd.grad(each, x, g)[0])

    for a, b in zip(run(plain, index, logprob, up), run(dirty, index2, logprob2, bad)):
        assert torch.equal(a, b)
        if a.dim() and a.dtype != torch.int64:
            assert not torch.nan_to_num(a[pad], neginf=0.0).any()


@pytest.mark.parametrize("V,k,low", [(V, k, low) for V, k in [(65, 65), (128, 128), (1000, 128), (5003, 60), (50021, 128)]
                                     for low in (float("-inf"), -3.0e38, -1e9, None) if low is not None or k == V])
def test_distill_tail_where_the_slots_name_all_that_counts(V, k, low):
    """Slots that name the whole vocabulary (None), or all that a mask leaves to teacher and student.  What their fp32 log
    probabilities leave of the mass is rounding, and the student has nothing outside: no bucket to compare it with."""
    z, t = make_logits(4, 8, V, torch.float32, seed=1), make_logits(4, 8, V, torch.float32, seed=2)
    if low is not None:
        gone = torch.ones(V, dtype=torch.bool, device=DEV)
        gone[torch.randperm(V, device=DEV)[:k // 2]] = False
        z[..., gone] = t[..., gone] = low
    for tau in (1.0, 2.0):
        top = token_logprobs(t, None, k, temperature=tau)
        mass = top.top_logprob.double().exp().sum(-1)
        assert mass.max() > 1.0 > mass.min()  # rounded to either side
        leaf = z.clone().requires_grad_(True)
        loss = distill_loss(leaf, top.top_index, top.top_logprob, temperature=tau, tail=True, reduction="none")
        (got,) = torch.autograd.grad(loss, leaf, torch.ones_like(loss))
        want, d, err, size = distill64(z, top.top_index, top.top_logprob, None, 1.0, tau, False, "none")
        # the same but for the slots' sum, which is not 1: a factor of q, and the logarithm of that factor
        off = (mass - 1).abs()
        near(loss.detach(), want, err + 2 * off * (want.abs() + tau ** 2), "loss")
        near(got, d, (2 * prob_tol(V) + (k + 24) * F32 + 2 * off[..., None]) * size + F32 * d.abs() + 1e-37, "grad")


def test_distill_tail_of_mass_that_the_student_masks():
    """More than rounding, where the student has nothing: the divergence is infinite."""
    for V in (65, 5003):
        z = make_logits(1, 2, V, torch.float32)
        index = torch.arange(8, device=DEV).expand(1, 2, 8)
        logprob = torch.full((1, 2, 8), 1 / 8, device=DEV).log()
        logprob[0, 0, 7] -= 0.01  # leaves 1e-3
        z[..., 8:] = float("-inf")
        loss = distill_loss(z, index, logprob, tail=True, reduction="none")
        assert torch.isposinf(loss[0, 0]) and torch.isfinite(loss[0, 1])
