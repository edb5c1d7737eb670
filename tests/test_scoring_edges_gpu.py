"""token_logprobs and distill_loss on the GPU where they once went wrong: logits whose exponents change form on the
way, saved tensors that hooks replace."""
import pytest
import torch

from aiwn_b200 import distill_loss, token_logprobs
from aiwn_b200._lib import ILError
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
