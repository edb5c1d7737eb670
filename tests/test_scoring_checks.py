"""token_logprobs and distill_loss refuse, before anything reaches the device (no GPU needed), calls that would give
wrong results without a word."""
from types import SimpleNamespace

import pytest
import torch
from torch.autograd import forward_ad

from aiwn_b200 import distill_loss, scoring, token_logprobs
from aiwn_b200._lib import ILError
from aiwn_b200.gpt import GraphedTrainStep

B, T, V, K = 2, 3, 40, 4


def test_forward_mode_is_refused():
    """A tangent would be dropped, which forward mode reads as a derivative of zero."""
    for grad in (False, True):
        with forward_ad.dual_level(), torch.set_grad_enabled(grad):
            z = forward_ad.make_dual(torch.randn(B, T, V), torch.randn(B, T, V))
            for logits in (z, z.detach().requires_grad_(True) + z, z[:, :2], z[0], z.transpose(0, 1)):
                lead = logits.shape[:-1]
                with pytest.raises(ILError, match="forward-mode"):
                    token_logprobs(logits, torch.zeros(lead, dtype=torch.long))
                with pytest.raises(ILError, match="forward-mode"):
                    token_logprobs(logits, None, 3)
                with pytest.raises(ILError, match="forward-mode"):
                    distill_loss(logits, torch.zeros(*lead, K, dtype=torch.long), torch.zeros(*lead, K))
            with pytest.raises(ILError, match="CUDA"):  # no tangent: the next check
                token_logprobs(torch.randn(B, T, V), None)


def test_tensors_of_more_dimensions_than_the_rows_are_refused():
    z, tokens = torch.randn(B, T, V), torch.zeros(B, T, dtype=torch.long)
    index, logprob = torch.zeros(B, T, K, dtype=torch.long), torch.zeros(B, T, K)
    for logits, t in ((z, tokens[..., None]), (z, tokens[..., None].expand(B, T, 2)), (z[0], tokens[0][:, None]),
                      (z[0, 0], tokens[0, :1]), (z[None], tokens[None, ..., None])):
        with pytest.raises(ILError, match="shape"):
            token_logprobs(logits, t)
        lead = logits.shape[:-1]
        with pytest.raises(ILError, match="shape"):
            distill_loss(logits, torch.zeros(*lead, K, dtype=torch.long), torch.zeros(*lead, K), t)
    with pytest.raises(ILError, match="shape"):
        distill_loss(z, index[0], logprob[0])
    with pytest.raises(ILError, match="shape"):
        distill_loss(z[0], index, logprob)


class _Ctx:
    """What a backward gets, with saved tensors as a hook may have replaced them."""

    def __init__(self, saved, opts, k=K):
        self.saved_tensors, self.opts, self.k = saved, opts, k
        self.like = scoring._like(torch.empty(B, T, V))
        self.d = self.ws = None


def test_saved_tensors_that_hooks_replace_by_others_are_refused():
    """Hooks may return tensors of another device, type or size: their addresses must not reach a kernel.  All are on the
    CPU here, the forward's and the replaced ones, but for the one on another device."""
    rows, tokens = torch.randn(B, T, V), torch.zeros(B, T, dtype=torch.long)
    per_row, stats = torch.empty(B, T), torch.empty(B, T, 2)
    index, top = torch.zeros(B, T, K, dtype=torch.long), torch.empty(B, T, K)

    scores = (rows, tokens, per_row, stats, index)
    slots = (rows, tokens, index, top)
    like = scoring._like(rows)
    for t in (tokens, None, tokens.t().contiguous().t()):
        got, n, dev = scoring._saved_rows(rows, t, like)
        assert got is rows and n == B * T and dev == -1
    turned = rows.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(scoring._saved_rows(turned, tokens, like)[0], turned)
    assert scoring._saved_rows(turned, tokens, like)[0].is_contiguous()

    for i, other in [(0, rows.bfloat16()), (0, rows[..., :-1]), (0, rows[0]), (0, rows.transpose(0, 1)), (1, tokens.int()),
                     (1, tokens.t()), (1, tokens[:1]), (2, per_row.double()), (2, per_row[:1]), (3, stats[..., :1]),
                     (4, index[..., :1]), (4, index.int())]:
        ctx = _Ctx([other if n == i else t for n, t in enumerate(scores)], (K, 1.0, -100))
        with pytest.raises(ILError, match="saved tensor"):
            scoring._TokenLogprobs._grad(ctx, per_row, None, None, top)
    for i, other in [(0, rows.bfloat16()), (0, rows[:1]), (1, tokens.int()), (1, tokens[..., None]), (2, index.int()),
                     (2, index[:, :1]), (3, top.double()), (3, top[..., :2])]:
        ctx = _Ctx([other if n == i else t for n, t in enumerate(slots)], (-100, 0.5, 1.0, 0, 1))
        with pytest.raises(ILError, match="saved tensor"):
            scoring._Distill._grad(ctx, torch.ones(()))
    for saved, grad in ((scores, lambda c: scoring._TokenLogprobs._grad(c, per_row, None, None, top)),
                        (slots, lambda c: scoring._Distill._grad(c, torch.ones(())))):
        ctx = _Ctx(saved, (K, 1.0, -100))
        ctx.like = (*ctx.like[:2], 0)  # the forward ran on a GPU
        with pytest.raises(ILError, match="saved tensor"):
            grad(ctx)


def test_graphed_step_keeps_nothing_of_the_teachers_graph():
    """A teacher scored with gradients on: copying its log probabilities must not tie the step's buffer to its graph."""
    step = GraphedTrainStep.__new__(GraphedTrainStep)
    step.x, step.y = torch.zeros(B, T, dtype=torch.long), torch.zeros(B, T, dtype=torch.long)
    step.top_index, step.top_logprob = torch.zeros(B, T, K, dtype=torch.long), torch.zeros(B, T, K)
    step.graph, step.loss = SimpleNamespace(replay=lambda: None), torch.zeros(())
    given = torch.randn(B, T, K, requires_grad=True).log_softmax(-1)
    for _ in range(2):
        step(step.x, step.y, torch.ones_like(step.top_index), given)
    assert not step.top_logprob.requires_grad and step.top_logprob.grad_fn is None
    assert torch.equal(step.top_logprob, given.detach()) and step.top_index.all()
