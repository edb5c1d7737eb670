"""token_logprobs and distill_loss refuse, before anything reaches the device (no GPU needed), calls that would give
wrong results without a word."""
import pytest
import torch
from torch.autograd import forward_ad

from aiwn_b200 import distill_loss, token_logprobs
from aiwn_b200._lib import ILError

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
