"""aiwn_b200 -- B200-native (sm_100a) IndexedLinear, a drop-in for the
reference package's ``aiwn.layers.indexed_linear`` hot path, and the
operators on logits beside its models (``token_logprobs``, ``distill_loss``)."""
from .layers import GaussianCDFNorm, IndexedLinear, IndexedLinearV2, StandardLinear, indexed_dims, indexed_lr
from .layers.indexed_linear import TRITON_OK, _Fn, triton_available
from .scoring import TokenScores, distill_loss, token_logprobs

__all__ = ["IndexedLinear", "IndexedLinearV2", "GaussianCDFNorm", "StandardLinear", "indexed_dims", "indexed_lr",
           "TRITON_OK", "triton_available", "_Fn", "TokenScores", "token_logprobs", "distill_loss"]
