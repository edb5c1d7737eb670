"""Operators on a language model's logits, through ``il_token_logprobs`` and ``il_distill``:

* ``token_logprobs`` -- the log probabilities of given tokens, the entropy of
  each position and its largest alternatives, differentiable in all three;
* ``distill_loss`` -- the loss of a student against a teacher's top log
  probabilities (as ``token_logprobs`` returns them), mixed with the hard
  labels' cross-entropy, with its gradient.

The reference has neither: its IndexedGPT returns logits and a mean
cross-entropy (transformer_validation.py:365-370).  ``IndexedGPT.score`` and
``IndexedGPT.distill`` call them on the model's own logits.

Both take fp32 or bf16 CUDA logits [..., V].  Up to two leading dimensions
may have any strides (the shifted view ``logits[:, :-1]`` or a head padded to
a round width, ``logits[..., :V]``, are read in place); more are flattened.
The sums are held in 32 bits whatever the logits' type.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch

from . import _lib
from ._lib import ILError


class TokenScores(NamedTuple):
    """What ``token_logprobs`` returns, over the logits' leading dimensions."""

    logprob: Optional[torch.Tensor]  # [...] fp32, None without tokens
    entropy: torch.Tensor            # [...] fp32, in nats
    top_index: torch.Tensor          # [..., k] int64, largest first, equal logits by index
    top_logprob: torch.Tensor        # [..., k] fp32


def _rows(logits):
    """logits as [B, T, V] rows that the kernels can read, without a copy where the strides allow it."""
    if logits.dim() < 1:
        raise ILError("logits must be [..., V]")
    V = logits.shape[-1]
    if V > 1 and logits.stride(-1) != 1:
        logits = logits.contiguous()
    if logits.dim() == 1:
        return logits[None, None]
    if logits.dim() == 2:
        return logits[None]
    return logits if logits.dim() == 3 else logits.reshape(1, -1, V)


def _per_row(name, t, lead, rows, dtype):
    """t [*lead, ...] as [B, T, ...] like the rows."""
    if t.dtype != dtype:
        raise ILError(f"{name}: dtype {t.dtype}, expected {dtype}")
    if tuple(t.shape[:len(lead)]) != tuple(lead):
        raise ILError(f"{name}: shape {tuple(t.shape)} for logits over {tuple(lead)}")
    return t.reshape(*rows.shape[:2], *t.shape[len(lead):])


def _gradient_like(rows):
    """Room for the gradient of rows, its rows aligned to 16 bytes as those of the logits are where it can be had by
    padding rows to less than 16 bytes (then the kernels load and store the same 16-byte vectors)."""
    B, T, V = rows.shape
    n = 16 // rows.element_size()
    start = rows.data_ptr() // rows.element_size() % n
    st = V + (rows.stride(1) - V) % n
    sb = T * st + (rows.stride(0) - T * st) % n
    buf = torch.empty(start + B * sb + n, dtype=rows.dtype, device=rows.device)
    return buf.as_strided((B, T, V), (sb, st, 1), start)


def _temperature(t):
    t = float(t)
    if not (t > 0.0 and math.isfinite(t)):
        raise ILError(f"temperature {t}: a positive number is needed")
    return t


def _score(rows, tokens, k, temperature, ignore_index, with_stats):
    B, T, V = rows.shape
    if not 0 <= k <= min(V, _lib.MAX_TOP):
        raise ILError(f"top_k {k}: at most {_lib.MAX_TOP}, and no more than the {V} logits of a row")
    new = dict(dtype=torch.float32, device=rows.device)
    logprob = torch.empty(B, T, **new) if tokens is not None else None
    entropy = torch.empty(B, T, **new)
    stats = torch.empty(B, T, 2, **new) if with_stats else None
    index = torch.empty(B, T, k, dtype=torch.int64, device=rows.device)
    top = torch.empty(B, T, k, **new)
    _lib.token_logprobs(rows, tokens, ignore_index, temperature, logprob, entropy, stats, index, top)
    return logprob, entropy, stats, index, top


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, tokens, k, temperature, ignore_index):
        logprob, entropy, stats, index, top = _score(rows, tokens, k, temperature, ignore_index, True)
        ctx.save_for_backward(rows, tokens, entropy, stats, index)
        ctx.temperature, ctx.ignore_index = temperature, ignore_index
        ctx.mark_non_differentiable(index)
        ctx.set_materialize_grads(False)
        return logprob, entropy, index, top

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_logprob, g_entropy, _, g_top):
        rows, tokens, entropy, stats, index = ctx.saved_tensors
        if g_logprob is None and g_entropy is None and g_top is None:
            return None, None, None, None, None
        g_logprob, g_entropy, g_top = (None if g is None else g.contiguous() for g in (g_logprob, g_entropy, g_top))
        d = _gradient_like(rows)
        _lib.token_logprobs_backward(rows, tokens, ctx.ignore_index, ctx.temperature, entropy, stats, index,
                                     g_logprob, g_entropy, g_top, d)
        return d, None, None, None, None


def token_logprobs(logits, tokens=None, top_k: int = 0, *, temperature: float = 1.0,
                   ignore_index: int = -100) -> TokenScores:
    """Log probabilities of ``tokens`` [...] (int64) under softmax(logits / temperature) of ``logits`` [..., V], the
    entropy of each row and its ``top_k`` (at most 128) largest alternatives.

    ``tokens=None`` leaves the log probabilities out.  Rows whose token is ``ignore_index`` are padding: log
    probability 0, entropy 0, alternatives -1 at -inf, no gradient; their logits are not read.  A row whose logits are
    all -inf gives log probability -inf and entropy 0; a token outside [0, V), a NaN or a +inf logit gives NaN.
    The gradient of the logits is that of all three floating results (not twice differentiable)."""
    rows = _rows(logits)
    lead = logits.shape[:-1]
    temperature = _temperature(temperature)
    tok = None if tokens is None else _per_row("tokens", tokens, lead, rows, torch.int64)
    if torch.is_grad_enabled() and logits.requires_grad:
        logprob, entropy, index, top = _TokenLogprobs.apply(rows, tok, int(top_k), temperature, int(ignore_index))
    else:
        logprob, entropy, _, index, top = _score(rows, tok, int(top_k), temperature, int(ignore_index), False)
    return TokenScores(None if logprob is None else logprob.reshape(lead), entropy.reshape(lead),
                       index.reshape(*lead, index.shape[-1]), top.reshape(*lead, top.shape[-1]))


class _Distill(torch.autograd.Function):
    """Reductions to one value write the gradient (for an upstream gradient of 1) in the forward's launch; the
    backward's returns at once where that is what it gets, and writes the gradient anew otherwise.  A second backward
    of the same graph gets a tensor of its own.  "none" writes the gradient in the backward."""

    @staticmethod
    def forward(ctx, rows, index, logprob, targets, opts):
        loss, d, ws = _distill(rows, index, logprob, targets, opts, opts["reduction"] != "none")
        ctx.save_for_backward(rows, index, logprob, targets)
        ctx.opts, ctx.d, ctx.ws = opts, d, ws
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        rows, index, logprob, targets = ctx.saved_tensors
        d, ctx.d = ctx.d, None
        ready = d is not None
        if not ready:
            d = _gradient_like(rows)
        _lib.distill(rows, index, logprob, targets, loss=None, dlogits=d, workspace=ctx.ws, g=g.contiguous(),
                     only_if_not_one=ready, **ctx.opts)
        return d, None, None, None, None


def _distill(rows, index, logprob, targets, opts, gradient):
    B, T, _ = rows.shape
    each = opts["reduction"] == "none"
    loss = torch.empty((B, T) if each else (), dtype=torch.float32, device=rows.device)
    ws = None if each else torch.empty(_lib.distill_workspace_bytes(B * T), dtype=torch.uint8, device=rows.device)
    d = _gradient_like(rows) if gradient else None
    _lib.distill(rows, index, logprob, targets, loss=loss, dlogits=d, workspace=ws, **opts)
    return loss, d, ws


def distill_loss(logits, top_index, top_logprob, targets=None, *, alpha: float = 1.0, temperature: float = 1.0,
                 tail: bool = False, ignore_index: int = -100, reduction: str = "mean") -> torch.Tensor:
    """alpha * temperature^2 * KL(teacher || softmax(logits / temperature)) + (1 - alpha) * cross-entropy(targets).

    ``top_index`` (int64) and ``top_logprob`` (fp32) [..., k], k <= 128: the teacher's largest log probabilities at the
    same ``temperature``, as ``token_logprobs(teacher_logits, top_k=k, temperature=temperature)`` returns them; a
    negative index is an empty slot, so rows may hold fewer.  With ``tail=False`` they are normalised to sum to one
    (any constant may be added to a row of them); with ``tail=True`` what they leave of the mass is compared with the
    student's mass outside the slots, as one bucket.  ``targets`` [...] (int64): the hard labels, needed for
    ``alpha < 1``; rows whose target is ``ignore_index`` are left out with either alpha.  ``reduction``: "mean" over
    the rows that are not left out (0 where there are none), "sum", or "none" for the rows' losses [...].

    For "mean" and "sum" the gradient of logits that need one is written along with the loss, in the logits' type and
    rounded once; call it under ``torch.no_grad()`` where no gradient is wanted.  An upstream gradient other than 1
    (a scaled loss) costs a second pass.  Not twice differentiable; the teacher's values get no gradient."""
    rows = _rows(logits)
    lead = logits.shape[:-1]
    alpha = float(alpha)
    if not 0.0 <= alpha <= 1.0:
        raise ILError(f"alpha {alpha}: between 0 and 1")
    if reduction not in _lib.REDUCTIONS:
        raise ILError(f"reduction {reduction!r}: one of {sorted(_lib.REDUCTIONS)}")
    index = _per_row("top_index", top_index, lead, rows, torch.int64).contiguous()
    logprob = _per_row("top_logprob", top_logprob.detach(), lead, rows, torch.float32).contiguous()
    tgt = None if targets is None else _per_row("targets", targets, lead, rows, torch.int64)
    opts = dict(ignore_index=int(ignore_index), alpha=alpha, temperature=_temperature(temperature), tail=bool(tail),
                reduction=reduction)
    if torch.is_grad_enabled() and logits.requires_grad:
        loss = _Distill.apply(rows, index, logprob, tgt, opts)
    else:
        loss, _, _ = _distill(rows, index, logprob, tgt, opts, False)
    return loss.reshape(lead) if reduction == "none" else loss
