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
The sums are held in 32 bits whatever the logits' type.  Gradients are those of
reverse mode; logits with a forward-mode tangent are refused.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

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
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ILError(f"logits must be [..., V] with V >= 1, got shape {tuple(logits.shape)}")
    _lib.x_dtype_code(logits)
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(logits).tangent is not None:
        raise ILError("logits have a forward-mode tangent: these operators have gradients in reverse mode only")
    V = logits.shape[-1]
    if V > _lib.MAX_VOCAB:
        raise ILError(f"logits: {V} logits a row, at most {_lib.MAX_VOCAB}")
    if V > 1 and logits.stride(-1) != 1:
        logits = logits.contiguous()
    d = logits.dim()
    return logits if d == 3 else logits[None] if d == 2 else logits[None, None] if d == 1 else logits.reshape(1, -1, V)


def _per_row(name, t, lead, rows, dtype, more=0):
    """t, of the leading dimensions `lead` and `more` others, as [B, T, ...] like the rows."""
    if t.dtype != dtype:
        raise ILError(f"{name}: dtype {t.dtype}, expected {dtype}")
    if t.dim() != len(lead) + more or t.shape[:len(lead)] != lead:
        raise ILError(f"{name}: shape {tuple(t.shape)} for logits over {tuple(lead)}")
    if t.device != rows.device:
        raise ILError(f"tensors on different devices: {name} on {t.device}, the logits on {rows.device}")
    return t if len(lead) == 2 else t.reshape(*rows.shape[:2], *t.shape[len(lead):])


def _need_cuda(rows):
    if not rows.is_cuda:
        raise ILError("aiwn_b200 kernels need CUDA tensors; there is no CPU path")


def _gradient_like(rows):
    """Room for the gradient of rows, its rows aligned to 16 bytes as those of the logits are where it can be had by
    padding rows to less than 16 bytes (then the kernels load and store the same 16-byte vectors)."""
    if rows.is_contiguous() and rows.data_ptr() % 16 == 0:
        return torch.empty_like(rows)
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


def _score(rows, tokens, k, temperature, ignore_index, lead, with_stats):
    """(logprob, entropy, top_index, top_logprob) over the leading dimensions `lead`, and stats or None."""
    entropy = torch.empty(lead, dtype=torch.float32, device=rows.device)
    logprob = torch.empty_like(entropy) if tokens is not None else None
    index = torch.empty((*lead, k), dtype=torch.int64, device=rows.device)
    top = entropy.new_empty((*lead, k))
    stats = entropy.new_empty((*lead, 2)) if with_stats else None
    _lib.run_token_logprobs(rows, tokens, ignore_index, temperature, k, logprob, entropy, stats, index, top)
    return logprob, entropy, index, top, stats


# Hooks on saved tensors (save_on_cpu, checkpoints) return others of the same values, maybe with other strides: the
# backward passes make sure of logits of a row side by side and of the rest without gaps.  Others than that, on another
# device, of another type or size, are refused, for the kernels go by the forward's sizes.  Written out, as every
# backward pass comes here: 0.9 us, in a loop over the tensors 2.7 us.
def _like(rows):
    """Of the forward's logits, for `_saved_rows`."""
    return rows.shape, rows.dtype, rows.get_device()


def _replaced():
    return ILError("a hook has replaced a saved tensor by one of another device, type or shape")


def _saved_rows(rows, tokens, like):
    """The logits that a forward saved (tokens: checked too), the number of rows and their device's index."""
    shape, dtype, dev = like
    if rows.shape != shape or rows.dtype is not dtype or rows.get_device() != dev or tokens is not None and (
            tokens.shape != shape[:2] or tokens.dtype is not torch.int64 or tokens.get_device() != dev):
        raise _replaced()
    return rows if shape[2] == 1 or rows.stride()[2] == 1 else rows.contiguous(), shape[0] * shape[1], dev


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, tokens, k, temperature, ignore_index, lead):
        logprob, entropy, index, top, stats = _score(rows, tokens, k, temperature, ignore_index, lead, True)
        ctx.save_for_backward(rows, tokens, entropy, stats, index)
        ctx.opts, ctx.like = (k, temperature, ignore_index), _like(rows)
        ctx.mark_non_differentiable(index)
        ctx.set_materialize_grads(False)
        return logprob, entropy, index, top

    @staticmethod
    def _grad(ctx, g_logprob, g_entropy, _, g_top):
        k, temperature, ignore_index = ctx.opts
        rows, tokens, entropy, stats, index = ctx.saved_tensors
        rows, n, dev = _saved_rows(rows, tokens, ctx.like)
        if (entropy.dtype is not torch.float32 or entropy.numel() != n or entropy.get_device() != dev
                or stats.dtype is not torch.float32 or stats.numel() != 2 * n or stats.get_device() != dev
                or index.dtype is not torch.int64 or index.numel() != k * n or index.get_device() != dev):
            raise _replaced()
        entropy, stats, index = entropy.contiguous(), stats.contiguous(), index.contiguous()
        if g_logprob is None and g_entropy is None and g_top is None:
            return None, None, None, None, None, None
        g_logprob, g_entropy, g_top = (None if g is None else g.contiguous() for g in (g_logprob, g_entropy, g_top))
        d = _gradient_like(rows)
        _lib.run_token_logprobs_backward(rows, tokens, ignore_index, temperature, k, entropy, stats, index, g_logprob,
                                         g_entropy, g_top, d)
        return d, None, None, None, None, None

    _once = staticmethod(torch.autograd.function.once_differentiable(_grad.__func__))

    @staticmethod
    def backward(ctx, *g):
        # once_differentiable only matters, and is only paid for, under create_graph=True
        return _TokenLogprobs._once(ctx, *g) if torch.is_grad_enabled() else _TokenLogprobs._grad(ctx, *g)


def token_logprobs(logits, tokens=None, top_k: int = 0, *, temperature: float = 1.0,
                   ignore_index: int = -100) -> TokenScores:
    """Log probabilities of ``tokens`` [...] (int64) under softmax(logits / temperature) of ``logits`` [..., V], the
    entropy of each row and its ``top_k`` (at most 128) largest alternatives.

    ``tokens=None`` leaves the log probabilities out.  Rows whose token is ``ignore_index`` are padding: log
    probability 0, entropy 0, alternatives -1 at -inf, no gradient.  A row whose logits are all -inf gives log
    probability -inf and entropy 0; a token outside [0, V), a NaN or a +inf logit gives NaN.
    The gradient of the logits is that of all three floating results (not twice differentiable)."""
    rows = _rows(logits)
    lead = logits.shape[:-1]
    temperature, k, ignore_index = _temperature(temperature), int(top_k), int(ignore_index)
    if not 0 <= k <= min(rows.shape[2], _lib.MAX_TOP):
        raise ILError(f"top_k {k}: at most {_lib.MAX_TOP}, and no more than the {rows.shape[2]} logits of a row")
    tok = None if tokens is None else _per_row("tokens", tokens, lead, rows, torch.int64)
    _need_cuda(rows)
    if logits.requires_grad and torch.is_grad_enabled():
        return TokenScores(*_TokenLogprobs.apply(rows, tok, k, temperature, ignore_index, lead))
    return TokenScores(*_score(rows, tok, k, temperature, ignore_index, lead, False)[:4])


class _Distill(torch.autograd.Function):
    """Reductions to one value write the gradient (for an upstream gradient of 1) in the forward's launch; the
    backward's returns at once where that is what it gets, and writes the gradient anew otherwise.  A second backward
    of the same graph gets a tensor of its own.  "none" writes the gradient in the backward."""

    @staticmethod
    def forward(ctx, rows, index, logprob, targets, opts, lead):
        loss, d, ws = _distill(rows, index, logprob, targets, opts, lead, opts[4] != 0)
        ctx.save_for_backward(rows, targets, index, logprob)
        ctx.opts, ctx.d, ctx.ws, ctx.like, ctx.k = opts, d, ws, _like(rows), index.shape[2]
        return loss

    @staticmethod
    def _grad(ctx, g):
        k = ctx.k
        rows, targets, index, logprob = ctx.saved_tensors
        rows, n, dev = _saved_rows(rows, targets, ctx.like)
        if (index.dtype is not torch.int64 or index.numel() != k * n or index.get_device() != dev
                or logprob.dtype is not torch.float32 or logprob.numel() != k * n or logprob.get_device() != dev):
            raise _replaced()
        index, logprob = index.contiguous(), logprob.contiguous()
        d, ctx.d = ctx.d, None
        ready = d is not None
        if not ready:
            d = _gradient_like(rows)
        _lib.run_distill(rows, index, logprob, k, targets, *ctx.opts, None, d, ctx.ws, g.contiguous(), int(ready))
        return d, None, None, None, None, None

    _once = staticmethod(torch.autograd.function.once_differentiable(_grad.__func__))

    @staticmethod
    def backward(ctx, g):
        # once_differentiable only matters, and is only paid for, under create_graph=True
        return _Distill._once(ctx, g) if torch.is_grad_enabled() else _Distill._grad(ctx, g)


def _distill(rows, index, logprob, targets, opts, lead, gradient):
    whole = opts[4] != 0
    loss = torch.empty(() if whole else lead, dtype=torch.float32, device=rows.device)
    ws = None
    if whole:
        ws = torch.empty(_lib.distill_workspace_bytes(loss.numel()), dtype=torch.uint8, device=rows.device)
    d = _gradient_like(rows) if gradient else None
    _lib.run_distill(rows, index, logprob, index.shape[2], targets, *opts, loss, d, ws)
    return loss, d, ws


def distill_loss(logits, top_index, top_logprob, targets=None, *, alpha: float = 1.0, temperature: float = 1.0,
                 tail: bool = False, ignore_index: int = -100, reduction: str = "mean") -> torch.Tensor:
    """alpha * temperature^2 * KL(teacher || softmax(logits / temperature)) + (1 - alpha) * cross-entropy(targets).

    ``top_index`` (int64) and ``top_logprob`` (fp32) [..., k], k <= 128: the teacher's largest log probabilities at the
    same ``temperature``, as ``token_logprobs(teacher_logits, top_k=k, temperature=temperature)`` returns them; a
    negative index is an empty slot, so rows may hold fewer.  With ``tail=False`` they are normalised to sum to one
    (any constant may be added to a row of them); with ``tail=True`` what they leave of the mass is compared with the
    student's mass outside the slots, as one bucket (none where less than 2^-16 is left and the student has nothing
    there: slots of a whole vocabulary, or of all that a mask leaves, whose sum is 1 but for rounding).
    ``targets`` [...] (int64): the hard labels, needed for ``alpha < 1``; rows whose target is ``ignore_index`` are left
    out with either alpha.  ``reduction``: "mean" over the rows that are not left out (0 where there are none), "sum", or
    "none" for the rows' losses [...].

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
    if alpha < 1.0 and targets is None:
        raise ILError(f"alpha {alpha} < 1 needs targets")
    if top_index.dim() != len(lead) + 1 or top_index.shape[-1] > _lib.MAX_TOP:
        raise ILError(f"top_index must be [..., k] with k <= {_lib.MAX_TOP}, got shape {tuple(top_index.shape)}")
    if top_logprob.shape != top_index.shape:
        raise ILError(f"top_logprob: shape {tuple(top_logprob.shape)}, expected {tuple(top_index.shape)}")
    index = _per_row("top_index", top_index, lead, rows, torch.int64, 1).contiguous()
    logprob = _per_row("top_logprob", top_logprob, lead, rows, torch.float32, 1).detach().contiguous()
    tgt = None if targets is None else _per_row("targets", targets, lead, rows, torch.int64)
    opts = (int(ignore_index), alpha, _temperature(temperature), int(bool(tail)), _lib.REDUCTIONS[reduction])
    _need_cuda(rows)
    if logits.requires_grad and torch.is_grad_enabled():
        return _Distill.apply(rows, index, logprob, tgt, opts, lead)
    return _distill(rows, index, logprob, tgt, opts, lead, False)[0]
