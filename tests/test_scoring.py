"""token_logprobs and distill_loss refuse what their kernels do not take,
before anything reaches the device (no GPU needed), in Python and at the C ABI."""
import ctypes

import pytest
import torch

from aiwn_b200 import _lib, distill_loss, token_logprobs
from aiwn_b200._lib import ILError

B, T, V, K = 2, 3, 40, 4


def _good():
    return (torch.randn(B, T, V), torch.zeros(B, T, dtype=torch.long), torch.zeros(B, T, K, dtype=torch.long),
            torch.zeros(B, T, K))


def test_score_refusals():
    z, tok, _, _ = _good()
    for args, kw, what in [
            ((z.half(), tok), {}, "dtype"), ((z.double(), tok), {}, "dtype"), ((z, tok.int()), {}, "dtype"),
            ((z, tok[:, :2]), {}, "shape"), ((z, tok.reshape(-1)), {}, "shape"), ((z, tok, V + 1), {}, "top_k"),
            ((torch.randn(B, T, 200), tok, 129), {}, "top_k"), ((z, tok, -1), {}, "top_k"),
            ((z, tok), dict(temperature=0.0), "temperature"), ((z, tok), dict(temperature=-1.0), "temperature"),
            ((z, tok), dict(temperature=float("inf")), "temperature"),
            ((z, tok), dict(temperature=float("nan")), "temperature"),
            ((torch.randn(()), None), {}, "logits"), ((torch.randn(2, 0), None), {}, "V"),
            ((z, tok, 2), {}, "CUDA")]:
        with pytest.raises(ILError, match=what):
            token_logprobs(*args, **kw)
    with pytest.raises(ILError, match="at most"):
        token_logprobs(torch.empty(1, 1).expand(1, (1 << 21) + 1).contiguous(), None)


def test_distill_refusals():
    z, tgt, idx, lp = _good()
    for args, kw, what in [
            ((z.half(), idx, lp), {}, "dtype"), ((z, idx.int(), lp), {}, "dtype"), ((z, idx, lp.double()), {}, "dtype"),
            ((z, idx[:, :2], lp), {}, "shape"), ((z, idx, lp[..., :3]), {}, "shape"),
            ((z, idx, lp, tgt.float()), {}, "dtype"), ((z, idx, lp, tgt[:1]), {}, "shape"),
            ((z, idx, lp), dict(alpha=0.5), "targets"), ((z, idx, lp, tgt), dict(alpha=1.5), "alpha"),
            ((z, idx, lp, tgt), dict(alpha=float("nan")), "alpha"), ((z, idx, lp), dict(temperature=0.0), "temperature"),
            ((z, idx, lp), dict(reduction="max"), "reduction"),
            ((z, torch.zeros(B, T, 129, dtype=torch.long), torch.zeros(B, T, 129)), {}, "k <="),
            ((z, idx, lp), {}, "CUDA")]:
        with pytest.raises(ILError, match=what):
            distill_loss(*args, **kw)


def test_binding_refusals():
    z, tok, idx, lp = _good()
    e = torch.empty(B, T)
    with pytest.raises(ILError, match="contiguous"):
        _lib.token_logprobs(z.transpose(1, 2), None, -100, 1.0, None, torch.empty(B, V), None, idx[..., :0], lp[..., :0])
    with pytest.raises(ILError, match="output"):
        _lib.token_logprobs(z, tok, -100, 1.0, None, e, None, idx, lp)
    with pytest.raises(ILError, match="stats"):
        _lib.token_logprobs(z, tok, -100, 1.0, e, e, torch.empty(B, T), idx, lp)
    with pytest.raises(ILError, match="without tokens"):
        _lib.token_logprobs_backward(z, None, -100, 1.0, e, torch.empty(B, T, 2), idx, e, None, None, torch.empty_like(z))
    with pytest.raises(ILError, match="dlogits"):
        _lib.token_logprobs_backward(z, tok, -100, 1.0, e, torch.empty(B, T, 2), idx, e, None, None, z.bfloat16())
    with pytest.raises(ILError, match="uint8"):
        _lib.distill(z, idx, lp, None, -100, 1.0, 1.0, False, "mean", torch.empty(()), None, torch.empty(9))
    with pytest.raises(ILError, match="loss"):
        _lib.distill(z, idx, lp, None, -100, 1.0, 1.0, False, "none", torch.empty(()), None, None)


def test_c_entry_points_check_their_arguments():
    lib = _lib.load()
    p, odd = ctypes.c_void_p(64), ctypes.c_void_p(65)

    def score(z=p, dt=0, b=2, t=3, v=40, tok=p, k=4, tau=1.0, lp=p, ent=p, stats=p, idx=p, top=p):
        return lib.il_token_logprobs(z, dt, b, t, v, 120, 40, tok, 3, 1, -100, k, tau, lp, ent, stats, idx, top, None)

    assert score(b=0) == 0 and score(t=0) == 0
    assert score(dt=7) == 2
    for bad in (dict(b=-1), dict(t=-1), dict(v=0), dict(v=(1 << 21) + 1), dict(k=-1), dict(k=41), dict(v=300, k=129),
                dict(b=1 << 20, t=1 << 20)):
        assert score(**bad) == 1, bad
    for tau in (0.0, -1.0, float("inf"), float("nan"), 1e-300, 1e300):
        assert score(tau=tau) == 9
    for bad in (dict(z=None), dict(ent=None), dict(lp=None), dict(idx=None), dict(top=None)):
        assert score(**bad) == 6, bad
    assert score(z=odd) == 3 and score(stats=ctypes.c_void_p(68)) == 3

    def grad(z=p, k=4, tok=p, ent=p, stats=p, idx=p, g=p, gt=p, d=p, dt=0):
        return lib.il_token_logprobs_backward(z, dt, 2, 3, 40, 120, 40, tok, 3, 1, -100, k, 1.0, ent, stats, idx, g, p,
                                              gt, d, 120, 40, None)

    for bad in (dict(z=None), dict(ent=None), dict(stats=None), dict(d=None), dict(tok=None), dict(idx=None)):
        assert grad(**bad) == 6, bad
    assert grad(d=odd) == 3 and grad(k=129) == 1 and grad(dt=3) == 2

    ws = lib.il_distill_workspace_bytes(6)
    assert ws >= 6 * 4 and lib.il_distill_workspace_bytes(-1) < 0

    def distill(z=p, dt=0, b=2, t=3, v=40, idx=p, lp=p, k=4, tgt=p, alpha=0.5, tau=1.0, red=1, g=None, only=0, loss=p,
                d=p, w=p, n=ws):
        return lib.il_distill(z, dt, b, t, v, 120, 40, idx, lp, k, tgt, 3, 1, -100, alpha, tau, 0, red, g, only, loss, d,
                              120, 40, w, n, None)

    assert distill(dt=9) == 2
    for bad in (dict(b=-1), dict(v=0), dict(k=129), dict(k=-1), dict(red=3), dict(red=-1)):
        assert distill(**bad) == 1, bad
    for bad in (dict(alpha=-0.1), dict(alpha=1.1), dict(alpha=float("nan")), dict(tau=0.0)):
        assert distill(**bad) == 9, bad
    for bad in (dict(z=None), dict(idx=None), dict(lp=None), dict(tgt=None), dict(loss=None, d=None), dict(only=1),
                dict(only=1, g=p, red=0)):
        assert distill(**bad) == 6, bad
    assert distill(w=None) == 5 and distill(n=ws - 1) == 5
    assert distill(z=odd) == 3 and distill(d=odd) == 3 and distill(w=ctypes.c_void_p(72)) == 3
    assert distill(b=0, red=0) == 0


def test_temperature_whose_reciprocal_overflows_is_refused():
    """1 / tau is finite in fp32 and log2(e) / tau is not."""
    lib, p = _lib.load(), ctypes.c_void_p(64)
    for tau in (3e-39, 4.2e-39):
        assert lib.il_token_logprobs(p, 0, 2, 3, 40, 120, 40, p, 3, 1, -100, 4, tau, p, p, p, p, p, None) == 9
