"""Calls of the C entry points from several host threads at once: the same kernel at different sizes, so that each
call asks for another amount of shared memory."""
import threading

import pytest
import torch

from aiwn_b200 import _lib

pytestmark = pytest.mark.gpu

DEV = "cuda"
CALLS = 1500


def _together(*calls):
    """Runs each call CALLS times in a thread of its own; the statuses that were not IL_OK."""
    start, bad = threading.Barrier(len(calls)), []

    def work(call):
        start.wait()
        for _ in range(CALLS):
            rc = call()
            if rc:
                bad.append(rc)

    threads = [threading.Thread(target=work, args=(c,)) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    return bad


def _check(*makers):
    """Each maker gives (call, outputs): the same outputs from calls at once as from one alone."""
    pairs = [m() for m in makers]
    want = []
    for call, outs in pairs:
        assert call() == 0
        torch.cuda.synchronize()
        want.append([o.clone() for o in outs])
        for o in outs:
            o.zero_()
    torch.cuda.synchronize()
    assert _together(*(call for call, _ in pairs)) == []
    for (_, outs), w in zip(pairs, want):
        for a, b in zip(outs, w):
            assert torch.equal(a, b)


def _distill(V):
    def make():
        lib, s = _lib.load(), torch.cuda.current_stream().cuda_stream
        z = torch.randn(1, 2, V, device=DEV)
        index = torch.randint(0, V, (1, 2, 4), device=DEV)
        logprob = torch.full((1, 2, 4), -2.0, device=DEV)
        loss = torch.zeros(1, 2, device=DEV)
        keep = (z, index, logprob)
        args = (z.data_ptr(), 0, 1, 2, V, 2 * V, V, index.data_ptr(), logprob.data_ptr(), 4, None, 0, 0, -100, 1.0, 1.0, 1,
                0, None, 0, loss.data_ptr(), None, 0, 0, None, 0, s)
        return lambda keep=keep: lib.il_distill(*args), [loss]
    return make


def _scores(V, k):
    def make():
        lib, s = _lib.load(), torch.cuda.current_stream().cuda_stream
        z = torch.randn(1, 2, V, device=DEV)
        entropy, top = torch.zeros(1, 2, device=DEV), torch.zeros(1, 2, k, device=DEV)
        index = torch.zeros(1, 2, k, dtype=torch.int64, device=DEV)
        args = (z.data_ptr(), 0, 1, 2, V, 2 * V, V, None, 0, 0, -100, k, 1.0, None, entropy.data_ptr(), None,
                index.data_ptr(), top.data_ptr(), s)
        return lambda keep=z: lib.il_token_logprobs(*args), [entropy, index, top]
    return make


def test_distill_of_two_vocabularies(monkeypatch):
    monkeypatch.setenv("AIWN_IL_LOGITS", "256,1")
    _check(_distill(5003), _distill(200003), _distill(40007), _distill(1500))


def test_scores_of_two_numbers_of_alternatives(monkeypatch):
    monkeypatch.setenv("AIWN_IL_LOGITS", "256,8")
    _check(_scores(50021, 128), _scores(50021, 8), _scores(9001, 100), _scores(9001, 3))


def _counts(K):
    def make():
        lib, s = _lib.load(), torch.cuda.current_stream().cuda_stream
        x = torch.rand(64, 8, device=DEV) * 2 - 1
        counts = torch.zeros(K, dtype=torch.int64, device=DEV)
        args = (x.data_ptr(), 0, 64, 8, K, 2.0 / K, counts.data_ptr(), s)
        return lambda keep=(x, counts): lib.il_bin_counts(*args), []  # the counts add up
    return make


def _forward(K, IN=20, OUT=20, N=256):
    def make():
        lib, s = _lib.load(), torch.cuda.current_stream().cuda_stream
        x, table = torch.rand(N, IN, device=DEV) * 2 - 1, torch.randn(K, IN, OUT, device=DEV)
        bias, out = torch.zeros(OUT, device=DEV), torch.zeros(N, OUT, device=DEV)
        args = (x.data_ptr(), 0, table.data_ptr(), bias.data_ptr(), out.data_ptr(), N, IN, OUT, K, 2.0 / K, s)
        return lambda keep=(x, table, bias): lib.il_forward(*args), [out]
    return make


def _attention(T, D=8):
    def make():
        lib, s = _lib.load(), torch.cuda.current_stream().cuda_stream
        q, k, v = (torch.randn(1, T, D, device=DEV) for _ in range(3))
        o, lse = torch.zeros(1, T, D, device=DEV), torch.zeros(1, 1, T, device=DEV)
        args = (q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr(), 1, T, 1, D, 0.5, 0.0, None, s)
        return lambda keep=(q, k, v): lib.il_attention_forward(*args), [o, lse]
    return make


def test_bin_counts_of_several_sizes():
    _check(_counts(13000), _counts(16384), _counts(14000), _counts(15000))


@pytest.mark.parametrize("family", ["token", "cluster"])
def test_layers_of_several_sizes(family, monkeypatch):
    monkeypatch.setenv("AIWN_IL_FORWARD", family)
    _check(_forward(512), _forward(64), _forward(256), _forward(16))


def test_attention_of_several_lengths():
    _check(_attention(1024), _attention(800), _attention(900), _attention(820))
