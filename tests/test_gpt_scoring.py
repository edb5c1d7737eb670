"""IndexedGPT.score, IndexedGPT.distill and the distilling GraphedTrainStep:
the operators on logits as a teacher and its student run them together."""
import pytest
import torch

from aiwn_b200 import distill_loss, token_logprobs
from aiwn_b200.gpt import GraphedTrainStep, IndexedGPT
from logits_oracle import F32, IGNORE, distill64, near, prob_tol

DEV = "cuda"
CFG = dict(vocab_size=65, block_size=24, n_layer=2, n_head=4, n_embd=64, K=16, dropout=0.0)


def _models(n):
    out = []
    for seed in range(n):
        torch.manual_seed(seed)
        m = IndexedGPT(**CFG)
        for p in m.parameters():  # larger than the initialisation, so that its distributions are not all alike
            p.data.mul_(3.0)
        out.append(m.to(DEV))
    return out


def _batch(B=3):
    torch.manual_seed(7)
    x = torch.randint(0, CFG["vocab_size"], (B, CFG["block_size"]), device=DEV)
    return x, torch.randint(0, CFG["vocab_size"], x.shape, device=DEV)


@pytest.mark.gpu
def test_score_is_the_cross_entropy_of_forward():
    m, = _models(1)
    x, y = _batch()
    logits, loss = m(x, y)
    s = m.score(x, y, 5)
    # two fp32 means of the same 72 values of size ~4
    assert abs(float(-s.logprob.mean() - loss)) < 1e-5
    torch.testing.assert_close(s.top_logprob[..., 0], logits.log_softmax(-1).amax(-1), rtol=0, atol=1e-5)
    g1 = torch.autograd.grad(loss, m.lm_head.weight, retain_graph=True)[0]
    g2 = torch.autograd.grad(-s.logprob.mean(), m.lm_head.weight)[0]
    torch.testing.assert_close(g1, g2, rtol=1e-4, atol=1e-6)
    for a, b in zip(s, token_logprobs(logits, y, 5)):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_distill_gradients_reach_the_parameters():
    teacher, student = _models(2)
    x, y = _batch()
    y[1, 10:] = IGNORE
    with torch.no_grad():
        s = teacher.score(x, None, 8, temperature=2.0)
    opts = dict(alpha=0.7, temperature=2.0, tail=True)
    logits, loss = student.distill(x, s.top_index, s.top_logprob, y, **opts)
    assert torch.equal(loss, distill_loss(logits, s.top_index, s.top_logprob, y, **opts))
    loss.backward()
    want, d, err, size = distill64(logits.detach(), s.top_index, s.top_logprob, y, 0.7, 2.0, True, "mean")
    near(loss.detach(), want, err, "loss")
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in student.parameters())
    # lm_head.weight's gradient is the logits' times the hidden states
    h = {}
    hook = student.lm_head.register_forward_pre_hook(lambda _, a: h.setdefault("x", a[0].detach()))
    student(x)
    hook.remove()
    hid = h["x"].double().reshape(-1, student.d_idx)
    by_hand = d.reshape(-1, CFG["vocab_size"]).t() @ hid
    # every product with the logits' gradient's error, and a sum over 72 rows in fp32
    tol = ((2 * prob_tol(65) + 60 * F32) * size.reshape(-1, 65).t() + 90 * F32 * d.abs().reshape(-1, 65).t()) @ hid.abs()
    near(student.lm_head.weight.grad, by_hand, tol + 1e-12, "lm_head.weight")


@pytest.mark.gpu
def test_graphed_distillation_matches_eager_steps():
    teacher, eager, graphed = _models(3)
    graphed.load_state_dict(eager.state_dict())
    opts = dict(alpha=0.5, temperature=2.0)
    opt_e = torch.optim.AdamW(eager.parameters(), lr=1e-3, weight_decay=1e-2)
    opt_g = torch.optim.AdamW(graphed.parameters(), lr=1e-3, weight_decay=1e-2, capturable=True)
    x, y = _batch()
    step = GraphedTrainStep(graphed, opt_g, *x.shape, teacher_k=6, distill=opts)
    for a, b in zip(eager.parameters(), graphed.parameters()):
        assert torch.equal(a, b)  # construction leaves the model as it was
    live = []
    for it in range(3):
        xi, yi = torch.roll(x, it, 1), torch.roll(y, it, 1)
        yi[0, : 4 * it] = IGNORE
        with torch.no_grad():
            s = teacher.score(xi, None, 6, temperature=2.0)
        opt_e.zero_grad()
        _, le = eager.distill(xi, s.top_index, s.top_logprob, yi, **opts)
        le.backward(retain_graph=True)
        live.append(le)  # an eager graph of the same leaves lives on while the captured one is replayed
        torch.nn.utils.clip_grad_norm_(eager.parameters(), 1.0)
        opt_e.step()
        lg = step(xi, yi, s.top_index, s.top_logprob)
        torch.cuda.synchronize()
        # table gradients are sums in atomic order, and Adam's first steps are ~lr sign(g): as the plain step's test
        assert abs(lg.item() - le.item()) <= 1e-3 * abs(le.item())
    with pytest.raises(ValueError):
        step(x, y)


def test_graphed_step_refuses_options_without_teacher():
    m = IndexedGPT(**CFG)
    opt = torch.optim.AdamW(m.parameters())
    with pytest.raises(ValueError):
        GraphedTrainStep(m, opt, 2, 24, distill=dict(alpha=0.5))


def test_graphed_step_refuses_other_alternatives():
    """Before anything is copied or replayed: alternatives that are missing, not asked for or of another number."""
    index, logprob = torch.zeros(2, 24, 6, dtype=torch.long), torch.zeros(2, 24, 6)
    step = GraphedTrainStep.__new__(GraphedTrainStep)
    step.top_index, step.top_logprob = index, logprob
    for given in ((None, None), (index, None), (None, logprob), (index[..., :1], logprob[..., :1]),
                  (index[:1], logprob[:1]), (index, logprob[..., :1])):
        with pytest.raises(ValueError):
            step(index[..., 0], index[..., 0], *given)
    step.top_index = step.top_logprob = None
    for given in ((index, logprob), (index, None), (None, logprob)):
        with pytest.raises(ValueError):
            step(index[..., 0], index[..., 0], *given)
