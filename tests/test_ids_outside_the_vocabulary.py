"""Ids that logits have no column for, at the callers of the log-probs: alike on the host and on the device."""

import pytest
import torch

from verl_b200.models.generic import _logprob_entropy_from_logits
from verl_b200.ops import audit
from verl_b200.trainer.distillation.losses import DistillationLossConfig, compute_forward_kl_topk


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def dev(request):
    return request.param


@pytest.mark.parametrize("config", [{}, dict(log_prob_min_clamp=None), dict(use_tail_term=True)])
def test_a_teacher_s_ids_that_the_student_does_not_have_do_not_count(dev, config):
    g = torch.Generator().manual_seed(1)
    V, k = 50, 6
    student = torch.randn(2, 3, V, generator=g)
    ids = torch.stack([torch.randperm(V, generator=g)[:k] for _ in range(6)]).view(2, 3, k)
    lps = torch.log_softmax(torch.randn(2, 3, V, generator=g), -1).gather(-1, ids)
    ids[0, 0, 1], ids[0, 1, 0], ids[1, 2, 5] = V, -1, 10**6
    ids[1, 0] = V + 7                                           # none of them is there
    ids, lps = ids.to(dev), lps.to(dev)
    conf = DistillationLossConfig(**config)
    x = student.to(dev).requires_grad_(True)
    out = compute_forward_kl_topk(x, lps, ids, conf)
    weight = torch.linspace(0.5, 1.5, 6, device=dev).view(2, 3)
    (grad,) = torch.autograd.grad((out["distillation_losses"] * weight).sum(), x)
    y = student.double().requires_grad_(True)
    logq, low = torch.log_softmax(y, -1), conf.log_prob_min_clamp
    loss, tm, sm = [], [], []
    for b in range(2):
        for t in range(3):
            keep = [j for j in range(k) if 0 <= int(ids[b, t, j]) < V]
            p, q = lps[b, t, keep].double().cpu(), logq[b, t, ids[b, t, keep].cpu()]
            if low is not None:
                p, q = p.clamp(min=low), q.clamp(min=low)
            tm.append(p.exp().sum())
            sm.append(q.exp().sum())
            kl = (p.exp() * (p - q)).sum()
            if conf.use_tail_term:
                tt, ts = (1 - tm[-1]).clamp(1e-6, 1.0), (1 - sm[-1]).clamp(1e-6, 1.0)
                kl = kl + tt * (tt.log() - ts.log())
            loss.append(kl)
    (want,) = torch.autograd.grad((torch.stack(loss).view(2, 3) * weight.double().cpu()).sum(), y)
    # fp32 sums of six terms below 16, of log-probs that are off by 2^-20 at most
    for got, ref in ((out["distillation_losses"], loss), (out["teacher_mass"], tm), (out["student_mass"], sm)):
        assert (got.double().cpu().view(-1) - torch.stack(ref).detach()).abs().max() < 16 * 2.0**-20
    assert (grad.double().cpu() - want).abs().max() < 16 * 2.0**-20 and (grad[1, 0] == 0).all()
    assert out["student_mass"][1, 0] == 0 and out["teacher_mass"][1, 0] == 0


def test_labels_outside_the_vocabulary_have_no_log_prob(dev):
    g = torch.Generator().manual_seed(2)
    x = torch.randn(4, 30, generator=g).to(dev).requires_grad_(True)
    labels = torch.tensor([3, -100, 30, 29], device=dev)
    lp, ent = _logprob_entropy_from_logits(x, labels)
    (grad,) = torch.autograd.grad(lp.sum(), x)
    ref = torch.log_softmax(x.detach().double().cpu(), -1)
    assert lp[1] == 0 and lp[2] == 0 and (grad[1:3] == 0).all() and (grad[[0, 3]] != 0).all()
    assert abs(float(lp[0]) - float(ref[0, 3])) < 2.0**-18 and abs(float(lp[3]) - float(ref[3, 29])) < 2.0**-18
    assert (ent.double().cpu() + (ref.exp() * ref).sum(-1)).abs().max() < 2.0**-18
    with audit.scope(), pytest.raises(audit.AuditError, match="labels"):
        _logprob_entropy_from_logits(x, labels)
