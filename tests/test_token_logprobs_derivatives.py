"""Which derivatives log-probs and entropy of logits have: none of them is dropped without an error."""

import pytest
import torch
import torch.autograd.forward_ad as fw

from verl_b200.models.generic import _logprob_entropy_from_logits
from verl_b200.utils.kernel import logprobs_of_logits, token_logprobs


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def dev(request):
    return request.param


@pytest.mark.parametrize("leaf", [False, True])
def test_tangents_are_refused(dev, leaf):
    x = torch.randn(3, 20, device=dev, requires_grad=leaf)
    ids = torch.zeros(3, dtype=torch.int64, device=dev)
    with fw.dual_level():
        dual = fw.make_dual(x, torch.ones_like(x))
        with pytest.raises((NotImplementedError, RuntimeError)):
            token_logprobs(dual, ids)
        assert token_logprobs(x.detach(), ids)[0].shape == (3,)     # those without one pass
    assert token_logprobs(x, ids)[0].requires_grad == leaf


# ------------------------------------------------------------------------------------------------ callers that were written over log_softmax
def plain(x, ids):
    logp = torch.log_softmax(x, -1)
    return logp.gather(-1, ids[..., None] if ids.dim() < x.dim() else ids).view(ids.shape), -(logp.exp() * logp).sum(-1)


TOL = 64 * 2.0**-24     # sums over 20 columns of numbers below 4, in fp32, a few roundings each


@pytest.mark.parametrize("many", [False, True])
def test_second_derivatives_of_a_library_model_s_log_probs(dev, many):
    g = torch.Generator().manual_seed(4)
    x = torch.randn(3, 20, generator=g).to(dev).requires_grad_(True)
    ids = torch.randint(0, 20, (3, 4) if many else (3,), generator=g).to(dev)
    y = x.detach().double().cpu().requires_grad_(True)
    results = []
    for leaf, f, at in ((x, _logprob_entropy_from_logits if not many else logprobs_of_logits, ids), (y, plain, ids.cpu())):
        for use in ((1, 1), (1, 0), (0, 1)):
            lp, ent = f(leaf, at)
            total = use[0] * lp.square().sum() + use[1] * ent.square().sum() if all(use) else (lp if use[0] else ent).square().sum()
            (first,) = torch.autograd.grad(total, leaf, create_graph=True)
            (second,) = torch.autograd.grad(first.square().sum(), leaf)
            (again,) = torch.autograd.grad(sum(t.sum() for t, u in zip(f(leaf, at), use) if u), leaf)
            results.append((first.detach().double().cpu(), second.double().cpu(), again.double().cpu()))
    n = len(results) // 2
    for got, want in zip(results[:n], results[n:]):
        for a, b in zip(got, want):
            assert (a - b).abs().max() <= TOL * (4 + b.abs().max()) * 4


def test_tangents_and_transformed_functions_of_a_library_model_s_log_probs(dev):
    g = torch.Generator().manual_seed(5)
    x, t = torch.randn(3, 20, generator=g).to(dev), torch.randn(3, 20, generator=g).to(dev)
    ids = torch.randint(0, 20, (3,), generator=g).to(dev)
    with fw.dual_level():
        got = [fw.unpack_dual(o).tangent for o in _logprob_entropy_from_logits(fw.make_dual(x, t), ids)]
    want = torch.autograd.functional.jvp(lambda v: plain(v, ids.cpu()), x.double().cpu(), t.double().cpu())[1]
    assert all((a.double().cpu() - b).abs().max() <= TOL * 16 for a, b in zip(got, want))
    grad = torch.func.grad(lambda v: _logprob_entropy_from_logits(v, ids)[0].sum())(x)
    y = x.double().cpu().requires_grad_(True)
    (want,) = torch.autograd.grad(plain(y, ids.cpu())[0].sum(), y)
    assert (grad.double().cpu() - want).abs().max() <= TOL


@pytest.mark.parametrize("case", ["many ids", "fewer rows", "64 bits", "leading dimensions", "16 bits", "no rows"])
def test_log_probs_of_whatever_gather_takes(dev, case):
    g = torch.Generator().manual_seed(6)
    x = torch.randn(2, 3, 6000, generator=g)
    ids = torch.randint(0, 6000, (2, 3, 5), generator=g)
    if case == "many ids":
        ids = torch.randint(0, 6000, (2, 3, 5000), generator=g)
    if case == "fewer rows":
        ids = ids[:1, :2]
    if case == "leading dimensions":
        ids = ids[..., 0]
    if case == "no rows":
        x, ids = x[:0], ids[:0]
    x = x.to({"64 bits": torch.float64, "16 bits": torch.bfloat16}.get(case, torch.float32))
    leaf = x.to(dev).requires_grad_(True)
    lp, ent = logprobs_of_logits(leaf, ids.to(dev))
    assert lp.shape == ids.shape and ent.shape == x.shape[:-1] and lp.dtype == ent.dtype == torch.float32
    assert logprobs_of_logits(leaf, ids.to(dev), entropy=False)[1] is None
    (grad,) = torch.autograd.grad(lp.sum() + ent.sum(), leaf)
    y = x.double().requires_grad_(True)
    want, ent64 = plain(y, ids)
    (g64,) = torch.autograd.grad(want.sum() + ent64.sum(), y)
    if case != "no rows":
        # sums of 6000 terms in fp32, numbers below 16; gradients below 5 n
        tol = (6000 / 128 + 60) * 2.0**-24 * 16
        assert (lp.double().cpu() - want.detach()).abs().max() <= tol and (ent.double().cpu() - ent64.detach()).abs().max() <= 2 * tol
        step = 2.0**-8 if case == "16 bits" else 0.0
        assert ((grad.double().cpu() - g64).abs() <= step * g64.abs() + 2.0**-24 * ids.shape[-1] * 4 + tol * g64.abs().max()).all()
    assert grad.shape == x.shape and grad.dtype == x.dtype
