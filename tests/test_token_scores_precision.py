"""Precision of the scores of logits and of their gradient where the logits are large or one token is all but certain: against 64 bits, with bounds that
grow with the differences between a row's logits and not with the logits themselves."""

import math

import pytest
import torch

from verl_b200.ops import functional as F
from verl_b200.utils.kernel import token_logprobs

U32 = 2.0**-24


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def dev(request):
    return request.param


def decided_rows(T, V, offset, temperature, gen, at):
    """Rows of spread 2 (times the temperature) around an offset; token `at` has 1 - p between about 1e-6 and 1e-2, from row to row."""
    z = torch.randn(T, V, generator=gen) * 2.0
    rest = torch.logsumexp(torch.cat([z[:, :at], z[:, at + 1 :]], 1).double(), 1)
    z[:, at] = (rest + torch.linspace(4.6, 13.8, T)).float()
    return (z * temperature + offset).float()


@pytest.mark.parametrize("V,at", [(32000, 7), (32000, 30011), (1003, 1002)])
@pytest.mark.parametrize("offset,temperature", [(0.0, 1.0), (30.0, 1.0), (1e3, 1.0), (9e4, 1.0), (-1e3, 1.0), (-9e4, 1.0), (0.0, 0.1), (300.0, 0.1)])
def test_gradient_of_decided_tokens_at_any_log_sum_exp(dev, V, at, offset, temperature):
    T = 12
    x = decided_rows(T, V, offset, temperature, torch.Generator().manual_seed(V + at), at).to(dev)
    ids = torch.full((T,), at, device=dev)
    g_lp = torch.linspace(0.5, 1.5, T, device=dev)
    leaf = x.clone().requires_grad_(True)
    lp, ent = token_logprobs(leaf, ids, temperature)
    (grad,) = torch.autograd.grad(lp, leaf, g_lp)
    out = F.token_scores(x, ids, 0, temperature)
    by_hand = F.token_scores_bwd(x, ids, out.lse, out.entropy, g_lp, None, temperature)
    z = x.double().cpu() / temperature
    logp = torch.log_softmax(z, -1)
    g = g_lp.double().cpu()[:, None] / temperature
    want = -logp.exp() * g
    q = -torch.expm1(logp[:, at])
    want[:, at] = q * g[:, 0]
    # What the row's sum is off by, in common to all of its tokens: half a step at 16 (2^-21) times log 2 of each of the decided token's two exponents, over
    # its thread's reference and over the row's, 2^-22 of an exponential, U32 of each of at most 16 sums that the decided token's
    # part meets, 4 U32 of the logarithm's part; sums of the other tokens (V / 128 + 40 roundings, their distances' roundings) are off relative to 1 - p.
    # What is added to the decided token's part by itself may be lost under it, value by value: the others of one of 256 threads, of one of 8 lanes on the
    # host, a few times the mean share at most.
    # A token's exponent in base 2 is rounded four times, at most at the row's range R (log2 of e times it); with a temperature its factor as well, twice,
    # and on the host the scaled logit, by its size.
    R = (z.amax(1) - z.amin(1)).max() * math.log2(math.e)
    own = math.log(2) * (4 + 2 * (temperature != 1.0)) * U32 * R + 2.0**-22 + (2 * U32 * float(z.abs().max()) if dev == "cpu" and temperature != 1.0 else 0.0)
    common = 2 * math.log(2) * 2.0**-21 + 2.0**-22 + 20 * U32 + q[:, None] * (U32 * (V / 128 + 40) + own + (1 / 32 if dev == "cuda" else 1 / 2))
    if dev == "cpu" and temperature != 1.0:
        common = common + 2 * U32 * float(z.abs().max())
    # the decided token's own exponent comes from a distance to the reference, at most R, and the reference's whole number: they cancel exactly but for
    # the temperature's factor, under which a logit of size |z| is a product of two numbers that were rounded in 64 bits otherwise
    scaled = 2 * U32 * R if temperature != 1.0 else 0.0
    tol = want.abs() * (own + common + scaled + 2.0**-23)
    tol[:, at] = (g * (common + scaled * q[:, None] * 2 + 2.0**-23))[:, 0]
    for got in (grad, by_hand):
        off = (got.double().cpu() - want).abs()
        assert (off <= tol + 2.0**-126).all(), (off / (tol + 2.0**-126)).max()
        # a row's gradients cancel
        total = got.double().cpu().sum(1).abs()
        assert (total <= g[:, 0] * (common[:, 0] + q * (own + scaled) + 2.0**-23)).all(), (total / g[:, 0]).max()
    assert ((lp.double().cpu() - logp[:, at]).abs() <= common[:, 0] + q * scaled * 2 + 2.0**-23).all()


@pytest.mark.parametrize("offset", [0.0, 1e3, 9e4])
def test_gradient_of_the_entropy_at_any_log_sum_exp(dev, offset):
    T, V = 6, 5003
    gen = torch.Generator().manual_seed(9)
    x = (torch.randn(T, V, generator=gen) * 3 + offset).to(dev)
    ids = torch.randint(0, V, (T,), generator=gen).to(dev)
    leaf = x.clone().requires_grad_(True)
    lp, ent = token_logprobs(leaf, ids)
    (grad,) = torch.autograd.grad(ent.sum(), leaf)
    logp = torch.log_softmax(x.double().cpu(), -1)
    H = -(logp.exp() * logp).sum(-1, keepdim=True)
    want = -logp.exp() * (logp + H)
    R = (x.double().amax(1) - x.double().amin(1)).max().cpu() * math.log2(math.e)
    rel = math.log(2) * 4 * U32 * R + 2.0**-22 + U32 * (V / 128 + 60)
    # p is off by rel; log p + H by the two terms' roundings and by H's own error, log s - w / s with terms up to R
    tol = logp.exp() * (rel * (logp + H).abs() + rel * (2 + R) + 4 * U32 * (logp.abs() + H))
    assert ((grad.double().cpu() - want).abs() <= tol + 2.0**-126).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,lead,at,hole", [
    (32003, 0, 32002, None),      # behind the last vector
    (32001, 1, 0, None),          # in front of the first one
    (32000, 0, 9000, 9001),       # in the vector of a logit of -inf
    (32000, 0, 9000, None), (70000, 0, 65000, None),
])
@pytest.mark.parametrize("big", [30.1, 1003.3, 10007.7, -1500.3])
def test_log_prob_of_a_value_that_is_all_of_its_row(dev, V, lead, at, hole, big, dtype):
    """Whatever its size and place, it is the row's sum: its log-prob is 0 and the entropy too, but for an exponential (2^-22) and the roundings of eight sums."""
    x = torch.full((2, V + lead), big - 5000.0)
    x[:, lead + at] = big
    if hole is not None:
        x[:, lead + hole] = float("-inf")
    x = x.to(dtype).to(dev)[:, lead:]
    out = F.token_scores(x, torch.full((2,), at, device=dev), 3)
    tol = 2.0**-22 + 8 * U32
    assert (out.logprob.abs() <= tol).all() and (out.top_logprob[:, 0].abs() <= tol).all() and (out.top_ids[:, 0] == at).all()
    assert (out.entropy.abs() <= tol).all()
