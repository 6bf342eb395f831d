"""Precision of the scores of logits and of their gradient where the logits are large or one token is all but certain: against 64 bits, with bounds that
grow with the differences between a row's logits and not with the logits themselves."""

import pytest
import torch

from verl_b200.ops import functional as F

U32 = 2.0**-24


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def dev(request):
    return request.param


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
