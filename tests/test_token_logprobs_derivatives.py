"""Which derivatives log-probs and entropy of logits have: none of them is dropped without an error."""

import pytest
import torch
import torch.autograd.forward_ad as fw

from verl_b200.utils.kernel import token_logprobs


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
