"""Autograd entry point of the scores of logits: ``(logits, ids) -> (log-probs, entropy)``, differentiable with respect to the logits, which are
read once forward and once backward; no [tokens, vocabulary] tensor is made beside the gradient. For heads whose logits exist (a soft cap
behind the product, a library module); where head and scores can be one step, ``linear_cross_entropy`` never forms them.

Parity target: ``verl/utils/torch_functional.py`` (``logprobs_from_logits``, ``entropy_from_logits``) and the top-k gather of
``verl/trainer/distillation/fsdp/losses.py``.
"""

from __future__ import annotations

import torch

from ...ops import functional as F

__all__ = ["TokenLogprobs", "token_logprobs"]


class _Once(torch.autograd.Function):
    @staticmethod
    def forward(ctx, grad, logits):
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, g):
        raise RuntimeError("token_logprobs can be differentiated once")


class TokenLogprobs(torch.autograd.Function):
    """The form on the host; on a GPU the same function is part of the native library."""

    @staticmethod
    def forward(ctx, logits: torch.Tensor, ids: torch.Tensor, temperature: float, valid_vocab: int):
        out = F.token_scores(logits, ids, 0, temperature, valid_vocab)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(logits, ids, out.lse, out.entropy.clone())
        ctx.meta = (temperature, valid_vocab)
        return out.logprob, out.entropy

    @staticmethod
    def backward(ctx, g_lp, g_ent):
        if g_lp is None and g_ent is None:
            return None, None, None, None
        logits, ids, lse, entropy = ctx.saved_tensors
        if g_lp is None:
            g_lp = torch.zeros(ids.shape, dtype=torch.float32, device=logits.device)
        with torch.no_grad():
            d = F.token_scores_bwd(logits, ids, lse, entropy, g_lp, g_ent, *ctx.meta)
        if torch.is_grad_enabled():   # a graph of the gradient is asked for: an error where it is used
            d = _Once.apply(d, logits)
        return d, None, None, None


def token_logprobs(logits: torch.Tensor, ids: torch.Tensor, temperature: float = 1.0, valid_vocab: int = 0):
    """(log-probs of ``ids``, entropy), fp32, under ``softmax(logits / temperature)``. ``logits`` [..., V]; ``ids`` int64 [...] (one token a row) or
    [..., n] (several: a teacher's support). The first ``valid_vocab`` columns count (0: all); ids outside them have log-prob 0 and no gradient."""
    lead = logits.shape[:-1]
    if ids.shape != lead and ids.shape[:-1] != lead:
        raise ValueError(f"token_logprobs: ids {tuple(ids.shape)} do not fit logits {tuple(logits.shape)}")
    run = F.token_logprobs if logits.is_cuda else TokenLogprobs.apply
    if logits.dim() == 2:
        return run(logits, ids, float(temperature), int(valid_vocab))
    flat = ids.reshape(-1) if ids.shape == lead else ids.reshape(-1, ids.shape[-1])
    lp, ent = run(logits.reshape(-1, logits.shape[-1]), flat, float(temperature), int(valid_vocab))
    return lp.view(ids.shape), ent.view(lead)
