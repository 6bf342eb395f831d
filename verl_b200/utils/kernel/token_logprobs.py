"""Autograd entry point of the scores of logits: ``(logits, ids) -> (log-probs, entropy)``, differentiable with respect to the logits, which are
read once forward and once backward; no [tokens, vocabulary] tensor is made beside the gradient. For heads whose logits exist (a soft cap
behind the product, a library module); where head and scores can be one step, ``linear_cross_entropy`` never forms them.

Parity target: ``verl/utils/torch_functional.py`` (``logprobs_from_logits``, ``entropy_from_logits``) and the top-k gather of
``verl/trainer/distillation/fsdp/losses.py``.
"""

from __future__ import annotations

import torch

from ...ops import functional as F

__all__ = ["TokenLogprobs", "token_logprobs", "logprobs_of_logits"]


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


# ----------------------------------------------------------------------------------------------- whatever the operator does not do
def _elementary(logits: torch.Tensor, ids: torch.Tensor, entropy: bool = True):
    logp = torch.log_softmax(logits.float(), -1)
    at = ids[..., None] if ids.dim() < logits.dim() else ids
    there = (at >= 0) & (at < logp.shape[-1])
    lp = torch.where(there, logp.gather(-1, torch.where(there, at, 0)), 0.0)
    return lp.view(ids.shape), -(logp.exp() * logp).sum(-1) if entropy else None


class _Scores(torch.autograd.Function):
    """The operator, with the elementary form behind a second derivative."""

    @staticmethod
    def forward(ctx, logits: torch.Tensor, ids: torch.Tensor):
        lp, entropy, lse, stat = F.token_scores_kept(logits, ids)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(logits, ids, lse, entropy, stat)
        return lp, entropy

    @staticmethod
    def backward(ctx, g_lp, g_ent):
        logits, ids, lse, entropy, stat = ctx.saved_tensors
        if g_lp is None and g_ent is None:
            return None, None
        if torch.is_grad_enabled():
            outs, grads = zip(*((o, g) for o, g in zip(_elementary(logits, ids, g_ent is not None), (g_lp, g_ent)) if g is not None))
            return torch.autograd.grad(outs, logits, grads, create_graph=True)[0], None
        if g_lp is None:
            g_lp = torch.zeros(ids.shape, dtype=torch.float32, device=logits.device)
        return F.token_scores_bwd(logits, ids, lse, entropy, g_lp, g_ent, stat=stat), None


def _takes(logits: torch.Tensor, ids: torch.Tensor) -> bool:
    if not logits.is_cuda or logits.dtype not in (torch.float32, torch.bfloat16, torch.float16) or torch._C._are_functorch_transforms_active():
        return False
    if torch.autograd.forward_ad.unpack_dual(logits).tangent is not None:
        return False
    lead = logits.shape[:-1]
    return ids.shape == lead or (ids.shape[:-1] == lead and 0 < ids.shape[-1] <= 4096)


def logprobs_of_logits(logits: torch.Tensor, ids: torch.Tensor, entropy: bool = True):
    """(log-probs of ``ids``, entropy or None), fp32, of ``logits`` [..., V] for code that is written over ``log_softmax`` and ``gather``: by the operator on a GPU,
    and by these where the operator does not go: a second derivative, tangents, transformed functions, 64-bit logits, more than 4096 ids a row, ids of
    fewer rows than the logits have, the host. Ids outside the vocabulary have log-prob 0 and no gradient."""
    if not _takes(logits, ids):
        return _elementary(logits, ids, entropy)
    flat = ids.reshape(-1) if ids.shape == logits.shape[:-1] else ids.reshape(-1, ids.shape[-1])
    lp, ent = _Scores.apply(logits.reshape(-1, logits.shape[-1]), flat)
    return lp.view(ids.shape), ent.view(logits.shape[:-1]) if entropy else None
