"""Precision of the attention over the 4-bit cache where fp16 operands and long sums could lose it: a token that outweighs all others, and contexts that one
warp works on alone. Against 64 bits, on a GPU."""

import math

import pytest
import torch

from verl_b200.ops import functional as F

pytestmark = pytest.mark.gpu


def pool_of(blocks, nkv, hd, bs, gen):
    """Pages of random codes around zero: scale 0.05 .. 0.3, least value -7.5 scales and some noise."""
    pages = torch.randint(0, 256, (blocks, nkv, F.kv4_page_bytes(bs, hd)), dtype=torch.uint8, device="cuda", generator=gen)
    for lo in range(0, blocks, 4096):
        n = min(4096, blocks - lo)
        par = torch.empty(n, nkv, 2, bs, hd // 32, 2, dtype=torch.float16, device="cuda")
        step = torch.rand(par.shape[:-1], device="cuda", generator=gen) * 0.25 + 0.05
        par[..., 0] = step
        par[..., 1] = -7.5 * step + 0.2 * torch.randn(step.shape, device="cuda", generator=gen)
        pages[lo : lo + n, :, bs * hd :] = par.reshape(n, nkv, -1).view(torch.uint8)
    return pages


def rows_of(pages, hd, bs):
    """Keys and values [2, nkv, tokens, hd] of pages [n, nkv, bytes], in 64 bits."""
    n, nkv = pages.shape[:2]
    code = pages[..., : bs * hd].reshape(n, nkv, 2, bs, hd // 2)
    x = torch.stack([code & 15, code >> 4], -1).view(n, nkv, 2, bs, hd // 32, 32).double()
    par = pages[..., bs * hd :].contiguous().view(torch.float16).view(n, nkv, 2, bs, hd // 32, 2).double()
    return (x * par[..., :1] + par[..., 1:]).permute(2, 1, 0, 3, 4, 5).reshape(2, nkv, n * bs, hd)


def attention(q, pages, hd, bs):
    """Output [heads, hd] and weights [nkv, group, tokens] of one sequence, in 64 bits."""
    k, v = rows_of(pages, hd, bs)
    w = torch.softmax(torch.einsum("hgd,htd->hgt", q.double().view(k.shape[0], -1, hd), k) / math.sqrt(hd), -1)
    return torch.einsum("hgt,htd->hgd", w, v).reshape(-1, hd), w


def beside_rounding(out, want):
    """What an output is off by, of its norm, beside its own rounding: half a step of its type at each value."""
    low, bits = (-126, 8) if out.dtype == torch.bfloat16 else (-14, 11)
    half = torch.exp2(torch.floor(torch.log2(want.abs().clamp(min=2.0**low))) - bits)
    return float(((out.double() - want).abs() - half).clamp(min=0).norm() / want.norm())


# Beside an output's rounding: fp16 roundings of numbers, queries and weights for bf16, together below 2^-10 of the norm; fp32 sums, and for fp16 halves of
# weights that leave at most 2^-22, below 2^-13.
BOUND = {torch.bfloat16: 2.0**-10, torch.float16: 2.0**-13}


def bound_with(up, dtype, want):
    """With a query that has one large channel: for bf16 what that channel adds to a score is a product of two numbers of 11 bits, off by 2^-11 of itself, which
    a weight is then off by. It is `up` for the token that outweighs the others and at most 3 for those (their values of that channel).

    The 63 tokens of its piece have weights in fp16 beside its own 2^8: off by half the least step, 2^-25, or 2^-33 of it, times values of at most 3."""
    mates = 2.0**-33 * math.sqrt(63) * 3 * math.sqrt(want.numel()) / float(want.norm())
    return BOUND[dtype] + (2.0**-11 * (up + 3) if dtype == torch.bfloat16 else 0.0) + mates


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("where", [0, 1, 700, 16383])
@pytest.mark.parametrize("nh,nkv,hd,B", [(8, 2, 64, 1), (8, 2, 128, 200), (24, 2, 64, 200), (16, 1, 128, 1)])
def test_a_token_that_outweighs_all_others(nh, nkv, hd, B, where, dtype):
    """Its value is next to nothing, as that of the first token of many models: the output is what the others leave, whose weights are down to 2^-40 of its.
    Alone, where a warp has few of its tokens, and as many sequences over the same pages, where it has thousands."""
    bs, n = 64, 16384
    gen = torch.Generator(device="cuda").manual_seed(hd + where)
    pages = pool_of(n // bs, nkv, hd, bs, gen)
    q = torch.randn(7, nh, hd, device="cuda", generator=gen)
    q[..., 0] = 8.0
    q[..., 1:] *= torch.tensor([1.0, 1.0, 1.0, 1.0, 1.0, 1.0, 0.05], device="cuda")[:, None, None]
    q = q.to(dtype)
    table = torch.arange(n // bs, device="cuda", dtype=torch.int32).expand(B, -1).contiguous()
    ctx = torch.full((B,), n, dtype=torch.int32, device="cuda")

    def off(q, up):
        want, w = attention(q, pages, hd, bs)
        out = F.paged_decode_attention_kv4(q.expand(B, -1, -1).contiguous(), pages, table, ctx)
        return max(beside_rounding(o, want) for o in out[:: max(1, B // 7)]) <= bound_with(up, dtype, want), w

    for i, up in enumerate((8.0, 11.0, 14.0, 17.0, 20.0, 27.0, 14.0)):      # the token's score
        k = torch.zeros(1, nkv, hd, device="cuda", dtype=torch.float16)
        k[..., 0] = up * math.sqrt(hd) / 8.0
        F.kv4_append_(k, torch.zeros_like(k), torch.full((1,), where, dtype=torch.int64, device="cuda"), pages)
        good, w = off(q[i], up)
        assert good, up
        if up == 20.0:
            assert float(w[..., where].min()) > 0.99
    # the same token twice, the second time with a value: now it is all of the output
    F.kv4_append_(k, torch.ones_like(k), torch.full((1,), (where + 5000) % n, dtype=torch.int64, device="cuda"), pages)
    assert off(q[0], up)[0]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("nh,nkv,hd,n", [(8, 8, 64, 98304), (32, 8, 128, 32768), (20, 2, 128, 98304), (12, 1, 64, 131072), (8, 8, 128, 131071)])
def test_contexts_that_one_warp_works_on_alone(nh, nkv, hd, n, dtype):
    """As many (sequence, head) pairs as there are warps: thousands of tokens are added up in one place, and as their values are of either sign what is left is
    small beside the codes that it comes from. The sequences share their pages, weights are nearly equal."""
    bs = 64
    B = -(-1776 // nkv)
    gen = torch.Generator(device="cuda").manual_seed(hd + n)
    pages = pool_of(-(-n // bs), nkv, hd, bs, gen)
    q = (torch.randn(nh, hd, device="cuda", generator=gen) * 0.05).to(dtype)
    table = torch.randperm(len(pages), device="cuda", generator=gen).to(torch.int32)
    out = F.paged_decode_attention_kv4(q.expand(B, -1, -1).contiguous(), pages, table.expand(B, -1).contiguous(), torch.full((B,), n, dtype=torch.int32, device="cuda"))
    k, v = rows_of(pages[table.long()], hd, bs)
    w = torch.softmax(torch.einsum("hgd,htd->hgt", q.double().view(nkv, -1, hd), k[:, :n]) / math.sqrt(hd), -1)
    want = torch.einsum("hgt,htd->hgd", w, v[:, :n]).reshape(-1, hd)
    off = max(beside_rounding(o, want) for o in out[:: B // 12])
    print(f"beside rounding {off:.2e}")
    assert off <= BOUND[dtype]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", [2.0**18, 2.0**24, 2.0**30, 2.0**40])
def test_scores_whose_steps_are_larger_than_weights_are_apart(size, dtype):
    """Scores up to `size`, where fp32 numbers are up to 2^-6 .. 2^16 apart: one token is all of its row's output, however coarse the distances to it are."""
    nh, nkv, hd, bs, n = 8, 2, 64, 64, 1000
    gen = torch.Generator(device="cuda").manual_seed(11)
    pages = pool_of(-(-n // bs), nkv, hd, bs, gen)
    table = torch.arange(len(pages), device="cuda", dtype=torch.int32).view(1, -1).expand(60, -1).contiguous()
    q = torch.randn(nh, hd, device="cuda", generator=gen).to(dtype)
    k, v = rows_of(pages, hd, bs)
    s = torch.einsum("hgd,htd->hgt", q.double().view(nkv, -1, hd), k[:, :n])
    scale = size / float(s.abs().max())
    first, second = (s * scale).topk(2, -1).values.unbind(-1)
    sure = (first - second > 2.0**-9 * size).flatten()           # what bf16's roundings leave in doubt is left out
    assert sure.sum() >= 2 and float((first - second).min()) > 100
    want = torch.gather(v[:, :n], 1, s.argmax(-1)[..., None].expand(-1, -1, hd)).reshape(nh, hd)
    out = F.paged_decode_attention_kv4(q.expand(60, -1, -1).contiguous(), pages, table, torch.full((60,), n, dtype=torch.int32, device="cuda"), scale=scale)
    assert out.isfinite().all()
    # the value itself: two fp16 numbers of at most 11 bits and a sum for bf16, and the output's rounding
    near = (out.double() - want).abs() <= (2.0**-10 * 5 + 2.0**-8 * want.abs() if dtype == torch.bfloat16 else 2.0**-11 * want.abs() + 2.0**-16)
    assert near[:, sure].all()
