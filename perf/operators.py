"""Operators of a rollout step over a 4-bit cache, as cases: the page bookkeeping in front of the layers, the append to the cache and the
gathering of its rows, the attention over it, and the scores (log-probs of given tokens, entropy, top alternatives) of the logits behind
the layers, for training with their gradient.

``listed()`` names the cases, ``draw(rng)`` gives others of the same ranges, ``prepare`` makes what a user's program has in hand, ``run`` is one
pass (the plain form in elementary torch operations, or the framework's entry points where ``own`` is set), ``work`` is what a pass cannot do
without, ``exact`` the same outputs from the definitions in 64 bits.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False
DEVICE = "cuda"
GROUP = 32    # channels of a head that share a scale and a least value in the cache
PIECE = 64    # tokens of a context that the attention's split counts in
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------ the cases
def listed() -> list[dict]:
    return [
        # one decode step's slot map, contexts and split of the attention, over a full set of sequence slots
        dict(name="maps step", kind="step_maps", slots=320, block=64, most=4096),
        # admission of a wave of prompts: pages from the free list, slots and positions of every prompt token
        dict(name="maps prompts", kind="prompt_maps", rows=512, block=64, most=8192),
        # the token of every sequence of a decode step goes to the cache (and is read back)
        dict(name="cache step", kind="cache", tokens=256, heads=4, dim=128, block=64, dtype="bf16"),
        # a batch of prompts goes to the cache and comes back as the prefix of its next portion
        dict(name="cache prompts", kind="cache", tokens=16384, heads=8, dim=128, block=64, dtype="bf16"),
        # a few short sequences of a small model: latency
        dict(name="attend few", kind="attend", rows=4, heads=14, kv=2, dim=64, block=16, most=160, dtype="bf16"),
        # a full batch of ragged sequences
        dict(name="attend batch", kind="attend", rows=320, heads=28, kv=4, dim=128, block=64, most=4096, dtype="bf16"),
        # one sequence with a long context
        dict(name="attend long", kind="attend", rows=1, heads=32, kv=8, dim=128, block=64, most=131072, dtype="bf16"),
        # a single request's next-token record
        dict(name="scores one row", kind="scores", rows=1, vocab=151936, valid=151936, ids=1, top=5, dtype="bf16", temperature=1.0),
        # the record of a decode step: sampled token, entropy, alternatives
        dict(name="scores step", kind="scores", rows=64, vocab=128256, valid=128256, ids=1, top=20, dtype="fp32", temperature=0.7),
        # a teacher's record of a batch of sequences, of a head with padded rows
        dict(name="scores teacher", kind="scores", rows=2048, vocab=152064, valid=151936, ids=1, top=64, dtype="bf16", temperature=1.0),
        # log-probs and entropy of a policy update, with the gradient of the logits
        dict(name="update", kind="update", rows=2048, vocab=152064, valid=152064, ids=1, dtype="bf16", temperature=1.0),
        # the student's log-probs on a teacher's support, with the gradient of the logits
        dict(name="update support", kind="update", rows=512, vocab=128256, valid=128256, ids=32, dtype="fp32", temperature=1.0),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(["step_maps", "prompt_maps", "cache", "attend", "attend", "attend", "scores", "scores", "update", "update"])
    block = rng.choice([16, 32, 64, 64, 128])
    if kind == "step_maps":
        return dict(kind=kind, slots=_log_int(rng, 1, 1024), block=block, most=_log_int(rng, 64, 16384))
    if kind == "prompt_maps":
        return dict(kind=kind, rows=_log_int(rng, 1, 512), block=block, most=_log_int(rng, 33, 8192))
    dim = rng.choice([64, 128])
    if kind == "cache":
        heads = rng.randint(1, 8)
        return dict(kind=kind, tokens=_log_int(rng, 1, 16384), heads=heads, dim=dim, block=block, dtype=rng.choice(["bf16", "bf16", "fp16"]))
    if kind == "attend":
        kv = rng.choice([1, 2, 4, 8])
        rows = _log_int(rng, 1, 256)
        most = _log_int(rng, 16, max(17, min(131072, 4000000 // (rows * kv))))
        return dict(kind=kind, rows=rows, heads=kv * rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16]), kv=kv, dim=dim, block=block, most=most,
                    dtype=rng.choice(["bf16", "bf16", "fp16"]))
    vocab = _log_int(rng, 200, 152064)
    rows = _log_int(rng, 1, max(1, min(4096, (300 if kind == "scores" else 100) * 1000000 // vocab)))
    case = dict(kind=kind, rows=rows, vocab=vocab, valid=vocab - rng.choice([0, 0, rng.randint(1, 64)]),
                ids=rng.choice([1, 1, rng.randint(2, 64)]), dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                temperature=rng.choice([1.0, round(rng.uniform(0.5, 1.5), 3)]))
    if kind == "scores":
        case["top"] = rng.choice([0, rng.randint(1, 20), rng.randint(21, 128)])
    return case


# ------------------------------------------------------------------------------------------------ inputs
def _lengths(case: dict, n: int) -> np.ndarray:
    """Ragged lengths up to case["most"]: a matter of the case and not of the seed, so that outputs of all seeds have one shape."""
    rs = np.random.RandomState(n * 7919 + case["most"] * 31 + case["block"])
    most = case["most"]
    lens = rs.randint(max(1, most // 4), most + 1, n)
    lens[0] = most
    return lens


def _pages_of(dim: int, block: int) -> int:
    return block * dim + block * dim // 4   # codes of keys and values, then a scale and a least value for each of their groups


def prepare(case: dict, seed: int) -> dict:
    kind = case["kind"]
    g = torch.Generator(device=DEVICE).manual_seed(seed % (1 << 30))
    randn = lambda *s: torch.randn(*s, device=DEVICE, generator=g)
    ints = lambda lo, hi, *s: torch.randint(lo, hi, s, device=DEVICE, generator=g)
    i32 = lambda x: torch.as_tensor(x, dtype=torch.int32, device=DEVICE)
    st = dict(case=case, kind=kind)
    if kind == "step_maps":
        S, width = case["slots"], -(-case["most"] // case["block"])
        st["table"] = torch.randperm(S * width, device=DEVICE, generator=g).view(S, width).to(torch.int32)
        st["pos"] = ints(0, case["most"], S).to(torch.int32)
        st["ctx"] = st["pos"] + 1
        st["active"] = torch.rand(S, device=DEVICE, generator=g) < 0.9
    elif kind == "prompt_maps":
        B, bs = case["rows"], case["block"]
        lens = _lengths(case, B)
        rs = np.random.RandomState(B)
        starts = np.where(rs.rand(B) < 0.25, rs.randint(0, lens), 0)   # a quarter of the rows continue what the cache holds
        width = -(-case["most"] // bs)
        have = -(-starts // bs)
        st.update(starts=i32(starts), ends=i32(lens), have=i32(have), total=int((lens - starts).sum()))
        st["table"] = ints(0, B * width, B + 7, width).to(torch.int32)
        st["rows"] = torch.randperm(B + 7, device=DEVICE, generator=g)[:B].to(torch.int32)
        st["pool"] = torch.randperm(B * width + 5, device=DEVICE, generator=g).to(torch.int32)
    elif kind == "cache":
        T, nkv, hd, bs = case["tokens"], case["heads"], case["dim"], case["block"]
        blocks = -(-T // bs) + 3
        dt = DTYPES[case["dtype"]]
        # the projection's output holds q, k and v side by side: k and v are views with a stride of their own
        qkv = randn(T, 3 * nkv * hd)
        qkv[:, nkv * hd : 2 * nkv * hd] *= torch.exp(randn(nkv * hd))     # some key channels are much larger than others
        st["qkv"] = qkv.to(dt)
        st["slots"] = torch.randperm(blocks * bs, device=DEVICE, generator=g)[:T]
        st["pages"] = torch.zeros(blocks, nkv, _pages_of(hd, bs), dtype=torch.uint8, device=DEVICE)
    elif kind == "attend":
        B, nkv, hd, bs = case["rows"], case["kv"], case["dim"], case["block"]
        lens = _lengths(case, B)
        width = -(-case["most"] // bs)
        per = -(-lens // bs)
        blocks = int(per.sum())
        table = np.zeros((B, width), dtype=np.int64)
        order = np.random.RandomState(seed % (1 << 31)).permutation(blocks)
        at = 0
        for i, n in enumerate(per):
            table[i, :n] = order[at : at + n]
            at += n
        st["table"], st["ctx"] = i32(table), i32(lens)
        st["plan"] = i32(np.concatenate([[0], np.cumsum(-(-lens // PIECE))]))   # made once a step, read by every layer
        pages = torch.randint(0, 256, (blocks, nkv, _pages_of(hd, bs)), dtype=torch.uint8, device=DEVICE, generator=g)
        params = torch.empty(blocks, nkv, 2 * bs * (hd // GROUP), 2, dtype=torch.float16, device=DEVICE)
        scale = torch.rand(params.shape[:-1], device=DEVICE, generator=g) * 0.25 + 0.05
        params[..., 0] = scale
        params[..., 1] = -7.5 * scale + 0.2 * torch.randn(scale.shape, device=DEVICE, generator=g)
        pages[..., bs * hd :] = params.view(blocks, nkv, -1).view(torch.uint8)
        st["pages"] = pages
        st["q"] = randn(B, case["heads"], hd).to(DTYPES[case["dtype"]])
    else:
        T, V = case["rows"], case["vocab"]
        logits = randn(T, V)
        logits *= 2.5
        logits[torch.arange(T, device=DEVICE), ints(0, case["valid"], T)] += 8.0    # most tokens are decided
        st["logits"] = logits.to(DTYPES[case["dtype"]])
        del logits
        n = case["ids"]
        st["ids"] = ints(0, case["valid"], T) if n == 1 else ints(0, case["valid"], T, n)
        if kind == "update":
            st["logits"].requires_grad_(True)
            st["g_lp"] = randn(*st["ids"].shape) / T
            st["g_ent"] = -0.01 * torch.rand(T, device=DEVICE, generator=g) / T
    return st


# ------------------------------------------------------------------------------------------------ one pass
def run(st: dict):
    case, kind = st["case"], st["kind"]
    if own:
        from verl_b200.ops import functional as F
        from verl_b200.utils.kernel import token_logprobs

        if kind == "step_maps":
            return F.decode_slot_map(st["table"], st["pos"], st["ctx"], st["active"], case["block"])
        if kind == "prompt_maps":
            used = F.extend_block_tables_(st["table"], st["rows"], st["have"], st["ends"], st["pool"], case["block"])
            return st["table"], used, *F.build_slot_map(st["table"], st["rows"], st["starts"], st["ends"], case["block"], st["total"])
        if kind == "cache":
            k, v = _key_value(st)
            F.kv4_append_(k, v, st["slots"], st["pages"])
            return F.kv4_gather(st["pages"], st["slots"], case["dim"], st["qkv"].dtype)
        if kind == "attend":
            return F.paged_decode_attention_kv4(st["q"], st["pages"], st["table"], st["ctx"], plan=st["plan"])
        if kind == "scores":
            out = F.token_scores(st["logits"], st["ids"], top_k=case["top"], temperature=case["temperature"], valid_vocab=case["valid"])
            return out.logprob, out.entropy, out.lse, out.top_ids, out.top_logprob
        lp, ent = token_logprobs(st["logits"], st["ids"], temperature=case["temperature"], valid_vocab=case["valid"])
        (grad,) = torch.autograd.grad((lp, ent), st["logits"], (st["g_lp"], st["g_ent"]))
        return lp.detach(), ent.detach(), grad
    if kind == "step_maps":
        return _step_maps(st)
    if kind == "prompt_maps":
        return _prompt_maps(st)
    if kind == "cache":
        return _cache(st)
    if kind == "attend":
        return _attend(st)
    if kind == "scores":
        return _scores(st)
    return _update(st)


def _key_value(st: dict):
    """The keys and the values, as views of the projection's output."""
    case = st["case"]
    n = case["heads"] * case["dim"]
    view = lambda i: st["qkv"][:, i * n : (i + 1) * n].unflatten(1, (case["heads"], case["dim"]))
    return view(1), view(2)


# ---- plain forms
def _step_maps(st: dict):
    bs = st["case"]["block"]
    pos = st["pos"].long()
    block = st["table"].gather(1, (pos // bs)[:, None])[:, 0].long()
    slots = torch.where(st["active"], block * bs + pos % bs, -1)
    ctx = torch.where(st["active"], st["ctx"], 0)
    plan = torch.cat([ctx.new_zeros(1), ((ctx + PIECE - 1) // PIECE).cumsum(0).to(torch.int32)])
    return slots, ctx, plan


def _prompt_maps(st: dict):
    bs = st["case"]["block"]
    table, rows, starts, ends = st["table"], st["rows"].long(), st["starts"].long(), st["ends"].long()
    have = st["have"].long()
    need = (ends + bs - 1) // bs
    new = (need - have).clamp(min=0)
    off = new.cumsum(0) - new
    col = torch.arange(table.shape[1], device=table.device)[None]
    fresh = (col >= have[:, None]) & (col < need[:, None])
    at = (off[:, None] + col - have[:, None]).clamp(0, st["pool"].numel() - 1)
    table[rows] = torch.where(fresh, st["pool"][at], table[rows])
    cu = torch.cat([starts.new_zeros(1), (ends - starts).cumsum(0)])
    t = torch.arange(st["total"], device=table.device)
    seq = torch.searchsorted(cu[1:], t, right=True)
    p = starts[seq] + t - cu[seq]
    slots = table[rows[seq], p // bs].long() * bs + p % bs
    return table, new.sum().to(torch.int32)[None], cu.to(torch.int32), p.to(torch.int32), slots


def _views(pages: torch.Tensor, hd: int, block: int):
    """(key codes, value codes [blocks, heads, block, dim / 2], key parameters, value parameters [blocks, heads, block, groups, 2])."""
    n = block * hd // 2
    codes = lambda a: pages[..., a : a + n].unflatten(-1, (block, hd // 2))
    params = lambda a: pages[..., a : a + n // 4].unflatten(-1, (block, hd // GROUP, 4)).view(torch.float16)
    return codes(0), codes(n), params(2 * n), params(2 * n + n // 4)


def _values(codes: torch.Tensor, params: torch.Tensor) -> torch.Tensor:
    """The numbers that codes [..., dim / 2] with parameters [..., groups, 2] stand for, in fp32."""
    q = torch.stack([codes & 15, codes >> 4], -1).float().flatten(-2).unflatten(-1, (-1, GROUP))
    p = params.float()
    return (q * p[..., :1] + p[..., 1:]).flatten(-2)


def _quantised(x: torch.Tensor):
    """Codes [..., dim / 2] and parameters [..., groups, 2] of x [..., dim]."""
    x = x.float().clamp(-65504.0, 65504.0).unflatten(-1, (-1, GROUP))
    least = x.amin(-1, keepdim=True)
    scale = ((x.amax(-1, keepdim=True) - least) / 15.0).half()
    least = least.half()
    q = torch.where(scale > 0, (x - least.float()) / scale.float(), 0.0).round().clamp(0, 15).to(torch.uint8).flatten(-2)
    return q[..., 0::2] | (q[..., 1::2] << 4), torch.cat([scale, least], -1)


def _cache(st: dict):
    case = st["case"]
    bs, hd = case["block"], case["dim"]
    block, off = st["slots"] // bs, st["slots"] % bs
    kc, vc, kp, vp = _views(st["pages"], hd, bs)
    k, v = _key_value(st)
    kc[block, :, off], kp[block, :, off] = _quantised(k)
    vc[block, :, off], vp[block, :, off] = _quantised(v)
    dt = st["qkv"].dtype
    return _values(kc[block, :, off], kp[block, :, off]).to(dt), _values(vc[block, :, off], vp[block, :, off]).to(dt)


def _attend(st: dict):
    case = st["case"]
    B, nkv, hd, bs = case["rows"], case["kv"], case["dim"], case["block"]
    kc, vc, kp, vp = _views(st["pages"][st["table"].long()], hd, bs)        # [rows, pages, heads, block, ...]
    rows = lambda codes, params: _values(codes, params).transpose(1, 2).reshape(B, nkv, -1, hd)
    q = st["q"].float().view(B, nkv, case["heads"] // nkv, hd)
    s = (q @ rows(kc, kp).transpose(2, 3)) * (1.0 / math.sqrt(hd))
    behind = torch.arange(s.shape[-1], device=DEVICE)[None] >= st["ctx"][:, None]
    s.masked_fill_(behind[:, None, None], float("-inf"))
    p = torch.exp(s - s.amax(-1, keepdim=True))
    out = (p @ rows(vc, vp)) / p.sum(-1, keepdim=True)
    return out.view(B, case["heads"], hd).to(st["q"].dtype)


def _statistics(z: torch.Tensor):
    """(log-sum-exp, entropy, e^(z - lse)) of rows of scaled logits."""
    m = z.amax(-1, keepdim=True)
    e = torch.exp(z - m)
    s = e.sum(-1, keepdim=True)
    lse = m + torch.log(s)
    p = e / s
    return lse, (lse - (p * z).sum(-1, keepdim=True)), p


def _given(z: torch.Tensor, ids: torch.Tensor, lse: torch.Tensor) -> torch.Tensor:
    return (z.gather(1, ids.view(z.shape[0], -1)) - lse).view(ids.shape)


def _scores(st: dict):
    case = st["case"]
    x = st["logits"][:, : case["valid"]].float()
    z = x * (1.0 / case["temperature"])
    lse, ent, _ = _statistics(z)
    # order of the values, ties by place: 32 bits of an order-preserving whole number, then the places backwards
    key = (x + 0.0).view(torch.int32)
    key = torch.where(key < 0, key ^ 0x7FFFFFFF, key).long() << 32
    key += torch.arange(x.shape[1] - 1, -1, -1, device=DEVICE)
    top = x.shape[1] - 1 - (key.topk(case["top"], -1).values & 0xFFFFFFFF)
    return _given(z, st["ids"], lse), ent[:, 0], lse[:, 0], top, z.gather(1, top) - lse


def _update(st: dict):
    case = st["case"]
    V, inv = case["vocab"], 1.0 / case["temperature"]
    x = st["logits"].detach()
    z = x[:, : case["valid"]].float() * inv
    lse, ent, p = _statistics(z)
    lp = _given(z, st["ids"], lse)
    T = z.shape[0]
    g, h = st["g_lp"].view(T, -1), st["g_ent"][:, None]
    d = -p * (g.sum(-1, keepdim=True) + h * (z - lse + ent))
    d.scatter_add_(1, st["ids"].view(T, -1), g)
    grad = torch.zeros(T, V, dtype=x.dtype, device=DEVICE)
    grad[:, : case["valid"]] = d * inv
    return lp, ent[:, 0], grad


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case: dict) -> dict:
    kind = case["kind"]
    if kind == "step_maps":
        return {"bytes": 29.0 * case["slots"], "flops": 0.0}
    if kind == "prompt_maps":
        lens = _lengths(case, case["rows"])
        pages = float((-(-lens // case["block"])).sum())
        return {"bytes": 16.0 * case["rows"] + 12.0 * pages + 12.0 * float(lens.sum()), "flops": 0.0}
    if kind == "cache":
        return {"bytes": case["tokens"] * case["heads"] * case["dim"] * (4.0 + 1.25 + 1.25 + 4.0), "flops": 0.0}
    if kind == "attend":
        tokens = float(_lengths(case, case["rows"]).sum())
        return {"bytes": tokens * case["kv"] * case["dim"] * 1.25 + 4.0 * case["rows"] * case["heads"] * case["dim"],
                "flops": 4.0 * tokens * case["heads"] * case["dim"]}
    size = 4.0 if case["dtype"] == "fp32" else 2.0
    n = float(case["rows"]) * case["valid"] * size
    if kind == "scores":
        return {"bytes": n + case["rows"] * (8.0 + 12.0 * case["ids"] + 12.0 * case["top"]), "flops": 0.0}
    return {"bytes": 2.0 * n + case["rows"] * (8.0 + 20.0 * case["ids"]), "flops": 0.0}


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case: dict, seed: int):
    kind = case["kind"]
    if kind in ("step_maps", "prompt_maps"):
        return None     # whole numbers: equal or wrong
    st = prepare(case, seed)
    with torch.no_grad():
        if kind == "cache":
            return [_rounded_to_codes(x.double()) for x in _key_value(st)]
        return _exact_attend(st) if kind == "attend" else _exact_scores(st)


def _rounded_to_codes(x: torch.Tensor) -> torch.Tensor:
    y = x.reshape(-1, GROUP)
    low, high = y.min(1, keepdim=True).values, y.max(1, keepdim=True).values
    step, low = ((high - low) / 15).to(torch.float16).double(), low.to(torch.float16).double()
    level = torch.round((y - low) / torch.where(step > 0, step, torch.ones_like(step))).clamp(0, 15)     # halves to the even level
    return (low + level * step).view(x.shape)


def _exact_attend(st: dict) -> torch.Tensor:
    case = st["case"]
    hd, bs, nkv = case["dim"], case["block"], case["kv"]
    group = case["heads"] // nkv
    half = bs * hd // 2
    out = torch.zeros(case["rows"], case["heads"], hd, dtype=torch.float64, device=DEVICE)
    for b, n in enumerate(st["ctx"].tolist()):
        used = st["pages"][st["table"][b, : -(-n // bs)].long()].transpose(0, 1).contiguous()          # [heads, pages, bytes]
        numbers = []
        for i in range(2):
            byte = used[:, :, i * half : (i + 1) * half].reshape(nkv, -1, hd // GROUP, GROUP // 2)
            par = used[:, :, 2 * half + i * half // 4 : 2 * half + (i + 1) * half // 4].contiguous().view(torch.float16)
            par = par.reshape(nkv, -1, hd // GROUP, 2).double()
            x = torch.empty(*byte.shape[:-1], GROUP, dtype=torch.float64, device=DEVICE)
            x[..., 0::2], x[..., 1::2] = torch.remainder(byte, 16).double(), torch.div(byte, 16, rounding_mode="floor").double()
            numbers.append((x * par[..., :1] + par[..., 1:]).reshape(nkv, -1, hd)[:, :n])
        k, v = numbers
        q = st["q"][b].double().view(nkv, group, hd)
        w = torch.softmax(torch.einsum("hgd,htd->hgt", q, k) / math.sqrt(hd), -1)
        out[b] = torch.einsum("hgt,htd->hgd", w, v).reshape(-1, hd)
    return out


def _exact_scores(st: dict):
    case = st["case"]
    T, n = case["rows"], case["valid"]
    many = st["ids"].dim() == 2
    parts = []
    for lo in range(0, T, 128):
        z = st["logits"][lo : lo + 128, :n].double() / case["temperature"]
        logp = torch.log_softmax(z, -1)
        p = logp.exp()
        ent = -(p * logp).sum(-1)
        ids = st["ids"][lo : lo + 128].view(z.shape[0], -1)
        lp = logp.gather(1, ids)
        if case["kind"] == "scores":
            parts.append((lp, ent, torch.logsumexp(z, -1), logp.topk(case["top"], -1).values))
            continue
        g, h = st["g_lp"][lo : lo + 128].double().view(z.shape[0], -1), st["g_ent"][lo : lo + 128].double()
        d = -p * g.sum(-1, keepdim=True) - h[:, None] * p * (logp + ent[:, None])
        d.scatter_add_(1, ids, g)
        full = torch.zeros(z.shape[0], case["vocab"], dtype=torch.float64, device=DEVICE)
        full[:, :n] = d / case["temperature"]
        parts.append((lp, ent, full.float() if case["dtype"] == "bf16" else full))
    cols = [torch.cat(c) for c in zip(*parts)]
    lp = cols[0] if many else cols[0][:, 0]
    if case["kind"] == "scores":
        return [lp, cols[1], cols[2], None, cols[3]]
    return [lp, cols[1], cols[2]]
