"""Page bookkeeping, the 4-bit cache with the attention over it, and the scores of logits, against plain forms in 64 bits: on the host, and
(marked gpu) on the device. Tolerances count the roundings of the kernels: each is written where it is used."""

import math

import numpy as np
import pytest
import torch

from verl_b200.ops import audit
from verl_b200.ops import functional as F
from verl_b200.utils.kernel import token_logprobs

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
U32, U16 = 2.0**-24, 2.0**-11       # half steps of fp32 and fp16
HALF = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}


@pytest.fixture(params=DEVICES)
def dev(request):
    return request.param


def i32(x, dev):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32).to(dev)


# ------------------------------------------------------------------------------------------------ page bookkeeping
def _tables(rs, rows, width, blocks):
    return rs.permutation(max(blocks, rows * width))[: rows * width].reshape(rows, width).astype(np.int32)


@pytest.mark.parametrize("n,bs,most", [(1, 16, 1), (3, 64, 200), (33, 16, 77), (70, 48, 1000), (1500, 64, 300)])
def test_tables_grow_from_the_pool_and_slots_follow_them(dev, n, bs, most):
    rs = np.random.RandomState(n)
    width = -(-most // bs) + 1
    table = rs.randint(0, 9999, (n + 5, width)).astype(np.int32)
    rows = rs.permutation(n + 5)[:n]
    ends = rs.randint(0, most + 1, n)
    starts = np.minimum(rs.randint(0, most + 1, n), ends) * (rs.rand(n) < 0.6)
    have = -(-starts // bs)
    need = -(-ends // bs)
    pool = rs.permutation(int(need.sum()) + 3)
    want = table.copy()
    at = 0
    for r, h, c in zip(rows, have, need):
        want[r, h:c] = pool[at : at + max(c - h, 0)]
        at += max(c - h, 0)
    wide = torch.full((n + 5, width + 3), -7, dtype=torch.int32, device=dev)       # rows that lie further apart than they are long
    t = wide[:, :width]
    t.copy_(torch.from_numpy(table))
    used = F.extend_block_tables_(t, i32(rows, dev), i32(have, dev), i32(ends, dev), i32(pool, dev), bs)
    assert used.tolist() == [at] and np.array_equal(t.cpu().numpy(), want) and bool((wide[:, width:] == -7).all())
    total = int((ends - starts).sum())
    for extra in (0, 5):
        cu, pos, slots = F.build_slot_map(t, i32(rows, dev), i32(starts, dev), i32(ends, dev), bs, total + extra)
        assert cu.tolist() == [0] + np.cumsum(ends - starts).tolist()
        p = np.concatenate([np.arange(a, b) for a, b in zip(starts, ends)]).astype(np.int64)
        r = np.repeat(rows, ends - starts)
        assert np.array_equal(pos.cpu().numpy()[:total], p) and slots.dtype == torch.int64
        assert np.array_equal(slots.cpu().numpy()[:total], want[r, p // bs].astype(np.int64) * bs + p % bs)
        assert pos[total:].tolist() == [0] * extra and slots[total:].tolist() == [-1] * extra
    if total > 1:      # fewer places than tokens: the first ones, and nothing behind them
        cu, pos, slots = F.build_slot_map(t, i32(rows, dev), i32(starts, dev), i32(ends, dev), bs, total - 1)
        assert np.array_equal(pos.cpu().numpy(), p[:-1]) and int(cu[-1]) == total - 1


def test_tables_that_do_not_fit_stay_as_they_were(dev):
    table = torch.arange(12, dtype=torch.int32, device=dev).view(3, 4)
    before = table.clone()
    call = lambda rows, have, ends, pool: F.extend_block_tables_(table, i32(rows, dev), i32(have, dev), i32(ends, dev), i32(pool, dev), 16).tolist()
    assert call([0, 1], [0, 0], [64, 33], [1, 2, 3, 4, 5, 6]) == [-1]       # 7 blocks from a pool of 6
    assert call([0], [0], [65], list(range(9))) == [-1]                     # 5 blocks in a row of 4
    assert call([3], [0], [1], [1]) == [-1] and call([-1], [0], [1], [1]) == [-1] and call([0], [5], [16], [1]) == [-1]
    assert torch.equal(table, before)
    assert call([0], [0], [0], []) == [0] and call([1], [2], [17], [9]) == [0] and torch.equal(table, before)
    none = i32([], dev)
    assert F.extend_block_tables_(table, none, none, none, none, 16).tolist() == [0]
    cu, pos, slots = F.build_slot_map(table, none, none, none, 16, 3)
    assert cu.tolist() == [0] and pos.tolist() == [0, 0, 0] and slots.tolist() == [-1, -1, -1]


def test_tokens_without_a_block_get_no_slot(dev):
    table = i32([[3, -1], [5, 6]], dev)
    cu, pos, slots = F.build_slot_map(table, i32([0, 7, 1], dev), i32([14, 0, 31], dev), i32([18, 2, 34], dev), 16, 9)
    assert slots.tolist() == [62, 63, -1, -1, -1, -1, 111, -1, -1] and pos.tolist() == [14, 15, 16, 17, 0, 1, 31, 32, 33]
    on = torch.tensor([True, True], device=dev)
    for p, want in (([15, 31], [63, 111]), ([16, 32], [-1, -1]), ([-1, 0], [-1, 80])):
        assert F.decode_slot_map(table, i32(p, dev), i32([1, 1], dev), on, 16)[0].tolist() == want


@pytest.mark.parametrize("S,bs", [(1, 16), (5, 64), (33, 48), (1024, 64), (2500, 16)])
def test_decode_step_bookkeeping(dev, S, bs):
    rs = np.random.RandomState(S)
    width = 9
    table = _tables(rs, S, width, 0)
    pos = rs.randint(0, width * bs, S)
    active = rs.rand(S) < 0.7
    slots, ctx, plan = F.decode_slot_map(i32(table, dev), i32(pos, dev), i32(pos + 1, dev), torch.from_numpy(active).to(dev), bs)
    assert np.array_equal(slots.cpu().numpy(), np.where(active, table[np.arange(S), pos // bs].astype(np.int64) * bs + pos % bs, -1))
    c = np.where(active, pos + 1, 0)
    assert np.array_equal(ctx.cpu().numpy(), c) and plan.tolist() == [0] + np.cumsum(-(-c // 64)).tolist()


def test_refusals_of_the_bookkeeping(dev):
    t = torch.zeros(2, 3, dtype=torch.int32, device=dev)
    v = torch.zeros(2, dtype=torch.int32, device=dev)
    on = torch.ones(2, dtype=torch.bool, device=dev)
    for bad in (lambda: F.extend_block_tables_(t.long(), v, v, v, v, 16), lambda: F.extend_block_tables_(t, v, v[:1], v, v, 16),
                lambda: F.build_slot_map(t[0], v, v, v, 16, 0), lambda: F.build_slot_map(t, v, v, v.long(), 16, 0),
                lambda: F.build_slot_map(t, v, v, v, 16, -1), lambda: F.decode_slot_map(t, v[:1], v[:1], on, 16),
                lambda: F.decode_slot_map(t, v, v, on.int(), 16)):
        with pytest.raises(ValueError):
            bad()


# ------------------------------------------------------------------------------------------------ 4-bit cache
def quantised(x):
    """Codes and parameters of x [..., channels] (numpy fp32), every step one rounded fp32 operation."""
    with np.errstate(invalid="ignore", divide="ignore"):
        g = np.clip(x.astype(np.float32), -7600, 7600).reshape(*x.shape[:-1], -1, 32)
        low = g.min(-1, keepdims=True)
        scale = ((g.max(-1, keepdims=True) - low) / np.float32(15)).astype(np.float16)
        low = low.astype(np.float16)
        q = np.rint((g - low.astype(np.float32)) / np.where(scale > 0, scale, 1).astype(np.float32))
        q = np.where(scale > 0, np.clip(q, 0, 15), 0)
    return np.nan_to_num(q).astype(np.uint8), scale, low


def unpacked(pages, bs, hd):
    """(codes [2, blocks, heads, bs, groups, 32], scales, least values) of a pool, from its bytes."""
    raw = pages.cpu().numpy()
    n = bs * hd // 2
    codes, scale, low = [], [], []
    for i in range(2):
        c = raw[..., i * n : (i + 1) * n].reshape(*raw.shape[:2], bs, hd // 2)
        codes.append(np.stack([c & 15, c >> 4], -1).reshape(*raw.shape[:2], bs, hd // 32, 32))
        p = np.ascontiguousarray(raw[..., 2 * n + i * n // 4 : 2 * n + (i + 1) * n // 4]).view(np.float16).reshape(*raw.shape[:2], bs, hd // 32, 2)
        scale.append(p[..., :1])
        low.append(p[..., 1:])
    return np.stack(codes), np.stack(scale), np.stack(low)


def rows_of(pages, bs, hd):
    """Values [2, blocks, heads, bs, channels] of a pool in 64 bits."""
    c, s, m = unpacked(pages, bs, hd)
    return (c.astype(np.float64) * s.astype(np.float64) + m.astype(np.float64)).reshape(*c.shape[:-2], hd)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,nkv,hd,bs", [(1, 1, 64, 16), (7, 2, 128, 64), (33, 3, 32, 16), (100, 4, 96, 48), (257, 8, 128, 128)])
def test_append_and_gather(dev, T, nkv, hd, bs, dtype):
    g = torch.Generator().manual_seed(T)
    blocks = -(-T // bs) + 2
    qkv = torch.randn(T, 3 * nkv * hd, generator=g) * torch.exp(torch.randn(3 * nkv * hd, generator=g))
    qkv[::5] *= 1e-3
    qkv[1::7, : 2 * nkv * hd] = 0.25                      # groups without a spread
    qkv = qkv.to(dtype).to(dev)
    k, v = (qkv[:, i * nkv * hd : (i + 1) * nkv * hd].view(T, nkv, hd) for i in (1, 2))
    slots = torch.randperm(blocks * bs, generator=g)[:T]
    slots[::9] = -1
    pages = torch.full((blocks, nkv, F.kv4_page_bytes(bs, hd)), 0x5A, dtype=torch.uint8, device=dev)
    F.kv4_append_(k, v, slots.to(dev), pages)
    codes, scale, low = unpacked(pages, bs, hd)
    seen = np.zeros((blocks, bs), dtype=bool)
    for x, c, s, m in zip((k, v), codes, scale, low):
        wc, ws, wm = quantised(x.float().cpu().numpy())
        for t, slot in enumerate(slots.tolist()):
            if slot >= 0:
                b, o = divmod(slot, bs)
                seen[b, o] = True
                assert np.array_equal(c[b, :, o], wc[t]) and np.array_equal(s[b, :, o], ws[t]) and np.array_equal(m[b, :, o], wm[t])
    other = ~seen[:, None].repeat(nkv, 1)
    assert (codes[:, other] == np.tile([10, 5], 16)).all() and (np.stack([scale, low])[:, :, other].view(np.uint16) == 0x5A5A).all()
    gk, gv = F.kv4_gather(pages, slots.to(dev), hd, dtype)
    values = rows_of(pages, bs, hd)
    for got, want in zip((gk, gv), values):
        want = np.stack([want[s // bs, :, s % bs] if s >= 0 else np.zeros((nkv, hd)) for s in slots.tolist()])
        off = np.abs(got.double().cpu().numpy() - want)
        assert got.dtype == dtype and (off <= np.abs(want) * (HALF[dtype] + 2 * U32) + 2.0**-24).all()   # one rounding to the type, one in fp32


@pytest.mark.parametrize("T,nkv,bs", [(5001, 16, 48), (9999, 8, 64)])
def test_append_of_many_tokens(dev, T, nkv, bs):
    if dev == "cpu":
        T //= 16
    g = torch.Generator().manual_seed(T)
    k, v = (torch.randn(T, nkv, 128, generator=g).bfloat16().to(dev) for _ in range(2))
    blocks = -(-T // bs) + 1
    slots = torch.randperm(blocks * bs, generator=g)[:T]
    pages = torch.zeros(blocks, nkv, F.kv4_page_bytes(bs, 128), dtype=torch.uint8, device=dev)
    F.kv4_append_(k, v, slots.to(dev), pages)
    b, o = (slots // bs).numpy(), (slots % bs).numpy()
    back = F.kv4_gather(pages, slots.to(dev), 128, torch.float16)
    for x, got, c, s, m in zip((k, v), back, *unpacked(pages, bs, 128)):
        wc, ws, wm = quantised(x.float().cpu().numpy())
        assert np.array_equal(c[b, :, o], wc) and np.array_equal(s[b, :, o], ws) and np.array_equal(m[b, :, o], wm)
        want = (wc * ws.astype(np.float64) + wm).reshape(T, nkv, 128)
        assert (np.abs(got.double().cpu().numpy() - want) <= np.abs(want) * (U16 + 2 * U32) + 2.0**-24).all()   # as above


def test_values_outside_the_range_of_the_cache(dev):
    x = torch.zeros(4, 1, 64, dtype=torch.bfloat16, device=dev)
    x[0, 0, 3], x[1, 0, 40], x[2, 0, 0], x[3, 0, 63] = float("nan"), float("inf"), -1e30, 1e-6
    pages = torch.zeros(1, 1, F.kv4_page_bytes(16, 64), dtype=torch.uint8, device=dev)
    slots = torch.arange(4, device=dev)
    F.kv4_append_(x, x, slots, pages)
    k, v = (t.float().cpu() for t in F.kv4_gather(pages, slots, 64))
    assert torch.equal(k.isnan(), v.isnan()) and k[0, 0, :32].isnan().all() and (k[0, 0, 32:] == 0).all() and not k[1:].isnan().any()
    top = float(torch.tensor(7600.0).bfloat16())
    assert k[1, 0, 40] == pytest.approx(top, rel=2.0**-7) and k[2, 0, 0] == -top and k[3].abs().max() <= 2e-6


def test_refusals_of_the_cache(dev):
    pages = torch.zeros(2, 2, F.kv4_page_bytes(16, 64), dtype=torch.uint8, device=dev)
    k = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device=dev)
    s = torch.arange(3, device=dev)
    for bad in (lambda: F.kv4_page_bytes(16, 48), lambda: F.kv4_page_bytes(24, 64), lambda: F.kv4_page_bytes(2048, 64),
                lambda: F.kv4_append_(k, k[:2], s, pages), lambda: F.kv4_append_(k, k.float(), s, pages), lambda: F.kv4_append_(k[:, :1], k[:, :1], s, pages),
                lambda: F.kv4_append_(k, k, s.int(), pages), lambda: F.kv4_append_(k, k, s[:2], pages), lambda: F.kv4_append_(k, k, s, pages.int()),
                lambda: F.kv4_append_(k, k, s, pages[..., :-4]), lambda: F.kv4_gather(pages, s.int(), 64), lambda: F.kv4_gather(pages, s, 128 + 32)):
        with pytest.raises(ValueError):
            bad()
    with audit.scope(), pytest.raises(audit.AuditError):
        F.kv4_append_(k, k, torch.tensor([0, 1, 32], device=dev), pages)
    if dev == "cuda":
        with pytest.raises(RuntimeError):
            F.kv4_append_(k.float(), k.float(), s, pages)
        with pytest.raises(RuntimeError):
            F.kv4_append_(k, k.cpu(), s, pages)


# ------------------------------------------------------------------------------------------------ attention over the cache
def make_pool(rs, lens, nkv, hd, bs, width, dev):
    """A pool whose blocks lie in any order, block table, contexts. Unused table entries name a block that holds NaN."""
    per = -(-np.asarray(lens) // bs)
    blocks = int(per.sum()) + 1
    raw = rs.randint(0, 256, (blocks, nkv, bs * hd + bs * hd // 4)).astype(np.uint8)
    scale = rs.rand(blocks, nkv, 2 * bs * (hd // 32)) * 0.25 + 0.05
    par = np.stack([scale, -7.5 * scale + 0.2 * rs.randn(*scale.shape)], -1).astype(np.float16)
    order = rs.permutation(blocks)
    par[order[-1]] = np.nan
    table = np.full((len(lens), width), order[-1], dtype=np.int32)
    at = 0
    for i, n in enumerate(per):
        table[i, :n] = order[at : at + n]
        at += n
    for i, n in enumerate(lens):     # what lies behind the last token of a block is not looked at
        if n % bs:
            p = par[table[i, n // bs]].reshape(nkv, 2, bs, hd // 32, 2)
            p[:, :, n % bs :] = np.nan
    raw[..., bs * hd :] = par.reshape(blocks, nkv, -1).view(np.uint8)
    return torch.from_numpy(raw).to(dev), i32(table, dev), i32(lens, dev)


def attention_64(q, pages, table, lens, bs, scale):
    """(output, largest |output| that the roundings of the kernel may change each value by), in 64 bits."""
    B, nh, hd = q.shape
    (codes, step, _), (k, v) = unpacked(pages, bs, hd), rows_of(pages, bs, hd)
    step = np.broadcast_to(step.astype(np.float64), codes.shape).reshape(*codes.shape[:-2], hd)
    part = codes.reshape(*codes.shape[:-2], hd) * step         # what a code adds to its group's least value
    nkv = k.shape[1]
    q = q.double().cpu().numpy().reshape(B, nkv, nh // nkv, hd)
    out, off = np.zeros((B, nkv, nh // nkv, hd)), np.zeros((B, nkv, nh // nkv, hd))
    for b, n in enumerate(lens):
        if n == 0:
            continue
        blk = table[b, : -(-n // bs)].cpu().numpy()
        kk, vv, kp, vp, ks, vs = (x[blk].transpose(1, 0, 2, 3).reshape(nkv, -1, hd)[:, :n] for x in (k, v, part[0], part[1], step[0], step[1]))
        s = np.einsum("hgd,htd->hgt", q[b], kk) * scale
        w = np.exp(s - s.max(-1, keepdims=True))
        w /= w.sum(-1, keepdims=True)
        out[b] = np.einsum("hgt,htd->hgd", w, vv)
        # The kernel rounds to fp16, for neighbours a, b of a pair of codes: a s / 16, (b + a / 16) s and (keys) 16 q_a - q_b. With a <= 15, and U16 of each:
        #   keys:   2 (16 |q_a| + |q_b|) a s / 16 + |q_b| (b + a / 16) s  <=  2 sum |q| code s + 3 sum |q| s
        #   values: a s, and b s + 2 a s / 16 <= b s + 2 s
        # (or half the least fp16 number, at most 16 times: 2^-21). The least values are fp16 already, their factor is held in two halves (2^-22).
        # Sums of products are fp32 (their length times U32). A score is off by at most ds, a weight by 2 ds and by the rounding of
        # e^(s - reference) to fp16 (U16, and 2^-25 of the largest where it is small), which acts on the whole value.
        dot = lambda x: np.einsum("hgd,htd->hgt", np.abs(q[b]), np.abs(x))
        ds = abs(scale) * (U16 * dot(2 * kp + 3 * ks) + 2.0**-21 * np.abs(q[b]).sum(-1, keepdims=True) + (2.0**-22 + (hd + 8) * U32) * dot(np.abs(kk) + 3 * kp))
        ds = ds.max(-1, keepdims=True)
        size, codes_size = (np.einsum("hgt,htd->hgd", w, np.abs(x)) for x in (vv, vp + 2 * vs))
        off[b] = ((2 * ds + 2 * U16) * size + U16 * codes_size + 2.0**-21 + (n + 64) * U32 * (size + 3 * codes_size)
                  + 2.0**-24 * n * w.max(-1, keepdims=True) * np.abs(vv).max(1)[:, None])
    return out.reshape(B, nh, hd), off.reshape(B, nh, hd)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("nh,nkv,hd,bs,lens", [
    (1, 1, 64, 16, [1]), (2, 2, 128, 64, [1, 0, 64, 65]), (14, 2, 64, 16, [160, 3, 0, 77, 16]), (28, 4, 128, 64, [700, 1, 63, 129, 1000, 0, 2]),
    (16, 1, 128, 32, [1200, 31]), (32, 2, 64, 128, [127, 128, 129, 640]), (12, 1, 64, 256, [255, 257, 33]), (8, 8, 128, 16, [0, 0, 0]),
    (5, 1, 128, 64, [20000]), (40, 8, 128, 64, [333] * 40),
])
def test_attention_over_the_cache(dev, nh, nkv, hd, bs, lens, dtype):
    rs = np.random.RandomState(nh * hd + len(lens))
    width = max(1, -(-max(lens) // bs)) + 1
    pages, table, ctx = make_pool(rs, lens, nkv, hd, bs, width, dev)
    q = torch.from_numpy(rs.randn(len(lens), (nh + 2 * nkv) * hd)).to(dtype).to(dev)[:, : nh * hd].view(-1, nh, hd)
    out = F.paged_decode_attention_kv4(q, pages, table, ctx)
    want, off = attention_64(q, pages, table, lens, bs, 1.0 / math.sqrt(hd))
    assert out.dtype == dtype and out.shape == q.shape
    assert (np.abs(out.double().cpu().numpy() - want) <= off + HALF[dtype] * np.abs(want) + 2.0**-24).all()
    plan = torch.tensor([0] + np.cumsum([-(-n // 64) for n in lens]).tolist(), dtype=torch.int32, device=dev)
    assert torch.equal(F.paged_decode_attention_kv4(q, pages, table, ctx, plan=plan), out)
    assert torch.equal(F.paged_decode_attention_kv4(q, pages, table, ctx), out)       # and again the same bits
    again = F.paged_decode_attention_kv4(q, pages, table, ctx, scale=0.5)
    want, off = attention_64(q, pages, table, lens, bs, 0.5)
    assert (np.abs(again.double().cpu().numpy() - want) <= off + HALF[dtype] * np.abs(want) + 2.0**-24).all()


@pytest.mark.parametrize("nh,nkv,hd,bs,lens", [(28, 4, 128, 64, [700, 129, 1000]), (12, 1, 64, 16, [255, 33]), (16, 1, 128, 32, [1200, 31]), (14, 2, 64, 64, [5000])])
def test_attention_in_fp16_is_rounded_once(dev, nh, nkv, hd, bs, lens):
    """What the output's own rounding (at most 2^-11 of each value) does not explain is fp32 sums: scores below 2^4 from products whose magnitudes, with the
    64 that a code is held on, sum to below 2^10; 2^5 roundings of random sign of 2^-24 of that, weighed by a softmax, are below 2^-14."""
    rs = np.random.RandomState(nh + hd)
    pages, table, ctx = make_pool(rs, lens, nkv, hd, bs, -(-max(lens) // bs), dev)
    q = torch.from_numpy(rs.randn(len(lens), nh, hd)).half().to(dev)
    out = F.paged_decode_attention_kv4(q, pages, table, ctx).double().cpu().numpy()
    want, _ = attention_64(q, pages, table, lens, bs, 1.0 / math.sqrt(hd))
    assert np.linalg.norm(out - want) <= (2.0**-11 + 2.0**-14) * np.linalg.norm(want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attention_over_long_contexts(dtype):
    """Values of either sign cancel over a long context: what is left is small beside the codes, on which the sums must not lose it. The bound is the output's
    rounding, at most HALF of each value, and for bf16 as much again for the fp16 roundings of codes and weights (together below 2^-10 of the norm)."""
    B, nkv, G, hd, bs, n = 4, 2, 8, 64, 64, 80000
    g = torch.Generator(device="cuda").manual_seed(3)
    blocks = n // bs
    pages = torch.randint(0, 256, (B * blocks, nkv, F.kv4_page_bytes(bs, hd)), dtype=torch.uint8, device="cuda", generator=g)
    par = torch.empty(B * blocks, nkv, 2, bs, hd // 32, 2, dtype=torch.float16, device="cuda")
    step = torch.rand(par.shape[:-1], device="cuda", generator=g) * 0.25 + 0.05
    par[..., 0] = step
    par[..., 1] = -7.5 * step + 0.2 * torch.randn(step.shape, device="cuda", generator=g)
    pages[..., bs * hd :] = par.reshape(B * blocks, nkv, -1).view(torch.uint8)
    table = torch.randperm(B * blocks, device="cuda", generator=g).to(torch.int32).view(B, blocks)
    q = torch.randn(B, nkv * G, hd, device="cuda", generator=g).to(dtype)
    out = F.paged_decode_attention_kv4(q, pages, table, torch.full((B,), n, dtype=torch.int32, device="cuda")).double()
    want = torch.empty_like(out)
    for b in range(B):
        rows = table[b].long()
        code = pages[rows, :, : bs * hd].view(blocks, nkv, 2, bs, hd // 2)
        x = torch.stack([code & 15, code >> 4], -1).view(blocks, nkv, 2, bs, hd // 32, 32).double()
        pr = par[rows].double()
        k, v = (x * pr[..., :1] + pr[..., 1:]).permute(2, 1, 0, 3, 4, 5).reshape(2, nkv, n, hd)
        w = torch.softmax(torch.einsum("hgd,htd->hgt", q[b].double().view(nkv, G, hd), k) / math.sqrt(hd), -1)
        want[b] = torch.einsum("hgt,htd->hgd", w, v).view(nkv * G, hd)
    bound = HALF[dtype] + (2.0**-10 if dtype == torch.bfloat16 else 2.0**-14)
    assert float((out - want).norm() / want.norm()) <= bound


@pytest.mark.parametrize("factor", [1e-20, 1e-3, 300.0, 1e12])
def test_attention_with_queries_of_any_size(dev, factor):
    """Queries are brought to a common power of two before they are rounded to fp16: tiny ones keep their bits, large ones do not overflow."""
    rs = np.random.RandomState(5)
    pages, table, ctx = make_pool(rs, [100, 30], 2, 64, 64, 2, dev)
    q = (torch.from_numpy(rs.randn(2, 6, 64)) * factor).to(torch.bfloat16).to(dev)
    q[:, 3] *= 2.0**-9
    scale = 1.0 / (8.0 * factor)
    out = F.paged_decode_attention_kv4(q, pages, table, ctx, scale=scale)
    want, off = attention_64(q, pages, table, [100, 30], 64, scale)
    assert (np.abs(out.double().cpu().numpy() - want) <= off + 2.0**-8 * np.abs(want) + 2.0**-24).all()


def test_attention_with_a_scale_of_any_sign(dev):
    rs = np.random.RandomState(8)
    pages, table, ctx = make_pool(rs, [90, 1], 2, 64, 64, 2, dev)
    q = torch.from_numpy(rs.randn(2, 6, 64)).to(torch.bfloat16).to(dev)
    for scale in (-0.125, 0.0):
        out = F.paged_decode_attention_kv4(q, pages, table, ctx, scale=scale)
        want, off = attention_64(q, pages, table, [90, 1], 64, scale)
        assert (np.abs(out.double().cpu().numpy() - want) <= np.abs(off) + 2.0**-8 * np.abs(want) + 2.0**-20).all()


@pytest.mark.gpu
def test_attention_of_two_streams_and_of_a_wrong_plan():
    """Calls on two streams at once keep apart; a plan for other contexts gives other numbers, and nothing outside its tensors is touched."""
    rs = np.random.RandomState(9)
    pages, table, ctx = make_pool(rs, [700, 300, 0, 64], 2, 64, 64, 12, "cuda")
    q = torch.from_numpy(rs.randn(4, 6, 64)).to(torch.bfloat16).cuda()
    want = F.paged_decode_attention_kv4(q, pages, table, ctx)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i in range(20):
        with torch.cuda.stream(streams[i % 2]):
            got.append(F.paged_decode_attention_kv4(q, pages, table, ctx))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    for plan in ([0, 0, 0, 0, 0], [0, 40, 80, 120, 160], [5, 3, 9, 2, 7], [0, -5, 3, 2, 1], [0, 2**30, 0, 0, 2**31 - 1]):
        F.paged_decode_attention_kv4(q, pages, table, ctx, plan=i32(plan, "cuda"))
    torch.cuda.synchronize()
    assert torch.equal(F.paged_decode_attention_kv4(q, pages, table, ctx), want)
    from verl_b200.ops import native

    native.check_status()


def test_blocks_that_do_not_exist_are_skipped(dev):
    """A table entry outside the pool (within the context) is refused in audit mode; without it nothing outside the pool is read: on the GPU the
    tokens of such a block count as behind the context."""
    rs = np.random.RandomState(6)
    pages, table, ctx = make_pool(rs, [200, 64], 2, 64, 64, 4, dev)
    q = torch.from_numpy(rs.randn(2, 4, 64)).to(torch.bfloat16).to(dev)
    good = F.paged_decode_attention_kv4(q, pages, table, ctx)
    for wrong in (-1, pages.shape[0], 2**31 - 1):
        t = table.clone()
        t[0, 3] = wrong
        with audit.scope(), pytest.raises(audit.AuditError):
            F.paged_decode_attention_kv4(q, pages, t, ctx)
        if dev == "cuda":
            out = F.paged_decode_attention_kv4(q, pages, t, ctx)
            assert torch.equal(out[1], good[1])
            want, off = attention_64(q, pages, table, [192, 64], 64, 0.125)
            assert (np.abs(out.double().cpu().numpy() - want) <= off + 2.0**-8 * np.abs(want) + 2.0**-24).all()
    with audit.scope(), pytest.raises(audit.AuditError):
        F.paged_decode_attention_kv4(q, pages, table, i32([257, 64], dev))


def test_refusals_of_the_attention(dev):
    pages = torch.zeros(2, 2, F.kv4_page_bytes(16, 64), dtype=torch.uint8, device=dev)
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16, device=dev)
    t, c = torch.zeros(3, 1, dtype=torch.int32, device=dev), torch.zeros(3, dtype=torch.int32, device=dev)
    assert (F.paged_decode_attention_kv4(q, pages, t, c) == 0).all() and F.paged_decode_attention_kv4(q[:0], pages, t[:0], c[:0]).shape == (0, 4, 64)
    for bad in (lambda: F.paged_decode_attention_kv4(q[0], pages, t, c), lambda: F.paged_decode_attention_kv4(q[:, :3], pages, t, c),
                lambda: F.paged_decode_attention_kv4(q, pages, t[:2], c), lambda: F.paged_decode_attention_kv4(q, pages, t, c.long()),
                lambda: F.paged_decode_attention_kv4(q, pages, t.long(), c), lambda: F.paged_decode_attention_kv4(q, pages, t, c, plan=c),
                lambda: F.paged_decode_attention_kv4(q, pages[..., :-4], t, c), lambda: F.paged_decode_attention_kv4(q.int(), pages, t, c)):
        with pytest.raises(ValueError):
            bad()
    if dev == "cuda":
        for bad in (lambda: F.paged_decode_attention_kv4(q.float(), pages, t, c),                                        # type
                    lambda: F.paged_decode_attention_kv4(q.repeat(1, 9, 1), pages, t, c),                                # 18 heads to one
                    lambda: F.paged_decode_attention_kv4(q.transpose(0, 1).contiguous().transpose(0, 1), pages, t, c),   # heads apart
                    lambda: F.paged_decode_attention_kv4(q, pages, t.cpu(), c)):                                          # another device
            with pytest.raises(RuntimeError):
                bad()


# ------------------------------------------------------------------------------------------------ scores
def scores_64(logits, ids, top, temperature, valid):
    z = logits[:, :valid].double().cpu() / temperature
    logp = torch.log_softmax(z, -1)
    p = logp.exp()
    ent = -torch.where(p > 0, p * logp, 0.0).sum(-1)
    flat = ids.cpu().view(len(z), -1)
    ok = (flat >= 0) & (flat < valid)
    lp = torch.where(ok, logp.gather(1, flat.clamp(0, valid - 1)), 0.0).view(ids.shape)
    order = torch.sort(logits[:, :valid].float().cpu(), dim=-1, descending=True, stable=True).indices[:, :top]
    return lp, ent, torch.logsumexp(z, -1), order, logp.gather(1, order)


def slack(logits, valid, temperature):
    """How far a log-sum-exp may be off. A term e^(z - m) is off by 2^-22 and by its exponent's rounding (|z - m| U32, twice); a sum of n
    terms by U32 for each addition of its longest chain (a thread adds at most one term in 128 by itself, 40 more joins follow); z by U32 |z|."""
    z = logits[:, :valid].double().abs().cpu() / temperature
    big = torch.where(z.isfinite(), z, 0.0).amax(-1)
    return U32 * (8 + 6 * big + valid / 128 + 40)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,V,valid,n,top,temperature", [
    (1, 1, 1, 1, 1, 1.0), (3, 7, 5, 2, 5, 0.7), (5, 129, 129, 1, 128, 1.0), (2, 1003, 1000, 4, 20, 1.3), (1, 151936, 151936, 1, 5, 1.0),
    (33, 32000, 31990, 3, 64, 1.0), (300, 2049, 2049, 1, 1, 0.5), (7, 50257, 50257, 40, 0, 1.0), (20, 152064, 151936, 1, 128, 1.0),
])
def test_scores(dev, T, V, valid, n, top, temperature, dtype):
    g = torch.Generator().manual_seed(V + n)
    logits = (torch.randn(T, V + 3, generator=g) * 2.5).to(dtype).to(dev)[:, :V]      # rows on any boundary
    logits[:, valid:] = 1e4                                                           # columns that do not count
    ids = torch.randint(0, valid, (T, n), generator=g)
    ids[::3, 0] = -100
    ids = (ids[:, 0] if n == 1 else ids).to(dev)
    out = F.token_scores(logits, ids, top, temperature, valid if valid < V else 0)
    lp, ent, lse, order, top_lp = scores_64(logits, ids, top, temperature, valid)
    tol = slack(logits, valid, temperature)
    assert out.logprob.shape == ids.shape and out.logprob.dtype == torch.float32 and out.top_ids.dtype == torch.int64
    assert torch.equal(out.top_ids.cpu(), order)
    assert ((out.lse.double().cpu() - lse).abs() <= tol).all()
    t = tol.view(-1, *[1] * (ids.dim() - 1))
    assert ((out.logprob.double().cpu() - lp).abs() <= 2 * t).all() and ((out.top_logprob.double().cpu() - top_lp).abs() <= 2 * tol[:, None]).all()
    # entropy = log s - w / s: the terms of w are off as those of s, by their size
    z = logits[:, :valid].double().cpu() / temperature
    spread = (torch.softmax(z, -1) * (z.amax(-1, keepdim=True) - z)).sum(-1)
    assert ((out.entropy.double().cpu() - ent).abs() <= 2 * tol * (2 + spread)).all()
    assert all(torch.equal(a, b) for a, b in zip(out, F.token_scores(logits, ids, top, temperature, valid if valid < V else 0)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("top", [0, 20])
@pytest.mark.parametrize("V", [9000, 70000, 200000])
def test_scores_of_rows_that_grow(dev, V, top, dtype):
    """The first values of a row say nothing about the others: slopes, steps and single values far above what was there before, and all of it below zero."""
    g = torch.Generator().manual_seed(V)
    x = torch.randn(8, V, generator=g)
    slope = torch.linspace(-1, 1, V)
    x[0] += slope * 300
    x[1] -= slope * 300
    x[2, : V // 2] -= 5e4
    x[3, V - 3] = 80.0
    x[4, V // 2 :] += 45.0
    x[5] += slope * 20
    x[6] = x[6] - 1e3 + (torch.arange(V) // 3000) * 25.0
    x[7, : V - 100] = float("-inf")
    x = x.to(dtype).to(dev)
    ids = torch.full((8,), V - 3, device=dev)
    out = F.token_scores(x, ids, top)
    lp, ent, lse, order, top_lp = scores_64(x, ids, top, 1.0, V)
    tol = slack(x, V, 1.0)
    assert torch.equal(out.top_ids.cpu(), order)
    assert ((out.lse.double().cpu() - lse).abs() <= tol).all() and ((out.logprob.double().cpu() - lp).abs() <= 2 * tol).all()
    assert ((out.top_logprob.double().cpu() - top_lp).abs() <= 2 * tol[:, None]).all()
    # log s - w / s, with the terms of w up to 40 ln 2 (the least distance at which a reference moves) and the spread of the row larger than those of s
    z = x.double().cpu()
    p = torch.softmax(z, -1)
    spread = torch.where(p > 0, p * (z.amax(-1, keepdim=True) - z), 0.0).sum(-1)
    assert ((out.entropy.double().cpu() - ent).abs() <= tol * (2 + spread + 40 * math.log(2))).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [40, 3001, 70000])
def test_scores_of_masked_tied_and_undefined_rows(dev, V, dtype):
    g = torch.Generator().manual_seed(V)
    x = torch.randn(12, V, generator=g)
    inf = float("inf")
    x[0] = -inf                                       # nothing left
    x[1, 7:] = -inf                                   # fewer values than alternatives
    x[2] = 1.5                                        # all alike
    x[3] = torch.finfo(dtype).min                     # a mask of the type's lowest value on everything
    x[4, 5] = float("nan")
    x[5, 9] = inf
    x[6] = torch.arange(V) % 3                        # many ties
    x[7, ::2] = -inf
    x[8] = torch.sort(x[8], descending=True).values   # the largest ones side by side
    x[9] = torch.sort(x[9]).values
    x[10, ::256], x[10, 1::256] = 50 + torch.rand(len(x[10, ::256]), generator=g), 60   # the largest ones in one thread's columns
    x[11] = torch.finfo(dtype).min
    x[11, V - 1] = 3.0
    x = x.to(dtype).to(dev)
    x[6, 1::4] = -0.0
    x[6, 0::4] = 0.0
    k = min(V, 33)
    ids = torch.tensor([3, 10, 0, 1, 5, 9, 2, 1, 0, 1, 0, V - 1], device=dev)
    out = F.token_scores(x, ids, k)
    lp, ent, lse, order, top_lp = scores_64(x, ids, k, 1.0, V)
    good = [i for i in range(12) if i not in (0, 4, 5)]
    assert torch.equal(out.top_ids.cpu(), order)
    assert out.lse[0] == -inf and out.entropy[0] == 0 and out.logprob[0] == -inf and (out.top_logprob[0] == -inf).all()
    assert all(t[[4, 5]].isnan().all() for t in (out.lse, out.logprob, out.entropy))
    tol = slack(x, V, 1.0)[good]
    near = lambda a, b, t: ((a == b) | ((a - b).abs() <= t)).all()
    assert near(out.lse.double().cpu()[good], lse[good], tol) and near(out.logprob.double().cpu()[good], lp[good], 2 * tol)
    assert near(out.top_logprob.double().cpu()[good], top_lp[good], 2 * tol[:, None])
    assert near(out.entropy.double().cpu()[good], ent[good], 2 * slack(torch.randn(1, V), V, 1.0) * (2 + math.log(V)) + 60 * U32 * 200)
    d = F.token_scores_bwd(x, ids, out.lse, out.entropy, torch.ones(12, device=dev), torch.ones(12, device=dev))
    assert (d[0] == 0).all() and d[4].isnan().all() and d[5].isnan().all() and d[good].isfinite().all()


@pytest.mark.parametrize("V", [40, 30011])
def test_rows_of_the_type_s_lowest_value_are_uniform(dev, V):
    """A mask that is added as the type's lowest value and leaves nothing: all tokens alike, log-sum-exp at the value itself."""
    for dtype in (torch.bfloat16, torch.float32):
        low = torch.finfo(dtype).min
        x = torch.full((2, V), low, dtype=dtype, device=dev)
        x[1, 3] = 2.0
        ids = torch.tensor([V - 1, 3], device=dev)
        out = F.token_scores(x, ids, 4)
        assert out.lse[0] == low and out.top_ids.tolist() == [[0, 1, 2, 3], [3, 0, 1, 2]]
        tol = 16 * U32 * math.log(V)      # a logarithm of V ones, and their sum
        assert abs(float(out.logprob[0]) + math.log(V)) <= tol and abs(float(out.entropy[0]) - math.log(V)) <= tol
        assert abs(float(out.top_logprob[0, 0]) + math.log(V)) <= tol and out.logprob[1] == 0 and out.entropy[1] == 0
        d = F.token_scores_bwd(x, ids, out.lse, out.entropy, torch.ones(2, device=dev), None).double().cpu()
        want = torch.full((V,), -1.0 / V, dtype=torch.float64)
        want[V - 1] += 1
        assert ((d[0] - want).abs() <= want.abs() * (HALF[dtype] + 64 * U32)).all() and (d[1] == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [2000, 50257, 300000])
def test_alternatives_among_many_equal_values(dev, V, dtype):
    """More values at the k-th largest one than the kernel keeps: those above it, then the first of its equals."""
    g = torch.Generator().manual_seed(V)
    x = torch.randn(8, V, generator=g)
    few = torch.randint(0, V, (5,), generator=g)
    x[0, :] = float("-inf")
    x[0, few] = torch.arange(5.0)                                   # a mask that leaves five
    x[1] = 0.1                                                      # no short number in 32 bits
    x[2] = torch.randint(0, 4, (V,), generator=g) * 0.3 - 5.1       # four values, all negative
    x[3] = (torch.rand(V, generator=g) < 0.01) * 2.0                # one in a hundred
    x[4] = -0.1
    x[4, V - 1], x[4, V // 2] = 0.3, 0.2
    x[5] = torch.arange(V).flip(0) // 1000                          # equal ones side by side
    x[6, :] = -1e-30
    x[7, :] = float("-inf")
    x = x.to(dtype).to(dev)
    for k in (1, 20, 128):
        out = F.token_scores(x, torch.zeros(8, dtype=torch.int64, device=dev), k)
        _, _, _, order, top_lp = scores_64(x, torch.zeros(8, dtype=torch.int64), k, 1.0, V)
        assert torch.equal(out.top_ids.cpu(), order)
        got, tol = out.top_logprob.double().cpu(), 2 * slack(x, V, 1.0)[:, None]
        assert ((got == top_lp) | ((got - top_lp).abs() <= tol))[:7].all() and (got[7] == float("-inf")).all()


def grad_64(logits, ids, g_lp, g_ent, temperature, valid):
    z = (logits[:, :valid].double().cpu() / temperature).requires_grad_(True)
    logp = torch.log_softmax(z, -1)
    flat = ids.cpu().view(len(z), -1)
    ok = (flat >= 0) & (flat < valid)
    lp = torch.where(ok, logp.gather(1, flat.clamp(0, valid - 1)), 0.0)
    ent = -(logp.exp() * logp).sum(-1)
    obj = (lp * g_lp.double().cpu().view(lp.shape)).sum() + ((ent * g_ent.double().cpu()).sum() if g_ent is not None else 0.0)
    out = torch.zeros(logits.shape, dtype=torch.float64)
    out[:, :valid] = torch.autograd.grad(obj, z)[0] / temperature
    return out, logp.detach(), ent.detach()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,V,valid,n,temperature,entropy", [
    (1, 3, 3, 1, 1.0, True), (4, 129, 120, 5, 0.7, True), (3, 1003, 1003, 300, 1.0, False), (2, 151936, 151936, 1, 1.0, True),
    (65, 32000, 31990, 32, 1.3, True), (500, 513, 513, 1, 1.0, False),
])
def test_gradient_of_the_scores(dev, T, V, valid, n, temperature, entropy, dtype):
    g = torch.Generator().manual_seed(V * n)
    logits = (torch.randn(T, V + 5, generator=g) * 2).to(dtype).to(dev)[:, 1 : V + 1]
    ids = torch.randint(0, valid, (T, n), generator=g)
    if n > 2:
        ids[:, 2] = ids[:, 0]          # the same token twice
        ids[0, 1] = -100
        ids[-1, 1] = valid             # behind the vocabulary: no token
    ids = (ids[:, 0] if n == 1 else ids).to(dev)
    g_lp, g_ent = torch.randn(ids.shape, generator=g).to(dev), torch.randn(T, generator=g).to(dev) if entropy else None
    x = logits.detach().requires_grad_(True)
    lp, ent = token_logprobs(x, ids, temperature, valid if valid < V else 0)
    grads = torch.autograd.grad((lp, ent) if entropy else (lp,), x, (g_lp, g_ent) if entropy else (g_lp,))
    want, logp, ent64 = grad_64(logits, ids, g_lp, g_ent, temperature, valid)
    # p is off by the error of log p (slack, twice) and 2^-22; the bracket by its own terms; the sum over the given tokens by n U32
    tol = 2 * slack(logits, valid, temperature)[:, None] + 2.0**-22 + n * U32
    G = g_lp.abs().double().cpu().view(T, -1).sum(-1, keepdim=True)
    h = g_ent.abs().double().cpu()[:, None] if entropy else torch.zeros(T, 1, dtype=torch.float64)
    size = torch.zeros(T, V, dtype=torch.float64)
    size[:, :valid] = logp.exp() * (G + h * (logp.abs() + ent64[:, None] + 4 + math.log(valid)))
    size.scatter_add_(1, ids.cpu().view(T, -1).clamp(0, valid - 1), g_lp.abs().double().cpu().view(T, -1) * U32 * n / tol)
    off = (grads[0].double().cpu() - want).abs()
    small = {torch.bfloat16: 2.0**-134, torch.float16: 2.0**-25, torch.float32: 2.0**-126}[dtype]     # half the least step of the type
    assert grads[0].dtype == dtype and (off <= want.abs() * HALF[dtype] + size * tol / temperature * (1 + HALF[dtype]) + small).all()
    assert (grads[0][:, valid:] == 0).all()


def test_gradient_against_differences(dev):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(3, 17, generator=g).to(dev).requires_grad_(True)
    ids = torch.randint(0, 17, (3, 4), generator=g).to(dev)
    g_lp, g_ent = torch.randn(3, 4, generator=g), torch.randn(3, generator=g)
    lp, ent = token_logprobs(x, ids, temperature=0.8)
    ((lp * g_lp.to(dev)).sum() + (ent * g_ent.to(dev)).sum()).backward()

    def objective(v):
        logp = torch.log_softmax(v / 0.8, -1)
        return float((logp.gather(1, ids.cpu()) * g_lp.double()).sum() - ((logp.exp() * logp).sum(-1) * g_ent.double()).sum())

    base, h = x.detach().double().cpu(), 1e-4
    for i in range(3):
        for j in range(17):
            d = torch.zeros_like(base)
            d[i, j] = h
            want = (objective(base + d) - objective(base - d)) / (2 * h)     # off by h^2 times a third derivative (below 100) / 6, and 1e-15 / h
            assert abs(float(x.grad[i, j]) - want) < 1e-6 + 2e-6 * (1 + abs(want))


def test_log_probs_for_any_leading_shape_and_without_a_use(dev):
    x = torch.randn(2, 3, 50, device=dev, requires_grad=True)
    one, many = torch.randint(0, 50, (2, 3), device=dev), torch.randint(0, 50, (2, 3, 5), device=dev)
    ref = torch.log_softmax(x.detach().double(), -1)
    for ids in (one, many):
        lp, ent = token_logprobs(x, ids)
        want = ref.gather(-1, ids.view(2, 3, -1)).view(ids.shape)
        assert lp.shape == ids.shape and ent.shape == (2, 3) and (lp.double() - want).abs().max() < 1e-5
        (grad,) = torch.autograd.grad(ent.sum(), x)       # only one of the two is used
        assert grad.shape == x.shape and grad.abs().sum() > 0
    lp, _ = token_logprobs(x.transpose(0, 1), one.t())    # strides of another order
    assert (lp.t().double() - ref.gather(-1, one[..., None])[..., 0]).abs().max() < 1e-5
    lp, ent = token_logprobs(torch.zeros(0, 9, device=dev), torch.zeros(0, dtype=torch.int64, device=dev))
    assert lp.shape == (0,) and ent.shape == (0,)
    with torch.no_grad():
        wide = torch.randn(4, 10, device=dev).expand(4, 10)[:, ::2]     # columns apart
        assert (token_logprobs(wide, one.view(-1)[:4] % 5)[1] > 0).all()


def test_log_probs_are_differentiated_once(dev):
    x = torch.randn(3, 20, device=dev, requires_grad=True)
    lp, ent = token_logprobs(x, torch.zeros(3, dtype=torch.int64, device=dev))
    (g,) = torch.autograd.grad(lp.sum() + ent.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(g.square().sum(), x)
    lp, _ = token_logprobs(x, torch.zeros(3, dtype=torch.int64, device=dev))
    with torch.no_grad():
        x.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        lp.sum().backward()
    with torch.no_grad():
        assert not token_logprobs(x, torch.zeros(3, dtype=torch.int64, device=dev))[0].requires_grad


def test_entropy_changed_in_place_before_the_backward_pass(dev):
    """The gradient needs the entropy as it was: it has it, or says that it was changed."""
    x = torch.randn(3, 20, device=dev, requires_grad=True)
    ids = torch.zeros(3, dtype=torch.int64, device=dev)
    want = torch.autograd.grad(sum(t.sum() for t in token_logprobs(x, ids)), x)[0]
    lp, ent = token_logprobs(x, ids)
    total = lp.sum() + ent.sum()
    with torch.no_grad():
        ent.mul_(2.0)
    try:
        assert torch.equal(torch.autograd.grad(total, x)[0], want)
    except RuntimeError as e:
        assert "modified by an inplace operation" in str(e)


@pytest.mark.gpu
@pytest.mark.parametrize("T,V", [(3, 1003), (2, 70000)])
def test_scores_and_their_gradient_captured_and_replayed(T, V):
    x = torch.randn(T, V, device="cuda", requires_grad=True)
    ids = torch.randint(0, V, (T, 2), device="cuda")
    g_lp, g_ent = torch.randn(T, 2, device="cuda"), torch.randn(T, device="cuda")

    def step():
        lp, ent = token_logprobs(x, ids)
        return lp, ent, torch.autograd.grad((lp, ent), x, (g_lp, g_ent))[0], F.token_scores(x.detach(), ids, 9)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for _ in range(2):
        with torch.no_grad():
            x.copy_(torch.randn(T, V))
        graph.replay()
        eager = step()
        for a, b in zip((*captured[:3], *captured[3]), (*eager[:3], *eager[3])):
            assert torch.equal(a, b)


def test_refusals_of_the_scores(dev):
    x, ids = torch.zeros(2, 9, device=dev), torch.zeros(2, dtype=torch.int64, device=dev)
    for bad in (lambda: F.token_scores(x[0], ids), lambda: F.token_scores(x, ids[:1]), lambda: F.token_scores(x, ids.int()),
                lambda: F.token_scores(x, ids, 10), lambda: F.token_scores(x, ids, -1), lambda: F.token_scores(x, ids, temperature=0.0),
                lambda: F.token_scores(x, ids, temperature=float("nan")), lambda: F.token_scores(x, ids, valid_vocab=10),
                lambda: F.token_scores(x, ids, 6, valid_vocab=5), lambda: F.token_scores(x.long(), ids), lambda: F.token_scores(x[:, :0], ids),
                lambda: F.token_scores(torch.zeros(2, 300, device=dev), ids, 129), lambda: token_logprobs(x, torch.zeros(3, dtype=torch.int64, device=dev)),
                lambda: F.token_scores(x, torch.zeros(2, 4097, dtype=torch.int64, device=dev)),
                lambda: F.token_scores_bwd(x, ids, x[:, 0], x[:, 0], x[:1, 0], None), lambda: F.token_scores_bwd(x, ids, x[0], x[:, 0], x[:, 0], None)):
        with pytest.raises(ValueError):
            bad()
    if dev == "cuda":
        with pytest.raises(RuntimeError):
            F.token_scores(x.double(), ids)
        with pytest.raises(RuntimeError):
            F.token_scores(x, ids.cpu())
