"""Slots and positions of packed batches beyond a few million tokens or a few thousand sequences, on the host and on the device."""

import numpy as np
import pytest
import torch

from verl_b200.ops import functional as F


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def dev(request):
    return request.param


def i32(x, dev):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32).to(dev)


def check(dev, table, rows, starts, ends, bs, total):
    cu, pos, slots = F.build_slot_map(i32(table, dev), i32(rows, dev), i32(starts, dev), i32(ends, dev), bs, total)
    lens = np.maximum(ends - np.maximum(starts, 0), 0)
    want = np.minimum(np.concatenate([[0], np.cumsum(lens)]), total)
    assert np.array_equal(cu.cpu().numpy(), want)
    t = np.arange(total)
    seq = np.minimum(np.searchsorted(want[1:], t, side="right"), len(rows) - 1)
    on = t < want[-1]
    p = np.where(on, np.maximum(starts, 0)[seq] + t - want[seq], 0)
    page = table[rows[seq], np.minimum(p // bs, table.shape[1] - 1)].astype(np.int64)
    assert np.array_equal(pos.cpu().numpy(), p)
    assert np.array_equal(slots.cpu().numpy(), np.where(on & (p // bs < table.shape[1]), page * bs + p % bs, -1))


@pytest.mark.parametrize("n,most,bs", [(5, 2_000_003, 64), (600, 12_000, 48)])
def test_more_than_four_million_tokens(dev, n, most, bs):
    """Open sequences that continue long contexts: what the cache holds of them is looked up in one batch."""
    rs = np.random.RandomState(n)
    starts = rs.randint(0, 100, n).astype(np.int64)
    ends = rs.randint(most // 2, most, n).astype(np.int64) + starts
    table = rs.permutation(n * (-(-(most + 100) // bs))).reshape(n, -1).astype(np.int32)
    total = int((ends - starts).sum())
    assert total > 1 << 22
    for more in (0, 3, -1001):
        check(dev, table, rs.permutation(n), starts, ends, bs, total + more)


@pytest.mark.parametrize("n", [8192, 8193, 20011])
def test_more_sequences_than_a_block_holds_sums_of(dev, n):
    rs = np.random.RandomState(n)
    starts = rs.randint(0, 40, n).astype(np.int64)
    ends = starts + rs.randint(-3, 9, n)
    table = rs.permutation(n * 3).reshape(n, 3).astype(np.int32)
    total = int(np.maximum(ends - starts, 0).sum())
    for more in (0, 7, -5):
        check(dev, table, rs.permutation(n), starts, ends, 16, total + more)


def test_lengths_whose_sum_is_beyond_32_bits(dev):
    """Only as many tokens as there are places count, however long the sequences say that they are."""
    n = 1500
    starts = np.zeros(n, dtype=np.int64)
    ends = np.full(n, 2**31 - 1, dtype=np.int64)
    ends[:700:2] = 3
    ends[1:700:2] = -(2**31)
    starts[1:700:2] = 2**31 - 1
    check(dev, np.arange(2 * n, dtype=np.int32).reshape(n, 2), np.arange(n), starts, ends, 64, 5000)


@pytest.mark.gpu
def test_refusal_of_more_places_than_are_counted():
    t, v = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="fewer than"):
        F.build_slot_map(t, v, v, v, 64, 2**31 - 1)
