"""Scales of the 4-bit cache: what the append writes lies below the attention's limit, and audit mode names a pool that does not."""

import pytest
import torch

from verl_b200.ops import audit
from verl_b200.ops import functional as F


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def dev(request):
    return request.param


def test_a_scale_beyond_the_limit_is_named(dev):
    bs, hd, nkv = 16, 64, 2
    pages = torch.zeros(4, nkv, F.kv4_page_bytes(bs, hd), dtype=torch.uint8, device=dev)
    k = torch.randn(4 * bs, nkv, hd, device=dev).to(torch.bfloat16)
    k[3, 1, 5], k[40, 0, 9], k[41, 0, 9], k[50, 1, 0] = 3e38, -3e38, 3e38, float("nan")     # the largest scales that the append writes, and a NaN
    k[40, 0, 10] = 3e38
    F.kv4_append_(k, k, torch.arange(4 * bs, device=dev), pages)
    q = torch.randn(2, 4, hd, device=dev).to(torch.bfloat16)
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=dev)
    ctx = torch.tensor([32, 18], dtype=torch.int32, device=dev)
    with audit.scope():
        out = F.paged_decode_attention_kv4(q, pages, table, ctx)
    assert out[0].isfinite().all() and out[1, :2].isfinite().all()
    for value in (0, 1):
        bad = pages.clone()
        params = F._kv4_views(bad, bs, hd)[value][1]
        params[3, 1, 1, 0, 0] = 1024.0           # token 17 of the second sequence
        with audit.scope(), pytest.raises(audit.AuditError, match="token 17 of sequence 1"):
            F.paged_decode_attention_kv4(q, bad, table, ctx)
        with audit.scope():                      # behind the context it is nobody's
            F.paged_decode_attention_kv4(q, bad, table, ctx - torch.tensor([0, 1], dtype=torch.int32, device=dev))
