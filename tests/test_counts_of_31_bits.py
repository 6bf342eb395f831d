"""Sizes whose steps would leave 31 bits are refused before anything is launched or copied: tensors that only seem to be as large."""

import pytest
import torch

from verl_b200.ops import functional as F

pytestmark = pytest.mark.gpu


def test_sizes_that_are_not_counted_are_refused():
    dev = "cuda"
    small = torch.zeros(1, dtype=torch.int64, device=dev)
    vec = torch.zeros(1, dtype=torch.int32, device=dev)
    before = torch.cuda.memory_allocated()
    wide = torch.zeros(1, 1, dtype=torch.bfloat16, device=dev).expand(1, 2**31 - 2)
    high = torch.zeros(1, 4, dtype=torch.bfloat16, device=dev).expand(2**31 - 1, 4)
    stat = torch.zeros(1, device=dev)
    k = torch.zeros(1, 1, 64, dtype=torch.bfloat16, device=dev).expand(2**30 + 1, 1, 64)
    pages = torch.zeros(1, 1, F.kv4_page_bytes(16, 64), dtype=torch.uint8, device=dev)
    table = vec.view(1, 1).expand(2**30 + 1, 1)
    for bad in (lambda: F.token_scores(wide, small), lambda: F.token_scores(high, small.expand(2**31 - 1)),
                lambda: F.token_logprobs(wide, small), lambda: F.token_scores_bwd(wide, small, stat, stat, stat, None),
                lambda: F.kv4_append_(k, k, small.expand(2**30 + 1), pages), lambda: F.kv4_gather(pages, small.expand(2**30 + 1), 64),
                lambda: F.decode_slot_map(table, vec.expand(2**30 + 1), vec.expand(2**30 + 1), vec.bool().expand(2**30 + 1), 16)):
        with pytest.raises(RuntimeError, match="at most 2"):
            bad()
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before < 1 << 30
