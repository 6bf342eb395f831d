"""Block tables that the rollout engine writes from its block lists."""

import pytest
import torch

from verl_b200.models import FlatParams, get_preset
from verl_b200.workers.rollout.native.engine import RolloutEngine


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def engine(request):
    cfg = get_preset("tiny-qwen2")
    P = FlatParams(cfg, dtype=torch.bfloat16 if request.param == "cuda" else torch.float32, device=request.param)
    P.init_weights(seed=1, std=0.1)
    return RolloutEngine(cfg, P, max_num_seqs=6, max_model_len=128, block_size=16, num_blocks=64, eos_token_id=-1)


def test_tables_of_some_slots(engine):
    engine.block_table.fill_(77)
    engine._write_tables([4, 0, 2], [[5, 6, 7], [], [63, 1, 2, 3, 4, 8, 9, 10]])
    want = torch.full_like(engine.block_table, 77).cpu()
    want[4, :3], want[2, :8] = torch.tensor([5, 6, 7]), torch.tensor([63, 1, 2, 3, 4, 8, 9, 10])
    assert torch.equal(engine.block_table.cpu(), want)
    engine._write_tables([], [])
    assert torch.equal(engine.block_table.cpu(), want)


def test_what_would_not_be_written_is_refused(engine):
    engine.block_table.fill_(77)
    for slots, blocks in (([6], [[1]]), ([-1], [[1]]), ([0], [list(range(9))]), ([0, 1], [[1]])):
        with pytest.raises(AssertionError):
            engine._write_tables(slots, blocks)
    assert (engine.block_table == 77).all()


@pytest.mark.gpu
def test_the_host_does_not_wait_for_tables():
    cfg = get_preset("tiny-qwen2")
    P = FlatParams(cfg, dtype=torch.bfloat16, device="cuda")
    P.init_weights(seed=1, std=0.1)
    eng = RolloutEngine(cfg, P, max_num_seqs=6, max_model_len=128, block_size=16, num_blocks=64, eos_token_id=-1)
    torch.cuda.synchronize()
    mode = torch.cuda.get_sync_debug_mode()
    torch.cuda.set_sync_debug_mode("error")
    try:
        eng._write_tables([1, 3], [[1, 2], [4]])
    finally:
        torch.cuda.set_sync_debug_mode(mode)
    assert eng.block_table[1, :2].tolist() == [1, 2] and eng.block_table[3, 0] == 4
