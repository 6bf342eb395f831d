"""The rollout engine over the 4-bit cache and its records of alternatives: against the dense cache that holds the same quantised values, against
full forward passes, and the operators in a row as a decode step uses them, captured and replayed."""

import asyncio

import numpy as np
import pytest
import torch

from tests.test_rollout_step_ops import attention_64, quantised, scores_64, slack
from verl_b200.experimental.teacher_loop import TeacherServer
from verl_b200.models import DecoderModel, FlatParams, PackedBatch, get_preset
from verl_b200.ops import functional as F
from verl_b200.trainer.distillation.losses import DistillationLossConfig, compute_forward_kl_topk
from verl_b200.utils.kernel import token_logprobs
from verl_b200.workers.rollout.native import engine as E
from verl_b200.workers.rollout.native.engine import RolloutEngine, SamplingParams

PROMPTS = [[5, 6, 7, 8, 9], [10, 11, 12], list(range(20, 60)), [3, 4], [7] * 17, [10, 11, 12]]


def tiny(preset="tiny-qwen2", seed=3, device="cpu", dtype=torch.float32):
    cfg = get_preset(preset)
    P = FlatParams(cfg, dtype=dtype, device=device)
    P.init_weights(seed=seed, std=0.1)
    return cfg, P


def fake_quantised(x):
    q, s, m = quantised(x.float().numpy())
    return torch.from_numpy((q.astype(np.float32) * s.astype(np.float32) + m.astype(np.float32)).reshape(x.shape)).to(x.dtype)


def run(cfg, P, **kw):
    sampling = SamplingParams(temperature=kw.pop("temperature", 0.0), max_tokens=9, ignore_eos=True, top_logprobs=kw.pop("top", 0))
    eng = RolloutEngine(cfg, P, max_num_seqs=4, max_model_len=96, block_size=16, sync_interval=3, eos_token_id=-1, **kw)
    return eng, eng.generate(PROMPTS, sampling)


@pytest.mark.parametrize("preset", ["tiny-qwen2", "tiny-qwen3", "tiny-llama"])
def test_engine_over_the_4_bit_cache_equals_a_dense_cache_of_the_same_values(preset, monkeypatch):
    cfg, P = tiny(preset)
    four, outs = run(cfg, P, kv_cache_dtype="int4")
    assert four.kv.dtype == torch.uint8 and four.kv_bytes_per_block() * four.num_blocks == four.kv.numel()
    append = F.kv_append_
    monkeypatch.setattr(E.F, "kv_append_", lambda k, v, slots, kc, vc: append(fake_quantised(k), fake_quantised(v), slots, kc, vc))
    monkeypatch.setattr(E.F, "rope_kv_append_", None)
    qk = F.qk_norm_rope_
    monkeypatch.setattr(E.F, "qk_norm_rope_", lambda qkv, pos, cos, sin, wq, wk, eps, nh, nkv, hd, slots=None, kc=None, vc=None, **kw: (
        qk(qkv, pos, cos, sin, wq, wk, eps, nh, nkv, hd, **kw) if slots is None else
        (qk(qkv, pos, cos, sin, wq, wk, eps, nh, nkv, hd), E.F.kv_append_(qkv[:, nh * hd : (nh + nkv) * hd].reshape(-1, nkv, hd),
                                                                        qkv[:, (nh + nkv) * hd :].reshape(-1, nkv, hd), slots, kc, vc))[0]))
    monkeypatch.setenv("VERL_B200_FUSED_ROPE_APPEND", "0")
    _, dense = run(cfg, P)
    for a, b in zip(outs, dense):
        assert a.token_ids == b.token_ids
        assert torch.allclose(torch.tensor(a.log_probs), torch.tensor(b.log_probs), atol=1e-5)   # fp32 sums of the same numbers in another order
    assert not four.running and len(four.free_blocks) == four.num_blocks


def test_prefix_cache_handoff_and_release_with_the_4_bit_cache():
    cfg, P = tiny()
    plain = RolloutEngine(cfg, P, max_num_seqs=2, max_model_len=96, block_size=16, sync_interval=3, eos_token_id=-1, kv_cache_dtype="int4")
    kept = RolloutEngine(cfg, P, max_num_seqs=2, max_model_len=96, block_size=16, sync_interval=3, eos_token_id=-1, kv_cache_dtype="int4",
                         enable_prefix_caching=True)
    sp = SamplingParams(temperature=0.0, max_tokens=5, ignore_eos=True)
    prompt = list(range(30, 70))
    first = kept.generate([prompt], sp)[0]
    again = kept.generate([prompt[:32] + [9, 9]], sp)[0]       # 32 tokens come from the cache, dequantised
    assert kept.stats["prefix_cache_hit_tokens"] == 32
    assert first.token_ids == plain.generate([prompt], sp)[0].token_ids and len(again.token_ids) == 5
    hand = plain.prefill_only([prompt], sp)
    decode = RolloutEngine(cfg, P, max_num_seqs=2, max_model_len=96, block_size=16, sync_interval=3, eos_token_id=-1, kv_cache_dtype="int4")
    decode.add_prefilled(hand[0], sp)
    out = []
    while decode.has_unfinished():
        out += decode.step()
    assert out[0].token_ids == first.token_ids
    dense = RolloutEngine(cfg, P, max_num_seqs=2, max_model_len=96, block_size=16, eos_token_id=-1)
    dense.add_prefilled(hand[0], sp)
    with pytest.raises(AssertionError, match="kv_cache_dtype"):
        dense.step()
    plain.release_kv_cache()
    plain.resume_kv_cache()
    assert plain.generate([prompt], sp)[0].token_ids == first.token_ids


@pytest.mark.parametrize("temperature", [0.0, 0.7])
def test_records_of_alternatives_and_entropy(temperature):
    cfg, P = tiny()
    eng, outs = run(cfg, P, temperature=temperature, top=5)
    model = DecoderModel(cfg, P)
    t = temperature or 1.0
    for p, o in zip(PROMPTS, outs):
        rec = o.extra_fields
        assert rec["top_token_ids"].shape == rec["top_logprobs"].shape == (9, 5) and rec["entropy"].shape == (9,)
        ids = p + o.token_ids[:-1]
        logp = torch.log_softmax(model.forward_logits(PackedBatch.from_lengths(torch.tensor(ids), [len(ids)])).float()[len(p) - 1 :] / t, -1)
        want = logp.topk(5, -1)
        assert torch.equal(rec["top_token_ids"], want.indices)
        assert torch.allclose(rec["top_logprobs"], want.values, atol=1e-4) and torch.allclose(rec["entropy"], -(logp.exp() * logp).sum(-1), atol=1e-4)
        if temperature == 0:
            assert rec["top_token_ids"][:, 0].tolist() == o.token_ids
    assert "entropy" not in eng.generate([[3, 4]], SamplingParams(max_tokens=2, ignore_eos=True))[0].extra_fields
    hand = eng.prefill_only([[3, 4, 5]], SamplingParams(temperature=0.0, max_tokens=3, top_logprobs=2))
    eng.add_prefilled(hand[0], SamplingParams(temperature=0.0, max_tokens=3, ignore_eos=True, top_logprobs=2))
    while eng.has_unfinished():
        got = eng.step()
    assert got[0].extra_fields["top_token_ids"][:, 0].tolist() == got[0].token_ids


def test_refusals_of_the_engine():
    cfg, P = tiny()
    with pytest.raises(AssertionError, match="kv_cache_dtype"):
        RolloutEngine(cfg, P, max_num_seqs=2, max_model_len=32, block_size=16, kv_cache_dtype="fp4")
    with pytest.raises(ValueError, match="multiple of 16"):
        RolloutEngine(cfg, P, max_num_seqs=2, max_model_len=32, block_size=8, kv_cache_dtype="int4")
    eng = RolloutEngine(cfg, P, max_num_seqs=2, max_model_len=32, block_size=16)
    for bad in (-1, 129):
        with pytest.raises(ValueError, match="top_logprobs"):
            eng.add_request([1, 2], SamplingParams(top_logprobs=bad))


def test_given_tokens_through_the_4_bit_cache():
    """Sequences fed in portions and single tokens: the last logits follow from the tokens whichever way they came, up to what 4 bits lose."""
    cfg, P = tiny()
    ids = list(range(40, 75))
    eng = RolloutEngine(cfg, P, max_num_seqs=3, max_model_len=64, block_size=16, eos_token_id=-1, kv_cache_dtype="int4")
    for key in ("a", "b"):
        eng.open_sequence(key)
    whole = eng.feed([("a", ids, [len(ids) - 1])])[0]
    eng.feed([("b", ids[:20], [])])
    eng.feed([("b", ids[20:34], [])])
    last = eng.feed([("b", ids[34:], [0])])[0]
    exact = DecoderModel(cfg, P).forward_logits(PackedBatch.from_lengths(torch.tensor(ids), [len(ids)])).float()[-1:]
    assert torch.allclose(whole, exact, atol=1e-4)            # a whole prompt attends to its own keys, not to the cache's
    assert (last - exact).norm() < 0.2 * exact.norm() and not torch.equal(last, exact)
    for key in ("a", "b"):
        eng.close_sequence(key)


# ------------------------------------------------------------------------------------------------ on a GPU
def small_gpu(head_dim=64):
    cfg = get_preset("tiny-qwen2")
    cfg.hidden_size, cfg.num_attention_heads, cfg.num_key_value_heads, cfg.head_dim = 4 * head_dim, 4, 2, head_dim
    P = FlatParams(cfg, dtype=torch.bfloat16, device="cuda")
    P.init_weights(seed=5, std=0.05)
    return cfg, P


@pytest.mark.gpu
@pytest.mark.parametrize("head_dim", [64, 128])
def test_captured_steps_equal_eager_ones(head_dim):
    cfg, P = small_gpu(head_dim)
    kw = dict(kv_cache_dtype="int4", top=4, temperature=0.0)
    _, eager = run(cfg, P, use_cuda_graph=False, **kw)
    eng, captured = run(cfg, P, **kw)
    assert eng._graph is not None
    for a, b in zip(eager, captured):
        assert a.token_ids == b.token_ids and a.log_probs == b.log_probs
        for key in ("top_token_ids", "top_logprobs", "entropy"):
            assert torch.equal(a.extra_fields[key], b.extra_fields[key])
        assert b.extra_fields["top_token_ids"][:, 0].tolist() == b.token_ids
    dense_eng, dense = run(cfg, P, temperature=0.0)
    assert eng.kv_bytes_per_block() * 3.2 == dense_eng.kv_bytes_per_block()
    # two engines' graphs replayed in turn share nothing that they write
    other = RolloutEngine(cfg, P, max_num_seqs=4, max_model_len=96, block_size=16, sync_interval=3, eos_token_id=-1, kv_cache_dtype="int4")
    sp = SamplingParams(temperature=0.0, max_tokens=9, ignore_eos=True)
    want = [o.token_ids for o in other.generate(PROMPTS, sp)]
    for e in (other, eng):
        for p in PROMPTS[:3]:
            e.add_request(p, sp)
    done = {other: {}, eng: {}}
    while other.has_unfinished() or eng.has_unfinished():
        for e in (other, eng):
            for o in e.step():
                done[e][tuple(o.prompt_ids)] = o.token_ids
    for e in done:
        assert [done[e][tuple(p)] for p in PROMPTS[:3]] == want[:3]
    from verl_b200.ops import native

    native.check_status()


@pytest.mark.gpu
def test_operators_of_a_decode_step_in_a_row_captured_and_replayed():
    """Tables, slots, append, attention and scores as a step uses them: captured once, replayed while the sequences grow; every stage is held to
    the plain forms on what the stage before it left."""
    dev, bs, nh, nkv, hd, V, S = "cuda", 16, 8, 2, 64, 3001, 5
    rs = np.random.RandomState(1)
    width, scale = 6, 0.125
    lens = [1, 15, 16, 40, 33]
    g = torch.Generator().manual_seed(2)
    table = torch.zeros(S, width, dtype=torch.int32, device=dev)
    pool = torch.from_numpy(rs.permutation(S * width).astype(np.int32)).to(dev)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    rows = i32(list(range(S)))
    used = F.extend_block_tables_(table, rows, i32([0] * S), i32([n + 5 for n in lens]), pool, bs)
    assert int(used) == sum(-(-(n + 5) // bs) for n in lens)
    pages = torch.zeros(S * width, nkv, F.kv4_page_bytes(bs, hd), dtype=torch.uint8, device=dev)
    total = sum(lens)
    _, _, slots = F.build_slot_map(table, rows, i32([0] * S), i32(lens), bs, total)
    kv = torch.randn(2, total, nkv, hd, generator=g).to(torch.bfloat16).to(dev)
    F.kv4_append_(kv[0], kv[1], slots, pages)
    qkv = torch.zeros(S, (nh + 2 * nkv) * hd, dtype=torch.bfloat16, device=dev)
    head = (torch.randn(V, nh * hd, generator=g) * 0.2).to(torch.bfloat16).to(dev)
    pos, ctx, active = i32(lens), i32([n + 1 for n in lens]), torch.tensor([True, True, False, True, True], device=dev)
    keep = {}

    def step():
        k, v = qkv[:, nh * hd : (nh + nkv) * hd].view(S, nkv, hd), qkv[:, (nh + nkv) * hd :].view(S, nkv, hd)
        keep["slots"], keep["ctx"], plan = F.decode_slot_map(table, pos, ctx, active, bs)
        F.kv4_append_(k, v, keep["slots"], pages)
        keep["att"] = F.paged_decode_attention_kv4(qkv[:, : nh * hd].view(S, nh, hd), pages, table, keep["ctx"], scale, plan)
        keep["logits"] = keep["att"].view(S, nh * hd) @ head.t()
        keep["scores"] = F.token_scores(keep["logits"], keep["logits"].argmax(-1), 7)
        pos.add_(active.int())
        ctx.add_(active.int())

    state = [t.clone() for t in (pos, ctx, pages)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for t, s in zip((pos, ctx, pages), state):
        t.copy_(s)
    on = active.tolist()
    for n in range(5):
        qkv.copy_(torch.randn(qkv.shape, generator=g).to(torch.bfloat16))
        before = pages.clone()
        graph.replay()
        now = [m + n + 1 if a else 0 for m, a in zip(lens, on)]
        assert keep["ctx"].tolist() == now
        at = [m + n for m in lens]
        want = [int(table[i, p // bs]) * bs + p % bs if on[i] else -1 for i, p in enumerate(at)]
        assert keep["slots"].tolist() == want
        assert sorted(set((pages != before).any(-1).nonzero()[:, 0].tolist())) == sorted({s // bs for s in want if s >= 0})
        q = qkv[:, : nh * hd].view(S, nh, hd)
        out, off = attention_64(q, pages, table, now, bs, scale)
        assert (np.abs(keep["att"].double().cpu().numpy() - out) <= off + 2.0**-8 * np.abs(out) + 2.0**-24).all()
        rec, logits = keep["scores"], keep["logits"]
        lp, ent, lse, order, top_lp = scores_64(logits, logits.argmax(-1), 7, 1.0, V)
        tol = slack(logits, V, 1.0)
        assert torch.equal(rec.top_ids.cpu(), order) and ((rec.top_logprob.double().cpu() - top_lp).abs() <= 2 * tol[:, None]).all()
        assert ((rec.logprob.double().cpu() - lp).abs() <= 2 * tol).all()


@pytest.mark.gpu
def test_teacher_records_and_distillation_loss_on_the_device():
    cfg, P = small_gpu()
    teacher = TeacherServer(DecoderModel(cfg, P), topk=8)
    seq = list(range(30, 77))
    ids, lps = asyncio.run(teacher.compute_topk_logprobs(seq))
    hidden = DecoderModel(cfg, P).forward_hidden(PackedBatch.from_lengths(torch.tensor(seq, device="cuda"), [len(seq)], device="cuda")).detach()
    logits = hidden @ P.lm_head_weight.t()
    _, _, _, order, top_lp = scores_64(logits, torch.zeros(len(seq), dtype=torch.int64), 8, 1.0, logits.shape[1])
    tol = 2 * slack(logits, logits.shape[1], 1.0)[:-1, None]
    assert torch.equal(ids, order[:-1]) and ((lps.double() - top_lp[:-1]).abs() <= tol).all()
    one = TeacherServer(DecoderModel(cfg, P), topk=0)
    i, l = asyncio.run(one.compute_topk_logprobs(seq))
    assert i[:, 0].tolist() == seq[1:]
    want = torch.log_softmax(logits.double(), -1).cpu()[:-1].gather(1, i)
    assert ((l.double() - want).abs() <= tol).all()
    # the loss on the teacher's support, and its gradient, against the host's form in 64 bits
    student = torch.randn(len(seq) - 1, logits.shape[1], device="cuda", requires_grad=True)
    conf = DistillationLossConfig(log_prob_min_clamp=None)
    out = compute_forward_kl_topk(student, lps.cuda(), ids.cuda(), conf)
    (grad,) = torch.autograd.grad(out["distillation_losses"].sum(), student)
    x = student.detach().double().cpu().requires_grad_(True)
    ref = (lps.double().exp() * (lps.double() - torch.log_softmax(x, -1).gather(1, ids))).sum(-1)
    (g64,) = torch.autograd.grad(ref.sum(), x)
    # weights of the support sum to at most 1: the loss is off by the slack of a log-prob and some fp32 roundings of numbers below 32
    t = 2 * slack(student.detach(), student.shape[1], 1.0) + 64 * 2.0**-24
    assert ((out["distillation_losses"].double().cpu() - ref.detach()).abs() <= t).all()
    assert ((grad.double().cpu() - g64).abs() <= (t[:, None] + 2.0**-22) * (g64.abs() + torch.softmax(x.detach(), -1)) + 2.0**-24 * lps.double().exp().max()).all()
