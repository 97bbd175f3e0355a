"""Sequences cut back to a budget of cached rows, within the limits of a deployment: rows a step, scratch, pages."""
import pytest
import torch

from tensorrt_edge_llm_b200 import AutoModel
from tensorrt_edge_llm_b200.config import tiny_llama_config
from tensorrt_edge_llm_b200.runtime.kv_cache import KVCacheManager
from tensorrt_edge_llm_b200.runtime.llm import LLM
from tensorrt_edge_llm_b200.runtime.runner import ModelRunner, SamplingParams


def _cfg():
    return tiny_llama_config(num_hidden_layers=2, vocab_size=256, dtype="float32", head_dim=64, num_attention_heads=4, num_key_value_heads=2, hidden_size=128,
                             max_position_embeddings=512)


def _prompts(*lens):
    g = torch.Generator().manual_seed(6)
    return [torch.randint(0, 256, (n,), generator=g).tolist() for n in lens]


@pytest.mark.parametrize("most,vote_bytes", [(48, 512 << 20), (16, 512 << 20), (8192, 1), (80, 4 * 4 * 32 * 2 * 150)])
def test_votes_keep_within_the_rows_of_a_step_and_their_scratch(most, vote_bytes):
    """The prompts' last rows vote a few sequences at a time; what they vote for is the same."""
    cfg, prompts = _cfg(), _prompts(150, 20, 33, 100, 70)
    model = AutoModel.from_config(cfg, random_init=0)

    def run(limit, bytes_):
        kv = KVCacheManager(cfg, num_pages=80, page_size=16, max_seats=5, max_pages_per_seq=16, kv_dtype="nvfp4", keep_weights=True)
        r = ModelRunner(model, kv, max_num_tokens=limit)
        r.kv_budget, r.VOTE_BYTES = 400, bytes_
        rows, scratch = [], []
        step = r._meta

        def spy(seats, q_lens, *a, **kw):
            meta = step(seats, q_lens, *a, **kw)
            rows.append(meta.num_tokens)
            return meta

        r._meta = spy
        model_step = r.step

        def spy_step(seats, toks, **kw):
            if kw.get("votes", True):
                scratch.append((len(seats), 4 * 4 * max(map(len, toks)) * len(seats) * max(kv.lengths[s] + len(t) for s, t in zip(seats, toks))))
            return model_step(seats, toks, **kw)

        r.step = spy_step
        return r.prefill(list(range(5)), prompts), rows, scratch, kv

    want, _, one, kv_a = run(8192, 512 << 20)
    got, rows, scratch, kv_b = run(most, vote_bytes)
    assert len(one) == 1 and len(scratch) > 1
    assert max(rows) <= most and all(n == 1 or b <= vote_bytes for n, b in scratch)
    assert torch.allclose(got, want, rtol=1e-3, atol=1e-3 * float(want.abs().max()))
    for s, p in enumerate(prompts):
        assert kv_b.lengths[s] == len(p)
        slot = torch.arange(len(p))
        a, b = (k.weights[:, k.table[s].long()[slot // 16], :, slot % 16] for k in (kv_a, kv_b))
        if most >= 32:              # as many voters: one a row and query head
            assert torch.allclose(a, b, atol=1e-2) and abs(float(b.sum()) - min(32, len(p)) * 4 * 2) < 1e-1
        else:
            assert abs(float(b.sum()) - most * 4 * 2) < 1e-1


def test_a_generation_that_starts_has_the_pages_to_end():
    """Pages for a cut and for what a sequence grows to are there before the first step, or the call is refused before it."""
    prompts = _prompts(100, 30)
    kw = dict(device="cpu", max_batch_size=2, max_input_len=256, max_kv_cache_capacity=336, page_size=16, kv_cache_dtype="nvfp4", random_init_seed=0, kv_budget=48)
    sp = SamplingParams(max_tokens=150, ignore_eos=True)
    want = [o.token_ids for o in LLM(_cfg(), **kw).generate(prompts, sp)]
    enough = 2 * 8 + 3                       # 113 rows of either sequence, 48 of a cut
    llm = LLM(_cfg(), kv_pages=enough, **kw)
    for _ in range(2):
        assert [o.token_ids for o in llm.generate(prompts, sp)] == want
    logits = LLM(_cfg(), kv_pages=enough, **kw).generate(prompts, SamplingParams(max_tokens=150, temperature=0.7, seed=1, ignore_eos=True))
    assert [len(o.token_ids) for o in logits] == [150, 150]
    short = LLM(_cfg(), kv_pages=enough - 1, **kw)
    steps = []
    short.runner.step = lambda *a, **k: steps.append(1)
    with pytest.raises(Exception, match="page|pool|exhaust"):
        short.generate(prompts, sp)
    assert not steps
    with pytest.raises(ValueError):
        LLM(_cfg(), kv_pages=10, **kw)
    LLM(_cfg(), kv_pages=11, **kw).generate([prompts[1]], sp)
    kv = KVCacheManager(_cfg(), num_pages=4, max_seats=1, max_pages_per_seq=2, kv_dtype="nvfp4")
    with pytest.raises(ValueError):
        kv.hold_spare(16)


def test_several_tokens_at_once_stay_within_what_a_sequence_may_grow_to():
    """Grammar-forced tokens ride along with a sampled one."""
    llm = LLM(_cfg(), device="cpu", max_batch_size=1, max_input_len=64, max_kv_cache_capacity=128, page_size=16, kv_cache_dtype="nvfp4", random_init_seed=0, kv_budget=63)
    r = llm.runner
    r.prefill([0], _prompts(60))
    r.decode_greedy([0], torch.tensor([3], dtype=torch.int32), 66)
    total = r.kv.lengths[0] + r.dropped.get(0, 0)
    assert r.kv.lengths[0] > 120                    # nine more rows would not fit its 128
    r.step([0], [[5, 6, 7, 8, 9, 10, 11, 12, 13]])
    assert r.kv.lengths[0] == 63 + 9 and r.kv.lengths[0] + r.dropped[0] == total + 9


def test_a_generation_that_would_run_out_of_positions_is_refused_before_it_starts():
    """A sequence that drops rows goes on behind all its tokens: 512 positions here."""
    llm = LLM(_cfg(), device="cpu", max_batch_size=1, max_input_len=512, max_kv_cache_capacity=512, page_size=16, kv_cache_dtype="nvfp4", random_init_seed=0, kv_budget=48)
    for sp in (dict(), dict(temperature=0.9, seed=1)):
        assert len(llm.generate(_prompts(480), SamplingParams(max_tokens=33, ignore_eos=True, **sp))[0].token_ids) == 33
        step, runs = llm.runner.step, []
        llm.runner.step = lambda *a, **k: runs.append(1) or step(*a, **k)
        with pytest.raises(ValueError, match="positions"):
            llm.generate(_prompts(480), SamplingParams(max_tokens=34, ignore_eos=True, **sp))
        llm.runner.step = step
        assert not runs
