"""Sequences cut back to a budget of cached rows: which rows stay, where later rows stand, and what a whole generation does."""
import pytest
import torch

from tensorrt_edge_llm_b200 import AutoModel
from tensorrt_edge_llm_b200.config import tiny_llama_config
from tensorrt_edge_llm_b200.ops import build_step_meta
from tensorrt_edge_llm_b200.ops import reference as ref
from tensorrt_edge_llm_b200.runtime.kv_cache import KVCacheManager
from tensorrt_edge_llm_b200.runtime.llm import LLM
from tensorrt_edge_llm_b200.runtime.runner import ModelRunner, SamplingParams


def _cfg(**kw):
    return tiny_llama_config(num_hidden_layers=2, vocab_size=256, dtype="float32", head_dim=64, num_attention_heads=4, num_key_value_heads=2, hidden_size=128,
                             max_position_embeddings=512, **kw)


def test_steps_after_a_cut_go_on_over_the_rows_that_stayed():
    cfg = _cfg()
    model = AutoModel.from_config(cfg, random_init=0)
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, 256, (n,), generator=g).tolist() for n in (150, 60)]
    kv = KVCacheManager(cfg, num_pages=40, page_size=16, max_seats=2, max_pages_per_seq=16, kv_dtype="nvfp4", keep_weights=True)
    r = ModelRunner(model, kv)
    r.kv_budget = 40
    r.BUDGET_SLACK = 0
    free = kv.native.free_pages if kv.native is not None else kv.alloc.free_pages
    before = {}
    shorten = kv.shorten

    def spy(seat, keep, first, recent):           # what the cache held before the cut
        before[seat] = (kv.pool.clone(), kv.weights.clone(), kv.table_rows([seat]).clone(), kv.lengths[seat])
        return shorten(seat, keep, first, recent)

    kv.shorten = spy
    r.trim = lambda seats, slack=0: ModelRunner.trim(r, seats, slack)
    r.prefill([0, 1], prompts)
    assert kv.lengths[:2] == [40, 40] and r.dropped == {0: 110, 1: 20}
    assert len(kv.pages_of(0)) == 3 and len(kv.pages_of(1)) == 3
    assert (kv.native.free_pages if kv.native is not None else kv.alloc.free_pages) == free - 6
    for seat, n in ((0, 150), (1, 60)):
        pool, w, table, length = before[seat]
        assert length == n
        for layer in range(2):
            slot = torch.arange(n)
            got = w[layer][table[0].long()[slot // 16], :, slot % 16]
            # every voter spends one per query head; keys that only the voters saw have part of it
            assert abs(float(got.sum()) - 32 * 4) < 1e-2
            new = torch.zeros(1, 3, dtype=torch.int32)
            new[0] = torch.arange(pool.shape[1], pool.shape[1] + 3)
            room = torch.cat([pool[layer], torch.zeros_like(pool[layer][:3])])
            kept = ref.kv_evict(room, torch.cat([w[layer], torch.zeros_like(w[layer][:3])]), table, torch.tensor([n]), new, 40, r.BUDGET_FIRST, 10)
            assert kept.shape == (1, 2, 40) and kept[0, 0, :4].tolist() == [0, 1, 2, 3] and kept[0, 0, -10:].tolist() == list(range(n - 10, n))
            a, b = ref.fp4_page_parts(room), ref.fp4_page_parts(kv.pool[layer])
            for j in range(40):
                for x, y in zip(a, b):
                    assert torch.equal(x[pool.shape[1] + j // 16, :, :, j % 16], y[kv.table[seat, j // 16], :, :, j % 16])
    # a step stands at the positions behind all tokens, and sees the rows that stayed
    twin = KVCacheManager(cfg, num_pages=40, page_size=16, max_seats=2, max_pages_per_seq=16, kv_dtype="nvfp4")
    twin.pool.copy_(kv.pool)
    meta = build_step_meta([1, 1], [40, 40], kv.table_rows([0, 1]), 16, positions=[150, 60])
    for s in (0, 1):
        kv.reserve(s, 41)
    meta.page_table = kv.table_rows([0, 1]).to(torch.int32)
    want = model(torch.tensor([7, 9], dtype=torch.int32), meta, twin.pool)
    got = r.step([0, 1], [[7], [9]])
    assert torch.equal(got, want)
    assert kv.lengths[:2] == [40, 40] and r.dropped == {0: 111, 1: 21}       # cut back again
    kv.free(0)
    r.prefill([0], [prompts[1][:20]])                                        # a fresh sequence stands at its own positions
    assert r.dropped == {1: 21}


def test_generation_within_the_budget_is_unchanged_and_beyond_it_stays_in_bounds():
    cfg = _cfg()
    g = torch.Generator().manual_seed(4)
    prompts = [torch.randint(0, 256, (n,), generator=g).tolist() for n in (100, 30)]
    kw = dict(device="cpu", max_batch_size=2, max_input_len=256, max_kv_cache_capacity=336, page_size=16, kv_cache_dtype="nvfp4", random_init_seed=0)
    plain = LLM(cfg, **kw)
    for sp in (SamplingParams(max_tokens=40, ignore_eos=True), SamplingParams(max_tokens=12, temperature=0.8, seed=3, ignore_eos=True)):
        want = [o.token_ids for o in plain.generate(prompts, sp)]
        assert [o.token_ids for o in LLM(cfg, kv_budget=256, **kw).generate(prompts, sp)] == want
        tight = LLM(cfg, kv_budget=48, **kw)
        lengths = []
        run = tight.runner._decode_greedy_run
        tight.runner._decode_greedy_run = lambda s, f, n: (run(s, f, n), lengths.append(max(tight.kv.lengths[:2])))[0]
        outs = tight.generate(prompts, SamplingParams(**{**sp.__dict__, "max_tokens": 150}))
        assert all(len(o.token_ids) == 150 for o in outs) and all(x <= 48 + 64 + 1 for x in lengths)
        assert sp.temperature > 0 or len(lengths) > 1
        again = [o.token_ids for o in tight.generate(prompts, SamplingParams(**{**sp.__dict__, "max_tokens": 150}))]
        assert again == [o.token_ids for o in outs]                          # seats are left clean


def test_budget_refusals():
    cfg = _cfg()
    kw = dict(device="cpu", max_batch_size=1, max_input_len=64, max_kv_cache_capacity=160, random_init_seed=0)
    for bad in (dict(kv_budget=64), dict(kv_budget=64, kv_cache_dtype="fp8"), dict(kv_budget=8, kv_cache_dtype="nvfp4"), dict(kv_budget=96, kv_cache_dtype="nvfp4"),
                dict(kv_budget=64, kv_cache_dtype="nvfp4", enable_in_flight_batching=True)):
        with pytest.raises(ValueError):
            LLM(cfg, **kw, **bad)
    with pytest.raises(ValueError):
        LLM(_cfg(sliding_window=32), kv_budget=64, kv_cache_dtype="nvfp4", **kw)
    kv = KVCacheManager(cfg, num_pages=4, max_seats=1, max_pages_per_seq=2, kv_dtype="nvfp4")
    with pytest.raises(ValueError):
        kv.shorten(0, 10, 1, 1)
