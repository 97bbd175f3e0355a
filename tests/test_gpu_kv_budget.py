"""Sequences cut back to a budget of cached rows on the GPU: the captured decode step keeps account as the eager one does, and goes on after a cut."""
import pytest
import torch

from tensorrt_edge_llm_b200.config import tiny_llama_config
from tensorrt_edge_llm_b200.ops import build_step_meta
from tensorrt_edge_llm_b200.runtime.llm import LLM
from tensorrt_edge_llm_b200.runtime.runner import SamplingParams

pytestmark = pytest.mark.gpu


def _llm(budget, layers=2):
    cfg = tiny_llama_config(num_hidden_layers=layers, vocab_size=256, dtype="bfloat16", head_dim=64, num_attention_heads=4, num_key_value_heads=2, hidden_size=256,
                            max_position_embeddings=512)
    return LLM(cfg, device="cuda", max_batch_size=3, max_input_len=256, max_kv_cache_capacity=336, page_size=16, kv_cache_dtype="nvfp4", random_init_seed=0,
               kv_budget=budget)


def _prompts(*lens):
    g = torch.Generator().manual_seed(5)
    return [torch.randint(0, 256, (n,), generator=g).tolist() for n in lens]


@pytest.mark.parametrize("graphs", [True, False])
def test_decode_steps_keep_account_of_their_weights(graphs):
    llm = _llm(256)
    r, kv, prompts = llm.runner, llm.kv, _prompts(100, 40, 7)
    r.use_cuda_graphs = graphs
    for round_ in range(2):                                  # the second run replays the graph that the first one captured
        logits = r.prefill([0, 1, 2], prompts)
        r.decode_greedy([0, 1, 2], logits.argmax(-1).to(torch.int32), 20)
        torch.cuda.synchronize()
        assert kv.lengths[:3] == [120, 60, 27]
        for seat, n in enumerate((100, 40, 7)):
            slots = torch.arange(n + 20)
            w = kv.weights[:, kv.table[seat, slots // 16].long().cuda(), :, (slots % 16).cuda()]        # [rows, layers, heads]
            spent = (min(n, 32) + 20) * 2                    # every voter spends one per query head of a KV head
            # sums of some 2^7 additions of parts, each off by the rounding of an fp16 probability (2^-11) or of fp32
            assert torch.allclose(w.double().sum(0), torch.full((2, 2), float(spent), dtype=torch.float64, device="cuda"), rtol=2e-3)
            assert (w[-1] > 0).all() and bool((w >= 0).all())
        for s in range(3):
            kv.free(s)


@pytest.mark.parametrize("graphs", [True, False])
def test_decode_goes_on_after_a_cut(graphs):
    llm = _llm(48)
    r, kv, prompts = llm.runner, llm.kv, _prompts(150, 60)
    r.use_cuda_graphs = graphs
    logits = r.prefill([0, 1], prompts)
    assert kv.lengths[:2] == [48, 60] and r.dropped == {0: 102}
    toks = r.decode_greedy([0, 1], logits.argmax(-1).to(torch.int32), 80)
    total = [kv.lengths[s] + r.dropped.get(s, 0) for s in (0, 1)]
    assert total == [230, 140] and max(kv.lengths[:2]) <= 48 + 65 and r.dropped[1] > 0
    # the next token is that of a step over the rows that are there, at the positions behind all tokens
    before = kv.pool.clone()
    r.trim([0, 1])
    if not torch.equal(kv.pool, before):
        before = kv.pool.clone()
    past = list(kv.lengths[:2])
    nxt = r.decode_greedy([0, 1], toks[:, -1], 1)[:, 0].long()
    meta = build_step_meta([1, 1], past, kv.table_rows([0, 1]), 16, positions=total, device="cuda")
    want = llm.model(toks[:, -1].to("cuda", torch.int32), meta, before).float()
    # bf16 layers round by other orders of sums at most; the chosen logit is the largest within some steps of bf16
    best = want.max(-1).values
    assert bool((want[torch.arange(2), nxt.to(want.device)] >= best - 2 ** -5 * want.abs().amax(-1)).all())
    wrong = llm.model(toks[:, -1].to("cuda", torch.int32), build_step_meta([1, 1], past, kv.table_rows([0, 1]), 16, device="cuda"), before).float()
    assert not torch.allclose(want, wrong, atol=1e-3)        # positions that forgot the dropped rows would show


def test_generate_under_a_budget_ends_clean():
    llm = _llm(48)
    free = llm.kv.native.free_pages if llm.kv.native is not None else llm.kv.alloc.free_pages
    for sp in (SamplingParams(max_tokens=150, ignore_eos=True), SamplingParams(max_tokens=90, temperature=0.7, seed=2, ignore_eos=True)):
        outs = llm.generate(_prompts(100, 30, 200), sp)
        assert [len(o.token_ids) for o in outs] == [sp.max_tokens] * 3
    for s in range(3):
        llm.kv.free(s)
    assert (llm.kv.native.free_pages if llm.kv.native is not None else llm.kv.alloc.free_pages) == free


def test_requests_in_flight_over_four_bit_pages():
    """Eleven requests share the captured steps of 16 rows, whose last row stands there several times."""
    cfg = tiny_llama_config(num_hidden_layers=2, vocab_size=256, dtype="bfloat16", head_dim=64, num_attention_heads=4, num_key_value_heads=2, hidden_size=256)
    kw = dict(device="cuda", max_input_len=128, max_kv_cache_capacity=192, page_size=16, kv_cache_dtype="nvfp4", random_init_seed=0)
    flight = LLM(cfg, max_batch_size=16, enable_in_flight_batching=True, enable_prefix_cache=True, **kw)
    prompts = _prompts(60, 3, 100, 33, 17, 48, 5, 90, 77, 64, 21)
    outs = [o.token_ids for o in flight.generate(prompts, SamplingParams(max_tokens=24, ignore_eos=True))]
    alone = LLM(cfg, max_batch_size=1, **kw)
    for p, out in zip(prompts, outs):
        assert len(out) == 24
        alone.kv.free(0)
        logits = alone.runner.step([0], [p + out[:-1]], logits_all=True)[len(p) - 1:].float()
        # steps of one row and whole prompts round by other orders of sums and by 16-bit copies: the token taken is the largest within some steps of bf16
        assert bool((logits[torch.arange(24), torch.tensor(out)] >= logits.max(-1).values - 2 ** -5 * logits.abs().amax(-1)).all())
