"""Four-bit cache pages on the host: the format, the write, attention, accumulated weights and eviction against 64-bit oracles, and refusals."""
import math

import pytest
import torch

from fp4_kv_cases import make_step, oracle_attention, oracle_evict, page_values
from tensorrt_edge_llm_b200 import AutoModel, ops
from tensorrt_edge_llm_b200.config import QuantConfig, tiny_llama_config
from tensorrt_edge_llm_b200.ops import build_step_meta
from tensorrt_edge_llm_b200.ops import reference as ref
from tensorrt_edge_llm_b200.runtime.kv_cache import KVCacheManager
from tensorrt_edge_llm_b200.runtime.runner import ModelRunner


@pytest.mark.parametrize("d", [64, 128, 256])
def test_write_quantises_the_rows_of_a_16_bit_cache(d):
    """A level is at most half a gap away (a sixth of the block's largest value, whose scale is rounded by 2^-4): a value is off by at most
    (1 + 2^-4) / 6 of the largest of its block, and by 2^-4 more where the block scale was rounded down."""
    q_lens, past, hq, hkv, page = [3, 1, 20], [0, 37, 13], 4, 2, 16
    meta, layer, scales, g = make_step(q_lens, past, page, hkv, d)
    t = sum(q_lens)
    qkv = torch.randn(t, (hq + 2 * hkv) * d, generator=g).bfloat16()
    cs = ref.rope_cos_sin(64, d, 1e4)
    w = (1 + 0.1 * torch.randn(d, generator=g)).bfloat16()
    plain = torch.zeros(layer.shape[0], 2, hkv, page, d, dtype=torch.bfloat16)
    q_want = ref.rope_kv_write(qkv, plain, meta, cs, hq, hkv, d, w, w)
    before = layer.clone()
    stage = torch.zeros(layer.shape[0], 2, hkv, page, d, dtype=torch.bfloat16)
    q = ops.rope_kv_write_fp4(qkv, layer, meta, cs, hq, hkv, d, scales, w, w, stage=stage, stage_table=meta.page_table)
    assert torch.equal(q, q_want)
    got = page_values(layer, scales)
    touched = torch.zeros(layer.shape[0], page, dtype=torch.bool)
    for r in range(t):
        s = int(meta.seq_ids[r])
        slot = past[s] + r - int(meta.q_start[s])
        pg, at = int(meta.page_table[s, slot // page]), slot % page
        touched[pg, at] = True
        want = plain[pg, :, :, at].double().unflatten(-1, (-1, 16))
        top = want.abs().amax(-1, keepdim=True)
        assert ((got[pg, :, :, at].unflatten(-1, (-1, 16)) - want).abs() <= top * ((1 + 2 ** -4) / 6 + 2 ** -4)).all()
        assert torch.equal(stage[pg, :, :, at].double(), got[pg, :, :, at].bfloat16().double())
    # everything else is as it was
    c0, f0 = ref.fp4_page_parts(before)
    c1, f1 = ref.fp4_page_parts(layer)
    for a, b in ((c0, c1), (f0, f1)):
        assert torch.equal(a.permute(0, 3, 1, 2, 4)[~touched], b.permute(0, 3, 1, 2, 4)[~touched])


def test_borders_round_to_the_even_code_and_odd_values_keep_their_block():
    x = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -0.75, -5.0, 0.0, -0.0, 6.0, 0.2500001, 4.9999])
    codes, sf, vals = ref.fp4_encode_rows(x, torch.tensor(1.0))
    assert vals.tolist() == [6.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, -0.0, -1.0, -4.0, 0.0, -0.0, 6.0, 0.5, 4.0]
    y = torch.stack([torch.full((16,), math.inf), torch.zeros(16), torch.full((16,), 1e-30), torch.tensor([math.nan] + [1.0] * 15)])
    _, sf, vals = ref.fp4_encode_rows(y, torch.tensor(1.0))
    assert (vals[0] == 6 * 448).all() and (vals[1] == 0).all() and (vals[2] == 0).all() and vals[3].isnan().all()


STEPS = [([1], [0], 0), ([1, 1, 1], [5, 64, 130], 0), ([3, 0, 2], [40, 7, 0], 0), ([2, 5], [300, 17], 33), ([1], [400], 64)]


@pytest.mark.parametrize("q_lens,past,window", STEPS)
@pytest.mark.parametrize("sunk", [False, True])
def test_attention_and_weights(q_lens, past, window, sunk):
    hq, hkv, d = 6, 2, 64
    meta, layer, scales, g = make_step(q_lens, past, 16, hkv, d, seed=len(past) + window, window=window)
    q = torch.randn(sum(q_lens), hq, d, generator=g) * 2
    sinks = torch.randn(hq, generator=g) if sunk else None
    w = torch.rand(layer.shape[0], hkv, 16, generator=g)
    want, want_w = oracle_attention(q, layer, meta, d ** -0.5, scales, window, sinks, w, 0.9)
    got = ops.paged_attention_fp4(q, layer, meta, d ** -0.5, scales, sliding_window=window or None, sinks=sinks, weights=w, decay=0.9)
    # 32-bit sums: 64 features, a few hundred keys
    assert (got.double() - want).abs().max() < 2e-5 * want.abs().max()
    assert (w.double() - want_w).abs().max() < 1e-5


def test_stage_holds_the_rows_and_zeros_behind_them():
    meta, layer, scales, _ = make_step([2, 1], [70, 3], 32, 2, 64)
    vals = page_values(layer, scales)
    for new in (False, True):
        stage, staged = ops.kv_fp4_stage(layer, meta, scales, torch.bfloat16, new_rows=new)
        for s, (ql, past) in enumerate(((2, 70), (1, 3))):
            for slot in range(staged.page_table.shape[1] * 64):
                if past <= slot < past + ql and not new:          # left for the write
                    continue
                got = stage[staged.page_table[s, slot // 64], :, :, slot % 64]
                want = vals[meta.page_table[s, slot // 32], :, :, slot % 32].bfloat16() if slot < past + ql else torch.zeros(())
                assert (got == want).all()


@pytest.mark.parametrize("d", [64, 128, 256])
def test_commit_path_moves_codes_and_scales(d):
    g = torch.Generator().manual_seed(d)
    pool = torch.randint(0, 256, (2, 6, 2, 3, 16, d * 9 // 16), generator=g, dtype=torch.uint8)
    table = torch.tensor([[4, 1, 0], [2, 5, -1]], dtype=torch.int32)
    past, path, plen = torch.tensor([14, 3]), torch.tensor([[0, 2, 5, 6], [0, 1, 4, 0]]), torch.tensor([4, 3])
    want = pool.clone()
    for layer in range(2):
        src, dst = ref.fp4_page_parts(pool[layer]), ref.fp4_page_parts(want[layer])
        for b in range(2):
            for j in range(1, int(plen[b])):
                a, z = int(past[b] + path[b, j]), int(past[b]) + j
                for x, y in zip(src, dst):
                    y[table[b, z // 16], :, :, z % 16] = x[table[b, a // 16], :, :, a % 16]
    ops.kv_commit_path(pool, table, past, path, plen)
    assert torch.equal(pool, want)


def _run(model, cfg, prompts, feed, kv_dtype, page=64, max_tokens=8192):
    kv = KVCacheManager(cfg, num_pages=40, page_size=page, max_seats=2, max_pages_per_seq=16, kv_dtype=kv_dtype)
    r = ModelRunner(model, kv, max_num_tokens=max_tokens)
    out = [r.prefill([0, 1], prompts)]
    for toks in feed:
        out.append(r.step([0, 1], [[t] for t in toks]))
    return torch.stack(out), kv


@pytest.mark.parametrize("head,page,chunk", [(64, 64, 8192), (128, 16, 64), (64, 32, 32)])
def test_model_over_four_bit_pages_is_the_model_whose_rows_are_rounded(head, page, chunk, monkeypatch):
    """The same logits as a 16-bit cache whose rows are rounded to what four bits hold as they are written, in whole and chunked prompts and steps."""
    cfg = tiny_llama_config(num_hidden_layers=2, vocab_size=256, dtype="float32", head_dim=head, num_attention_heads=4, num_key_value_heads=2, hidden_size=128)
    model = AutoModel.from_config(cfg, random_init=0)
    g = torch.Generator().manual_seed(7)
    prompts = [torch.randint(0, 256, (n,), generator=g).tolist() for n in (90, 67)]
    feed = torch.randint(0, 256, (4, 2), generator=g).tolist()
    for layer in model.model.layers:
        layer.self_attn.kv_scales.copy_(torch.tensor([0.003, 0.002]))
    got, kv4 = _run(model, cfg, prompts, feed, "nvfp4", page, chunk)
    assert kv4.pool.dtype == torch.uint8 and kv4.bytes_per_token == 2 * 2 * 2 * head * 9 // 16
    plain = ref.rope_kv_write

    def rounded(qkv, kv_layer, meta, *a, **kw):
        q = plain(qkv, kv_layer, meta, *a, **kw)
        sid = meta.seq_ids.long()
        slot = meta.past_len.long()[sid] + torch.arange(qkv.shape[0]) - meta.q_start.long()[sid]
        pg, at = meta.page_table.long()[sid, slot // page], slot % page
        kv_layer[pg, :, :, at] = ref.fp4_encode_rows(kv_layer[pg, :, :, at].float(), torch.tensor([0.003, 0.002]).view(1, 2, 1, 1))[2]
        return q

    full, _ = _run(model, cfg, prompts, feed, "model", page, chunk)
    monkeypatch.setattr(ops, "rope_kv_write", rounded)
    want, kv16 = _run(model, cfg, prompts, feed, "model", page, chunk)
    assert kv16.bytes_per_token * 9 == kv4.bytes_per_token * 64       # fp32 pool here
    # 32-bit sums of another order; a code on a border may fall to the other side of it in a later layer
    assert (got - want).norm() < 1e-3 * want.norm()
    cos = torch.nn.functional.cosine_similarity(full.flatten(1), got.flatten(1), dim=1)
    assert float(cos.min()) > 0.97


def test_cache_manager_chooses_and_refuses_four_bits():
    cfg = tiny_llama_config(num_hidden_layers=2, vocab_size=256, dtype="bfloat16", head_dim=64, num_attention_heads=4, num_key_value_heads=2, hidden_size=128)
    make = lambda c=cfg, **kw: KVCacheManager(c, num_pages=4, max_seats=1, max_pages_per_seq=2, **{"page_size": 64, **kw})
    assert make(kv_dtype="nvfp4").kv_fp4 and not make().kv_fp4 and not make(kv_dtype="model").kv_fp4
    cfg.quant = QuantConfig(kv_cache_quant="nvfp4")
    assert make().kv_fp4 and make().pool.shape == (2, 4, 2, 2, 64, 36) and not make(kv_dtype="model").kv_fp4
    odd = tiny_llama_config(num_hidden_layers=2, vocab_size=256, dtype="bfloat16", head_dim=32, num_attention_heads=4, num_key_value_heads=2, hidden_size=128)
    for c, kw in ((odd, {}), (cfg, dict(page_size=48)), (cfg, dict(page_size=8))):
        with pytest.raises(ValueError):
            make(c, kv_dtype="nvfp4", **kw)
    odd.quant = QuantConfig(kv_cache_quant="nvfp4")
    assert not make(odd).kv_fp4 and make(odd).pool.dtype == torch.bfloat16        # a checkpoint's own setting gives way
    with pytest.raises(TypeError):
        ops.cuda_ops().paged_attention(torch.zeros(1, 4, 64), make().pool[0], None, 0.1)


def test_native_configuration_counts_four_bit_rows(tmp_path):
    import json
    from tensorrt_edge_llm_b200.checkpoint.artifacts import runtime_config_dict
    from tensorrt_edge_llm_b200.config import parse_quant_config, qwen3_8b_config
    from tensorrt_edge_llm_b200.quantization.quantize import build_quant_config
    from tensorrt_edge_llm_b200.runtime import native as rt
    body = build_quant_config("nvfp4", kv_cache_quantization="nvfp4")
    (tmp_path / "hf_quant_config.json").write_text(json.dumps(body))
    assert body["quantization"]["kv_cache_quant_algo"] == "NVFP4" and parse_quant_config(str(tmp_path), {}).kv_cache_quant == "nvfp4"
    dense = qwen3_8b_config(dtype="float16", quant=QuantConfig(quant_type="nvfp4", group_size=16, kv_cache_quant="nvfp4"))
    c = rt.LLMEngineConfig.from_runtime_config(json.dumps(runtime_config_dict(dense, 64, 1024, 1216, 1), default=str))
    small = qwen3_8b_config(dtype="float16", num_hidden_layers=2, quant=dense.quant)
    assert KVCacheManager(small, num_pages=2, page_size=64, max_seats=1, max_pages_per_seq=2).bytes_per_token * 18 == c.kv_bytes_per_token() == 36 * 2 * 8 * 72


@pytest.mark.parametrize("kind", ["fp4", "fp8", "bf16"])
def test_evict_keeps_first_recent_and_heaviest(kind):
    g = torch.Generator().manual_seed(5)
    lengths, page, hkv, keep, first, recent = [50, 12, 0, 20, 21], 16, 2, 20, 3, 5
    n, wide, pages = 5, 4, 40
    table = torch.randperm(20, generator=g).int().view(n, wide)
    to = (20 + torch.randperm(n * 2, generator=g)).int().view(n, 2)
    w = torch.randint(0, 6, (pages, hkv, page), generator=g).float() / 4          # many ties
    w[table[0, 1], 0, 3] = math.nan
    layer = torch.randint(0, 256, (pages, 2, hkv, page, 36 if kind == "fp4" else 32), generator=g, dtype=torch.uint8)
    if kind != "fp4":
        layer = layer.view({"fp8": torch.float8_e4m3fn, "bf16": torch.bfloat16}[kind])
    want = oracle_evict(w, table, lengths, page, keep, first, recent)
    before, w0 = layer.clone(), w.clone()
    kept = ops.kv_evict(layer, w, table, torch.tensor(lengths, dtype=torch.int32), to, keep, first, recent)
    parts = lambda x: [v for v in ref.fp4_page_parts(x)] if kind == "fp4" else [x.view(torch.uint8)]
    changed = torch.zeros(pages, hkv, page, dtype=torch.bool)
    for s in range(n):
        for h in range(hkv):
            rows = want[s][h]
            assert kept[s, h].tolist() == rows + [-1] * (keep - len(rows))
            for j, i in enumerate(rows):
                dst, src = (int(to[s, j // page]), j % page), (int(table[s, i // page]), i % page)
                changed[dst[0], h, dst[1]] = True
                for a, b in zip(parts(layer), parts(before)):
                    assert torch.equal(a[dst[0], :, h, dst[1]], b[src[0], :, h, src[1]])
                assert torch.equal(w[dst[0], h, dst[1]], w0[src[0], h, src[1]]) or w0[src[0], h, src[1]].isnan()
    for a, b in zip(parts(layer), parts(before)):
        assert torch.equal(a.permute(0, 2, 3, 1, 4)[~changed], b.permute(0, 2, 3, 1, 4)[~changed])


def test_refusals():
    meta, layer, scales, g = make_step([2], [5], 16, 2, 64)
    q, qkv, cs = torch.randn(2, 4, 64), torch.randn(2, 8 * 64), torch.ones(32, 64)
    w = torch.zeros(layer.shape[0], 2, 16)
    for bad in (layer.view(torch.int8), layer[..., :35], layer[:, :1], layer[:, :, :, :8]):
        with pytest.raises(ValueError):
            ops.rope_kv_write_fp4(qkv, bad, meta, cs, 4, 2, 64, scales)
        with pytest.raises(ValueError):
            ops.paged_attention_fp4(q, bad, meta, 0.1, scales)
        with pytest.raises(ValueError):
            ops.kv_fp4_stage(bad, meta, scales, torch.bfloat16)
    with pytest.raises(ValueError):
        ops.rope_kv_write_fp4(qkv, layer, meta, cs, 4, 2, 64, scales, stage=torch.zeros(1, 2, 2, 16, 64))
    with pytest.raises(ValueError):
        ops.paged_attention_fp4(torch.randn(2, 5, 64), layer, meta, 0.1, scales)
    with pytest.raises(ValueError):
        ops.paged_attention_fp4(q, layer, meta, 0.0, scales)
    long = build_step_meta([200], [0], torch.zeros(1, 13, dtype=torch.int32), 16)
    with pytest.raises(ValueError):
        ops.paged_attention_fp4(torch.randn(200, 4, 64), layer, long, 0.1, scales, weights=w)
    table, to, n = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, 1, dtype=torch.int32), torch.tensor([20])
    for kw in (dict(keep=0), dict(keep=17), dict(keep=4, first=3, recent=2), dict(keep=4, first=-1)):
        with pytest.raises(ValueError):
            ops.kv_evict(layer, w, table, n, to, **kw)
    with pytest.raises(ValueError):
        ops.kv_evict(layer, w.double(), table, n, to, 4)
    with pytest.raises(ValueError):
        ops.kv_evict(layer, w, table, torch.tensor([1, 2]), to, 4)


def test_evict_takes_rows_without_a_page_last_and_the_earlier_first():
    g = torch.Generator().manual_seed(8)
    table = torch.tensor([[5, -1, 2, -1, 7]], dtype=torch.int32)
    w = -torch.rand(10, 1, 16, generator=g)
    w[2, 0, 4] = -math.inf
    w[0, 0, ::3] = math.nan                 # of a page that the table does not name
    layer = torch.randint(0, 256, (10, 2, 1, 16, 36), generator=g, dtype=torch.uint8)
    for keep in (30, 45, 60):
        got = ops.kv_evict(layer.clone(), w.clone(), table, torch.tensor([80], dtype=torch.int32), torch.tensor([[0, 1, 3, 4]], dtype=torch.int32), keep, 0, 0)[0, 0].tolist()
        there = sorted((i for i in range(80) if i // 16 in (0, 2, 4)), key=lambda i: (-float(w[table[0, i // 16], 0, i % 16]), i))
        gone = [i for i in range(80) if i // 16 in (1, 3)]
        assert got == sorted((there + gone)[:keep])


def test_requests_in_flight_over_four_bit_pages_are_the_static_ones():
    from tensorrt_edge_llm_b200.runtime.llm import LLM
    from tensorrt_edge_llm_b200.runtime.runner import SamplingParams
    cfg = tiny_llama_config(num_hidden_layers=2, vocab_size=256, dtype="float32", head_dim=64, num_attention_heads=4, num_key_value_heads=2, hidden_size=128)
    g = torch.Generator().manual_seed(9)
    head = torch.randint(0, 256, (40,), generator=g).tolist()
    prompts = [head + torch.randint(0, 256, (n,), generator=g).tolist() for n in (50, 3, 21)]          # a shared prefix of whole pages
    sp = SamplingParams(max_tokens=12, ignore_eos=True)
    kw = dict(device="cpu", max_batch_size=3, max_input_len=128, max_kv_cache_capacity=128, page_size=16, kv_cache_dtype="nvfp4", random_init_seed=0)
    want = [LLM(cfg, **kw).generate([p], sp)[0].token_ids for p in prompts]
    assert [o.token_ids for o in LLM(cfg, **kw).generate(prompts, sp)] == want
    flight = LLM(cfg, enable_in_flight_batching=True, enable_prefix_cache=True, **kw)
    assert [o.token_ids for o in flight.generate(prompts, sp)] == want
    assert [o.token_ids for o in flight.generate(prompts, sp)] == want


@pytest.mark.parametrize("flight", [False, True])
def test_draft_trees_over_four_bit_pages_are_lossless(flight):
    """Verification goes through 16-bit copies, steps read the pages in place, accepted rows move: the tokens are those of plain decoding."""
    from tensorrt_edge_llm_b200.runtime.llm import LLM
    from tensorrt_edge_llm_b200.runtime.runner import SamplingParams
    from tensorrt_edge_llm_b200.runtime.speculative import SpecConfig
    sizes = dict(vocab_size=256, dtype="float32", head_dim=64, num_attention_heads=4, num_key_value_heads=2, hidden_size=128)
    cfg, dcfg = tiny_llama_config(num_hidden_layers=4, **sizes), tiny_llama_config(num_hidden_layers=1, **sizes)
    dcfg.draft_type, dcfg.eagle3_target_hidden_size, dcfg.draft_vocab_size = "eagle3", 128, 0
    g = torch.Generator().manual_seed(12)
    prompts = [torch.randint(0, 256, (n,), generator=g).tolist() for n in (19, 34)]
    sp = SamplingParams(max_tokens=10, ignore_eos=True)
    kw = dict(device="cpu", max_batch_size=2, max_input_len=64, max_kv_cache_capacity=128, page_size=16, kv_cache_dtype="nvfp4", random_init_seed=0)
    want = [o.token_ids for o in LLM(cfg, **kw).generate(prompts, sp)]
    spec = LLM(cfg, draft_model=dcfg, speculative=SpecConfig(draft_steps=3, top_k=2, verify_tokens=8), enable_in_flight_batching=flight, **kw)
    assert spec.kv.kv_fp4 and [o.token_ids for o in spec.generate(prompts, sp)] == want
