"""Four-bit cache pages on the host: the format, the write, attention, accumulated weights and eviction against 64-bit oracles, and refusals."""
import math

import pytest
import torch

from fp4_kv_cases import make_step, oracle_attention, oracle_evict, page_values
from tensorrt_edge_llm_b200 import ops
from tensorrt_edge_llm_b200.ops import build_step_meta
from tensorrt_edge_llm_b200.ops import reference as ref


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
            rows = past + (ql if new else 0)
            for slot in range(staged.page_table.shape[1] * 64):
                got = stage[staged.page_table[s, slot // 64], :, :, slot % 64]
                want = vals[meta.page_table[s, slot // 32], :, :, slot % 32].bfloat16() if slot < rows else torch.zeros(())
                assert (got == want).all()


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
