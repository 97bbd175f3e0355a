"""Steps that are too long to read four-bit pages in place, on the GPU: tables with holes, trees and windows against a 64-bit oracle."""
from dataclasses import replace

import pytest
import torch

from fp4_expanded_cases import holey_step, oracle, poison_before_the_window
from fp4_kv_cases import make_step
from tensorrt_edge_llm_b200 import ops

pytestmark = pytest.mark.gpu


def bound(want, top, kq, dtype):
    """Codes times block scales have at most six significant bits: keys and values are exact in 16 bits.  Left are half a step of the result; half a step of the
    probabilities, of the largest value; scores whose 32-bit sums over 16 steps of a matrix product are off by 16 steps of 2^-22 of |q| |k| at most, a probability
    by as much and its sum again; and fp16 probabilities below 2^-14 of the largest, off by 2^-25 each, some thousand of them."""
    half = torch.finfo(dtype).eps / 2
    return half * want.abs() + (half + 2 * 2 ** -18 * kq + 2 ** -14) * top


# q_lens, past, query heads, KV heads, head size, page, missing logical pages, window, tree
STEPS = [([40], [100], 8, 2, 128, 64, [[0]], 0, False), ([70, 5, 300], [30, 200, 0], 8, 2, 128, 64, [[1], [0, 2], [2]], 0, False), ([600], [900], 32, 8, 128, 16, [[3, 50, 51, 70]], 0, False),
         ([40, 100], [260, 7], 16, 4, 64, 32, [[0, 3], [2]], 0, False), ([33], [500], 8, 2, 256, 16, [[0, 1, 20]], 0, False), ([8, 20], [300, 64], 4, 2, 128, 32, [[2, 5], [0]], 0, True),
         ([40], [130], 4, 2, 64, 16, [[3, 9]], 0, True), ([50], [700], 8, 2, 128, 64, [[9, 11]], 260, False), ([40], [700], 8, 2, 64, 64, [[9, 11]], 260, False),
         ([90], [38], 8, 2, 128, 128, [[0]], 0, False), ([90, 30], [38, 0], 8, 2, 64, 16, [list(range(8)), [0, 1]], 0, False), ([24], [3000], 8, 2, 128, 64, [[2, 3, 30]], 0, False)]


@pytest.mark.parametrize("q_lens,past,hq,hkv,d,page,missing,window,tree", STEPS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sunk", [False, True])
def test_holes_are_hidden_from_expanded_steps(q_lens, past, hq, hkv, d, page, missing, window, tree, dtype, sunk):
    meta, layer, scales, g = holey_step(q_lens, past, page, hkv, d, missing, seed=sum(past) + d, window=window, tree=tree)
    q = (torch.randn(sum(q_lens), hq, d, generator=g) * 2).to(dtype)
    sinks = torch.randn(hq, generator=g) if sunk else None
    want, top, kq = oracle(q, layer, meta, d ** -0.5, scales, window, sinks)
    got = ops.cuda_ops().paged_attention_fp4(q.cuda(), layer.cuda(), meta.to("cuda"), d ** -0.5, scales.cuda(), window or None, None if sinks is None else sinks.cuda(), direct=False)
    assert ((got.cpu().double() - want).abs() <= bound(want, top, kq, dtype)).all()
    assert torch.equal(got, ops.paged_attention_fp4(q.cuda(), layer.cuda(), meta.to("cuda"), d ** -0.5, scales.cuda(), sliding_window=window or None,
                                                    sinks=None if sinks is None else sinks.cuda())) or (not tree and max(q_lens) * hq // hkv <= ops.FP4_DIRECT_COLUMNS)


# q_lens, past, query heads, KV heads, head size, page, window; the first key that some row sees lies inside a tile of 16, 32, 64 and 128 keys
WINDOWS = [([1], [700], 8, 2, 128, 64, 130), ([1, 3], [333, 90], 10, 2, 64, 16, 45), ([2], [350], 4, 2, 256, 32, 40), ([5], [900], 16, 2, 128, 64, 257), ([8], [500], 16, 2, 128, 128, 100)]


@pytest.mark.parametrize("q_lens,past,hq,hkv,d,page,window", WINDOWS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("direct", [True, False])
def test_rows_that_a_window_hides_do_not_reach_the_outputs(q_lens, past, hq, hkv, d, page, window, dtype, direct):
    """A cached row with a NaN is seen while it is in the window and forgotten behind it, although the tile that holds it is still read."""
    meta, layer, scales, g = make_step(q_lens, past, page, hkv, d, seed=window + d)
    poison_before_the_window(meta, layer, window)
    q = (torch.randn(sum(q_lens), hq, d, generator=g) * 2).to(dtype)
    want, top, kq = oracle(q, layer, meta, d ** -0.5, scales, window)
    args = (layer.cuda(), meta.to("cuda"), d ** -0.5, scales.cuda(), window)
    got = ops.cuda_ops().paged_attention_fp4(q.cuda(), *args, direct=direct)
    assert ((got.cpu().double() - want).abs() <= bound(want, top, kq, dtype)).all()
    if direct:
        w = torch.zeros(layer.shape[0], hkv, page, device="cuda")
        for ctas in (None, 3, -1, -4):
            got = ops.cuda_ops().paged_attention_fp4(q.cuda(), *args, weights=w, ctas=ctas)
            assert ((got.cpu().double() - want).abs() <= bound(want, top, kq, dtype)).all() and w.isfinite().all()
    stage, staged = ops.kv_fp4_stage(layer.cuda(), args[1], args[3], dtype, window, True)
    plain = ops.paged_attention(q.cuda(), stage, staged, d ** -0.5, window)
    assert plain.isfinite().all()


@pytest.mark.parametrize("d", [64, 128, 256])
def test_copies_are_as_long_as_the_rows(d):
    """One long sequence beside short ones, 40 of them: the packed copy is the host's, the step's outputs are those of a step whose lengths the host does not
    know, and the memory is that of the rows, not of forty long sequences."""
    hkv, hq, page = 2, 8, 64
    q_lens, past = [1] * 39 + [70], [(7 * i) % 130 for i in range(38)] + [5000, 0]
    meta, layer, scales, g = make_step(q_lens, past, page, hkv, d, seed=d)
    q = (torch.randn(sum(q_lens), hq, d, generator=g) * 2).bfloat16().cuda()
    lg, m, sg = layer.cuda(), meta.to("cuda"), scales.cuda()
    want, host = ops.kv_fp4_stage(layer, meta, scales, torch.bfloat16, new_rows=True)
    got, staged = ops.kv_fp4_stage(lg, m, sg, torch.bfloat16, new_rows=True)
    assert torch.equal(staged.page_table.cpu(), host.page_table) and torch.equal(got.cpu(), want)
    assert got.shape[0] == sum(2 * max(1, -(-(a + b) // 128)) for a, b in zip(q_lens, past)) + 1
    del got
    loose = replace(m, host_lens=None, max_seq_len=6000)
    expect = ops.paged_attention_fp4(q, lg, loose, d ** -0.5, sg)
    ops.paged_attention_fp4(q, lg, m, d ** -0.5, sg)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = ops.paged_attention_fp4(q, lg, m, d ** -0.5, sg)
    used = torch.cuda.max_memory_allocated() - before
    assert used < 2 * (sum(q_lens) + sum(past) + 128 * 40) * 2 * hkv * d * 2 < 40 * 5001 * 2 * hkv * d * 2
    # the same sums, cut into other parts: half a step of the result and of the probabilities on either side
    top = 6 * 448 * float(scales[1])
    assert ((out.double() - expect.double()).abs() <= 2 ** -7 * (out.double().abs() + 1.01 * top)).all()
    ref, top, kq = oracle(q.cpu(), layer, meta, d ** -0.5, scales)
    for o in (out, expect):
        assert ((o.cpu().double() - ref).abs() <= bound(ref, top, kq, torch.bfloat16)).all()


def test_a_strided_page_table_names_the_same_pages():
    """Columns of a wider table on the device, as a program that keeps one table for all its seats hands them over."""
    for q_lens, past in (([1, 1], [100, 300]), ([40, 9], [130, 70])):
        meta, layer, scales, g = make_step(q_lens, past, 16, 2, 64, seed=5)
        m, lg, sg = meta.to("cuda"), layer.cuda(), scales.cuda()
        t = sum(q_lens)
        wide = torch.randint(0, layer.shape[0], (2, m.page_table.shape[1] + 7), generator=g).int().cuda()
        wide[:, 3:-4] = m.page_table
        strided = replace(m, page_table=wide[:, 3:-4])
        qkv, cs = torch.randn(t, 8 * 64, generator=g).bfloat16().cuda(), torch.randn(512, 64, generator=g).cuda()
        a, b = lg.clone(), lg.clone()
        qa, qb = (ops.rope_kv_write_fp4(qkv, x, step, cs, 4, 2, 64, sg) for x, step in ((a, m), (b, strided)))
        assert torch.equal(a, b) and torch.equal(qa, qb)
        assert torch.equal(ops.paged_attention_fp4(qa, a, m, 0.125, sg), ops.paged_attention_fp4(qa, a, strided, 0.125, sg))
        assert torch.equal(ops.kv_fp4_stage(a, m, sg, torch.bfloat16, 0, True)[0], ops.kv_fp4_stage(a, strided, sg, torch.bfloat16, 0, True)[0])


def test_steps_of_other_types_and_sizes_are_refused():
    meta, layer, scales, g = make_step([40, 9], [130, 70], 16, 2, 64, seed=5)
    m, lg, sg = meta.to("cuda"), layer.cuda(), scales.cuda()
    q, qkv, cs = torch.randn(49, 4, 64).half().cuda(), torch.randn(49, 8 * 64).half().cuda(), torch.ones(512, 64).cuda()
    one, pair = m.q_len[:1], torch.stack([m.past_len, m.past_len], 1)[:, 0]
    for bad in (dict(page_table=m.page_table.long()), dict(page_table=m.page_table[:1]), dict(past_len=m.past_len.long()), dict(past_len=m.past_len[:1]), dict(past_len=pair)):
        step = replace(m, **bad)
        for call in (lambda: ops.paged_attention_fp4(q, lg, step, 0.1, sg), lambda: ops.cuda_ops().paged_attention_fp4(q, lg, step, 0.1, sg, direct=True),
                     lambda: ops.rope_kv_write_fp4(qkv, lg, step, cs, 4, 2, 64, sg), lambda: ops.kv_fp4_stage(lg, step, sg, torch.float16)):
            with pytest.raises(ValueError):
                call()
    for bad in (dict(q_len=one), dict(q_len=m.q_len.long())):
        with pytest.raises(ValueError):
            ops.paged_attention_fp4(q, lg, replace(m, **bad), 0.1, sg)
    for bad in (dict(positions=m.positions[:5]), dict(seq_ids=m.seq_ids.long()), dict(positions=m.positions.float()), dict(kv_offsets=m.positions[:5])):
        with pytest.raises(ValueError):
            ops.rope_kv_write_fp4(qkv, lg, replace(m, **bad), cs, 4, 2, 64, sg)


# rows, cached rows, query heads, KV heads, head size, whether the prompt kernel takes the factors
PROMPTS = [(700, 0, 8, 2, 128, True), (300, 900, 8, 2, 128, True), (200, 300, 4, 2, 256, True), (60, 100, 8, 2, 64, False), (70, 0, 8, 2, 128, True), (100, 200, 8, 2, 128, False)]


@pytest.mark.parametrize("rows,past,hq,hkv,d,factors", PROMPTS)
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_prompt_steps_of_a_model_are_as_exact_as_the_operator(rows, past, hq, hkv, d, factors, dtype):
    """Scales that are no powers of two, and peaked scores: half a step of the result and of the probabilities (2^-8 or 2^-11, a third of its square on average: 0.8 of it
    for both), while keys rounded to 16 bits would move scores of |q| |k| some 16 by as many half steps."""
    from tensorrt_edge_llm_b200.config import tiny_llama_config
    from tensorrt_edge_llm_b200.models.default import Attention
    cfg = tiny_llama_config(num_hidden_layers=1, vocab_size=64, dtype=dtype, head_dim=d, num_attention_heads=hq, num_key_value_heads=hkv, hidden_size=128)
    layer = Attention(cfg, 0, "a").cuda()
    meta, pool, scales, g = make_step([rows], [past], 64, hkv, d, seed=rows)
    layer.kv_scales.copy_(scales)
    t = layer.kv_scales.dtype
    qkv = torch.randn(rows, (hq + 2 * hkv) * d, generator=g)
    qkv[:, :hq * d] *= 6.0
    qkv = qkv.to(getattr(torch, dtype)).cuda()
    cs = torch.cat([torch.ones(rows + past, d // 2), torch.zeros(rows + past, d // 2)], 1).cuda()
    m, lg = meta.to("cuda"), pool.cuda()
    assert t == torch.float32 and ops.fp4_exact(m, (hq, d), hkv) == factors and not ops.fp4_direct(m, hq // hkv)
    got = layer._forward_fp4(qkv, m, lg, cs).reshape(rows, hq, d)
    q = ops.rope_kv_write_fp4(qkv, lg, m, cs, hq, hkv, d, layer.kv_scales)
    want, top, kq = oracle(q.cpu(), lg.cpu(), meta, d ** -0.5, scales)
    err = float((got.cpu().double() - want).norm() / want.norm())
    half = torch.finfo(got.dtype).eps / 2
    if factors:
        assert torch.equal(got, ops.paged_attention_fp4(q, lg, m, d ** -0.5, layer.kv_scales))
        assert ((got.cpu().double() - want).abs() <= bound(want, top, kq, got.dtype)).all() and err < half
    else:
        assert err < 16 * half


@pytest.mark.parametrize("width", [64, 128, 256])
def test_commit_path_still_moves_rows_of_bytes(width):
    g = torch.Generator().manual_seed(2)
    pool = torch.randint(0, 256, (2, 6, 2, 3, 16, width), generator=g, dtype=torch.uint8)
    table, past = torch.tensor([[4, 1, 0], [2, 5, -1]], dtype=torch.int32), torch.tensor([14, 3])
    path, plen = torch.tensor([[0, 2, 5, 6], [0, 1, 4, 0]]), torch.tensor([4, 3])
    got = pool.cuda()
    if width == 64:                 # 32 elements of 16 bits: never had a kernel
        with pytest.raises(RuntimeError, match="head_dim"):
            ops.kv_commit_path(got, table.cuda(), past.int().cuda(), path.int().cuda(), plen.int().cuda())
        return
    ops.kv_commit_path(got, table.cuda(), past.int().cuda(), path.int().cuda(), plen.int().cuda())
    ops.kv_commit_path(pool, table, past, path, plen)
    assert torch.equal(got.cpu(), pool)


@pytest.mark.parametrize("d", [64, 128])
def test_a_captured_step_is_run_again_with_other_lengths(d):
    """The graph was captured with the lengths of one step; its tensors hold those of another by the time it runs."""
    hq, hkv, page = 8, 2, 64
    first, layer, scales, g = make_step([70, 40, 60], [0, 10, 5], page, hkv, d, seed=1)
    second, layer2, _, _ = make_step([70, 40, 60], [300, 0, 700], page, hkv, d, seed=2)
    m, lg, sg = first.to("cuda"), layer2.cuda(), scales.cuda()
    m.max_seq_len = 900
    m.page_table = torch.full(second.page_table.shape, -1, dtype=torch.int32, device="cuda")
    m.page_table[:, :first.page_table.shape[1]] = first.page_table.cuda()
    q = (torch.randn(170, hq, d, generator=g) * 2).bfloat16().cuda()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.paged_attention_fp4(q, lg, m, d ** -0.5, sg)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.paged_attention_fp4(q, lg, m, d ** -0.5, sg)
    m.past_len.copy_(second.past_len)
    m.page_table.copy_(second.page_table)
    for _ in range(2):
        graph.replay()
    want, top, kq = oracle(q.cpu(), layer2, second, d ** -0.5, scales)
    assert ((out.cpu().double() - want).abs() <= bound(want, top, kq, torch.bfloat16)).all()
