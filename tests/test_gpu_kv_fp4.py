"""Four-bit cache pages on the GPU: the write and the 16-bit copies bit by bit against the host formulation, attention and accumulated weights against
64-bit sums, eviction against sorting, and the calls that a program makes around them (other streams, captured graphs, refusals)."""
import math

import pytest
import torch

from fp4_kv_cases import make_step, oracle_attention, oracle_evict, page_values
from tensorrt_edge_llm_b200 import ops
from tensorrt_edge_llm_b200.ops import build_step_meta
from tensorrt_edge_llm_b200.ops import reference as ref

pytestmark = pytest.mark.gpu

WRITES = [([1], [0], 4, 1, 64, 16), ([1] * 5, [0, 15, 16, 63, 200], 32, 8, 128, 64), ([3, 1, 40], [0, 37, 13], 6, 2, 128, 32), ([2, 0, 7], [5, 9, 0], 8, 2, 256, 64),
          ([130], [0], 14, 2, 64, 128)]


@pytest.mark.parametrize("q_lens,past,hq,hkv,d,page", WRITES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("norm,rot", [(True, 1.0), (False, 1.0), (True, 0.5), (False, 0.25)])
def test_write_is_the_host_formulation_bit_by_bit(q_lens, past, hq, hkv, d, page, dtype, norm, rot):
    meta, layer, scales, g = make_step(q_lens, past, page, hkv, d, seed=hq)
    t = sum(q_lens)
    qkv = (torch.randn(t, (hq + 2 * hkv) * d, generator=g) * 3).to(dtype)
    qkv[0, hq * d] = math.inf if not norm else 0.0               # an infinite key feature fills its block with the largest number
    qkv[0, (hq + hkv) * d:(hq + hkv) * d + 16] = 0.0             # a block of zeros
    cs = ref.rope_cos_sin(max(a + b for a, b in zip(q_lens, past)), int(d * rot), 1e4)
    qw, kw = ((1 + 0.1 * torch.randn(d, generator=g)).to(dtype) for _ in range(2)) if norm else (None, None)
    stage = torch.randn(layer.shape[0], 2, hkv, page, d, generator=g).to(dtype)
    gpu = [x.cuda() if x is not None else None for x in (qkv, layer, cs, scales, qw, kw, stage)]
    stage_w, layer_w = stage.clone(), layer.clone()
    q_w = ref.rope_kv_write_fp4(qkv, layer_w, meta, cs, hq, hkv, d, scales, qw, kw, stage=stage_w, stage_table=meta.page_table)
    m = meta.to("cuda")
    q = ops.rope_kv_write_fp4(gpu[0], gpu[1], m, gpu[2], hq, hkv, d, gpu[3], gpu[4], gpu[5], stage=gpu[6], stage_table=m.page_table)
    alone = layer.cuda()
    q2 = ops.rope_kv_write_fp4(gpu[0], alone, m, gpu[2], hq, hkv, d, gpu[3], gpu[4], gpu[5])
    torch.cuda.synchronize()
    assert torch.equal(q.cpu().nan_to_num(7), q_w.nan_to_num(7)) and torch.equal(q2, q)
    assert torch.equal(gpu[1].cpu(), layer_w) and torch.equal(alone, gpu[1])
    assert torch.equal(gpu[6].cpu().nan_to_num(7), stage_w.nan_to_num(7))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rot", [1.0, 0.5])
def test_rows_as_small_as_eps_are_normalised_bit_by_bit(dtype, rot):
    """Mean squares near eps, whose own last bits count then; and far below and above it."""
    hq, hkv, d, t = 6, 3, 128, 400
    meta, layer, scales, g = make_step([t], [0], 64, hkv, d, seed=4)
    qkv = (torch.randn(t, (hq + 2 * hkv) * d, generator=g) * torch.tensor([1e-3, 2e-3, 1e-5, 30.0]).repeat(t // 4)[:, None]).to(dtype)
    cs = ref.rope_cos_sin(t, int(d * rot), 1e4)
    w = (1 + 0.1 * torch.randn(2, d, generator=g)).to(dtype)
    host = layer.clone()
    want = ref.rope_kv_write_fp4(qkv, host, meta, cs, hq, hkv, d, scales, w[0], w[1], 1e-6)
    gpu = layer.cuda()
    got = ops.rope_kv_write_fp4(qkv.cuda(), gpu, meta.to("cuda"), cs.cuda(), hq, hkv, d, scales.cuda(), w[0].cuda(), w[1].cuda(), 1e-6)
    assert torch.equal(got.cpu(), want) and torch.equal(gpu.cpu(), host)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,page", [(64, 16), (128, 64), (256, 32)])
def test_stage_is_the_host_formulation(dtype, d, page):
    meta, layer, scales, _ = make_step([2, 1, 5], [70, 0, 128], page, 2, d)
    for new in (False, True):
        want, meta_w = ref.kv_fp4_stage(layer, meta, scales, dtype, 0, new)
        got, meta_g = ops.kv_fp4_stage(layer.cuda(), meta.to("cuda"), scales.cuda(), dtype, 0, new)
        got = got.cpu()
        if not new:                                   # the step's own rows are left for the write
            for q, past, row in ((2, 70, 0), (1, 0, 1), (5, 128, 2)):
                for slot in range(past, past + q):
                    got[meta_w.page_table[row, slot // 64], :, :, slot % 64] = 0.0
        assert torch.equal(meta_g.page_table.cpu(), meta_w.page_table) and torch.equal(got, want)


# q_lens, past, query heads, KV heads, head size, page, window
STEPS = [([1], [0], 4, 1, 128, 64, 0), ([1, 1, 1], [5, 64, 700], 32, 8, 128, 64, 0), ([1] * 6, [0, 1, 15, 31, 32, 33], 8, 8, 128, 64, 0),
         ([4, 0, 1], [40, 9, 300], 14, 2, 128, 16, 0), ([5, 3], [200, 90], 16, 1, 64, 128, 0), ([2, 1], [129, 500], 8, 2, 256, 64, 0),
         ([1, 3], [700, 400], 10, 2, 64, 64, 130), ([3], [900], 16, 2, 128, 64, 257), ([2], [350], 4, 2, 256, 32, 40), ([20, 6], [100, 0], 6, 2, 128, 64, 0)]


def bound(want, vals, dtype):
    """Half a step of the result's type; 2^-11 of the largest value for the fp16 probabilities (half a step, numerator and sum); 2^-15 of it for 32-bit
    scores of up to 20 whose sums are off by some 2^-20, and for exp2."""
    return torch.finfo(dtype).eps / 2 * want.abs() * 1.01 + (2 ** -11 + 2 ** -15) * vals + 1e-7


@pytest.mark.parametrize("q_lens,past,hq,hkv,d,page,window", STEPS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sunk", [False, True])
def test_attention_in_place(q_lens, past, hq, hkv, d, page, window, dtype, sunk):
    meta, layer, scales, g = make_step(q_lens, past, page, hkv, d, seed=sum(past) + hq, window=window)
    q = (torch.randn(sum(q_lens), hq, d, generator=g) * 2).to(dtype)
    sinks = torch.randn(hq, generator=g) * 2 if sunk else None
    w = torch.rand(layer.shape[0], hkv, page, generator=g)
    want, want_w = oracle_attention(q, layer, meta, d ** -0.5, scales, window, sinks, w, 0.75)
    top = 6 * 448 * float(scales[1])
    m, lg, qg, sg = meta.to("cuda"), layer.cuda(), q.cuda(), scales.cuda()
    zg = sinks.cuda() if sunk else None
    for ctas in (None, 1, 3, -1, -2, -8):
        wg = w.cuda()
        got = ops.cuda_ops().paged_attention_fp4(qg, lg, m, d ** -0.5, sg, window or None, zg, wg, 0.75, ctas=ctas)
        again = ops.cuda_ops().paged_attention_fp4(qg, lg, m, d ** -0.5, sg, window or None, zg, direct=True, ctas=ctas)
        assert torch.equal(got, again)
        assert ((got.cpu().double() - want).abs() <= bound(want, top, dtype)).all(), ctas
        # a probability is off by the 32-bit error of its score and of the sum: 2^-15 of it, up to group * rows of them a key
        assert ((wg.cpu().double() - want_w).abs() <= 2 ** -15 * want_w + 1e-6).all(), ctas
    if not sunk:
        assert torch.equal(ops.paged_attention_fp4(qg, lg, m, d ** -0.5, sg, sliding_window=window or None, weights=w.cuda(), decay=0.75),
                           ops.paged_attention_fp4(qg, lg, m, d ** -0.5, sg, sliding_window=window or None, weights=torch.zeros_like(w).cuda()))


@pytest.mark.parametrize("q_lens,past,hq,hkv,d,page,window", [([70, 1], [30, 200], 8, 2, 128, 64, 0), ([40], [0], 16, 4, 64, 128, 0), ([33, 90], [260, 5], 8, 2, 128, 32, 100),
                                                              ([20], [50], 8, 1, 256, 16, 0)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_prompt_steps_go_through_16_bit_copies(q_lens, past, hq, hkv, d, page, window, dtype):
    meta, layer, scales, g = make_step(q_lens, past, page, hkv, d, seed=sum(past), window=window)
    q = (torch.randn(sum(q_lens), hq, d, generator=g) * 2).to(dtype)
    want, _ = oracle_attention(q, layer, meta, d ** -0.5, scales, window)
    got = ops.cuda_ops().paged_attention_fp4(q.cuda(), layer.cuda(), meta.to("cuda"), d ** -0.5, scales.cuda(), window or None, direct=False)
    # 16-bit keys and values (half a step each; a score is a sum of at most |q| |k| of them) and 16-bit probabilities
    half = torch.finfo(dtype).eps / 2
    top = 6 * 448 * float(scales[1])
    kq = float((q.double().norm(dim=-1).max()) * page_values(layer, scales).nan_to_num().norm(dim=-1).max()) * d ** -0.5
    assert ((got.cpu().double() - want).abs() <= half * want.abs() + (2 * half * min(kq, 40) + 3 * half) * top).all()
    err = (got.cpu().double() - want).norm() / want.norm()
    assert err < 8 * half


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_large_and_tiny_queries_and_peaked_scores(dtype):
    """One key takes everything, far above the others and last, first or in the middle; queries of 2^-10 and 2^6."""
    hq, hkv, d, past = 8, 2, 128, 1000
    meta, layer, scales, g = make_step([1, 1, 1], [past, past, past], 64, hkv, d, seed=3)
    q = torch.randn(3, hq, d, generator=g)
    vals = page_values(layer, scales)
    for s, key in enumerate((0, 500, past)):
        k = vals[meta.page_table[s, key // 64], 0, :, key % 64].float()           # the query points at this key
        q[s] = k.repeat_interleave(hq // hkv, 0) * (64.0 if s == 1 else 4.0)
    q[2, :4] *= 2.0 ** -10
    q = q.to(dtype)
    want, want_w = oracle_attention(q, layer, meta, d ** -0.5, scales, weights=torch.zeros(layer.shape[0], hkv, 64))
    w = torch.zeros(layer.shape[0], hkv, 64, device="cuda")
    got = ops.paged_attention_fp4(q.cuda(), layer.cuda(), meta.to("cuda"), d ** -0.5, scales.cuda(), weights=w)
    top = 6 * 448 * float(scales[1])
    # scores of up to 3000: off by 2^-21 of that, so probabilities by 2^-9 where they are not one
    assert ((got.cpu().double() - want).abs() <= bound(want, top, dtype) + 2 ** -9 * top * (want_w.max() < 0.999)).all()
    assert (w.cpu().double() - want_w).abs().max() < 2 ** -9


def test_rows_that_see_nothing_and_missing_pages():
    meta, layer, scales, g = make_step([1, 1], [100, 40], 64, 2, 128)
    meta.page_table[0, 0] = -1                      # a hole: its keys are not there
    meta.page_table[1, :] = layer.shape[0] + 5      # no page of this pool
    q = torch.randn(2, 8, 128, generator=g).bfloat16()
    want, _ = oracle_attention(q[:1], layer, build_step_meta([1], [100], meta.page_table[:1], 64), 0.1, scales)
    for sinks in (None, torch.zeros(8)):
        got = ops.paged_attention_fp4(q.cuda(), layer.cuda(), meta.to("cuda"), 0.1, scales.cuda(), sinks=None if sinks is None else sinks.cuda(),
                                      weights=torch.zeros(layer.shape[0], 2, 64, device="cuda"))
        assert (got[1] == 0).all()
        if sinks is None:
            assert ((got[0].cpu().double() - want[0]).abs() <= bound(want[0], 6 * 448 * float(scales[1]), torch.bfloat16)).all()
    out = ops.rope_kv_write_fp4(torch.randn(2, 12 * 128, device="cuda").bfloat16(), layer.cuda(), meta.to("cuda"), torch.ones(200, 128, device="cuda"), 8, 2, 128, scales.cuda())
    assert out.isfinite().all()


EVICTS = [([700, 64, 0, 130, 1], 64, 2, 96, 4, 32, 128), ([300], 16, 1, 17, 0, 0, 64), ([5000, 4000], 64, 4, 1000, 4, 32, 128), ([90], 32, 2, 40, 8, 32, 64), ([2100, 33], 32, 1, 2000, 1, 1, 256)]


@pytest.mark.parametrize("lengths,page,hkv,keep,first,recent,d", EVICTS)
@pytest.mark.parametrize("kind", ["fp4", "fp8", "bf16"])
@pytest.mark.parametrize("ties", [False, True])
def test_evict(lengths, page, hkv, keep, first, recent, d, kind, ties):
    g = torch.Generator().manual_seed(keep)
    n, wide, room = len(lengths), max((x + page - 1) // page for x in lengths) + 1, (keep + page - 1) // page
    pages = n * (wide + room)
    table = torch.randperm(n * wide, generator=g).int().view(n, wide)
    to = (n * wide + torch.randperm(n * room, generator=g)).int().view(n, room)
    w = torch.rand(pages, hkv, page, generator=g)
    w = (w * 4).floor() - 1 if ties else (w * 30 - 30).exp()
    w[table[0, 1], 0, 3] = math.nan
    w[table[0, 0], 0, min(6, page - 1)] = math.inf
    layer = torch.randint(0, 256, (pages, 2, hkv, page, {"fp4": d * 9 // 16, "fp8": d, "bf16": 2 * d}[kind]), generator=g, dtype=torch.uint8)
    layer = layer.view({"fp4": torch.uint8, "fp8": torch.float8_e4m3fn, "bf16": torch.bfloat16}[kind])
    lens = torch.tensor(lengths, dtype=torch.int32)
    lg, wg = layer.cuda(), w.cuda()
    got = ops.kv_evict(lg, wg, table.cuda(), lens.cuda(), to.cuda(), keep, first, recent)
    kept = ops.kv_evict(layer, w, table, lens, to, keep, first, recent)
    assert torch.equal(got.cpu(), kept)
    assert torch.equal(lg.cpu().view(torch.uint8), layer.view(torch.uint8)) and torch.equal(wg.cpu().view(torch.int32), w.view(torch.int32))
    want = oracle_evict(w, table, lengths, page, keep, first, recent)      # rows of the old pages, which nothing changed
    for s in range(n):
        for h in range(hkv):
            assert kept[s, h].tolist() == want[s][h] + [-1] * (keep - len(want[s][h]))


def test_evict_takes_rows_without_a_page_last():
    g = torch.Generator().manual_seed(8)
    table = torch.randperm(300, generator=g).int().view(2, 150)
    table[:, 3:40:3] = -1
    table[1, 90:] = -1
    to = torch.arange(300, 600, dtype=torch.int32).view(2, 150)
    w = (torch.rand(600, 2, 16, generator=g) - 0.5) * torch.tensor([1.0, math.inf])[torch.randint(0, 2, (600, 2, 16), generator=g)]
    w[0] = w[299] = math.nan
    layer, lens = torch.randint(0, 256, (600, 2, 2, 16, 36), generator=g, dtype=torch.uint8), torch.tensor([2400, 2000], dtype=torch.int32)
    for keep in (100, 1300, 2200):
        lg, wg, lh, wh = layer.cuda(), w.cuda(), layer.clone(), w.clone()
        got = ops.kv_evict(lg, wg, table.cuda(), lens.cuda(), to.cuda(), keep, 4, 32)
        assert torch.equal(got.cpu(), ops.kv_evict(lh, wh, table, lens, to, keep, 4, 32))
        assert torch.equal(lg.cpu(), lh) and torch.equal(wg.cpu().nan_to_num(7), wh.nan_to_num(7))


def test_write_attend_evict_attend_in_a_captured_graph_and_on_another_stream():
    """A conversation: the prompt is written and attended to, steps keep account of the weights, rows are dropped, steps go on over what is left."""
    hq, hkv, d, page, past, keep = 8, 2, 128, 64, 300, 128
    g = torch.Generator().manual_seed(9)
    pages = 16
    scales = torch.tensor([0.0021, 0.0034])
    cs = ref.rope_cos_sin(400, d, 1e4)
    rows = torch.randn(past + 4, (hq + 2 * hkv) * d, generator=g).bfloat16()
    table, to = torch.arange(6, dtype=torch.int32).view(1, 6), torch.arange(8, 14, dtype=torch.int32).view(1, 6)

    def talk(dev, call):
        layer, w = torch.zeros(pages, 2, hkv, page, 72, dtype=torch.uint8, device=dev), torch.zeros(pages, hkv, page, device=dev)
        sc, c, x = scales.to(dev), cs.to(dev), rows.to(dev)
        outs = []
        prompt = build_step_meta([past], [0], table, page, device=dev)
        steps = [build_step_meta([1], [past + i], table, page, device=dev) for i in range(2)]
        n = torch.tensor([past + 2], dtype=torch.int32, device=dev)
        after = [build_step_meta([1], [keep + i], to, page, device=dev, positions=[past + 2 + i]) for i in range(2)]
        t0, t1 = table.to(dev), to[:, :2].to(dev).contiguous()

        def everything():
            outs.clear()
            w.zero_()                     # a graph is run more than once: every run tells the same story from its beginning
            q = ops.rope_kv_write_fp4(x[:past], layer, prompt, c, hq, hkv, d, sc)
            outs.append(ops.paged_attention_fp4(q, layer, prompt, d ** -0.5, sc))
            for i, m in enumerate(steps):
                q = ops.rope_kv_write_fp4(x[past + i:past + i + 1], layer, m, c, hq, hkv, d, sc)
                outs.append(ops.paged_attention_fp4(q, layer, m, d ** -0.5, sc, weights=w))
            outs.append(ops.kv_evict(layer, w, t0, n, t1, keep, 4, 16))
            for i, m in enumerate(after):
                q = ops.rope_kv_write_fp4(x[past + 2 + i:past + 3 + i], layer, m, c, hq, hkv, d, sc)
                outs.append(ops.paged_attention_fp4(q, layer, m, d ** -0.5, sc, weights=w))
            outs.extend([layer, w])
        call(everything)
        return [o.clone() for o in outs]

    def graph(f):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            f()
        torch.cuda.current_stream().wait_stream(s)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            f()
        for _ in range(2):
            gr.replay()
        torch.cuda.synchronize()

    def other(f):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            f()
        torch.cuda.current_stream().wait_stream(s)

    eager = talk("cuda", lambda f: f())
    for call in (graph, other):
        for a, b in zip(eager, talk("cuda", call)):
            assert torch.equal(a, b)
    host = talk("cpu", lambda f: f())
    kept_g, kept_h = eager[3].cpu(), host[3]
    # the rows that stay may differ where two weights are equal but for their last bits
    assert (kept_g != kept_h).float().mean() < 0.02
    for a, b in zip(eager[:3], host[:3]):
        assert (a.float().cpu() - b.float()).norm() < 0.01 * b.float().norm()


def test_refusals_on_the_gpu():
    meta, layer, scales, g = make_step([1], [5], 16, 2, 64)
    m, lg, sg = meta.to("cuda"), layer.cuda(), scales.cuda()
    q, qkv, cs = torch.randn(1, 4, 64).cuda(), torch.randn(1, 8 * 64).cuda(), torch.ones(32, 64).cuda()
    w = torch.zeros(layer.shape[0], 2, 16).cuda()
    at = ops.paged_attention_fp4
    for call in (lambda: at(q, lg, m, 0.1, sg),                                                       # fp32 rows
                 lambda: ops.rope_kv_write_fp4(qkv, lg, m, cs, 4, 2, 64, sg),
                 lambda: ops.kv_fp4_stage(lg, m, sg, torch.float32)):
        with pytest.raises(TypeError):
            call()
    q, qkv = q.half(), qkv.half()
    many = build_step_meta([200], [0], torch.zeros(1, 13, dtype=torch.int32), 16).to("cuda")
    tree = build_step_meta([1], [5], meta.page_table, 16, tree_mask=torch.ones(1, 1, dtype=torch.int32)).to("cuda")
    for call in (lambda: at(q, lg[..., :35], m, 0.1, sg), lambda: at(q, lg.transpose(1, 2), m, 0.1, sg), lambda: at(q, lg, m, -1.0, sg), lambda: at(q, lg, m, math.nan, sg),
                 lambda: at(q[:, :3], lg, m, 0.1, sg), lambda: at(q, lg, m, 0.1, sg.double()), lambda: at(q, lg, m, 0.1, sg[:1]), lambda: at(q, lg, m, 0.1, sg, weights=w[:1]),
                 lambda: at(q, lg, m, 0.1, sg, weights=w.double()), lambda: at(q, lg, m, 0.1, sg, sinks=torch.zeros(3).cuda()), lambda: at(q, layer, m, 0.1, sg),
                 lambda: at(torch.randn(200, 4, 64).half().cuda(), lg, many, 0.1, sg, weights=w), lambda: at(q, lg, tree, 0.1, sg, weights=w),
                 lambda: ops.cuda_ops().paged_attention_fp4(q, lg, tree, 0.1, sg, direct=True), lambda: ops.cuda_ops().paged_attention_fp4(q, lg, m, 0.1, sg, weights=w, direct=False),
                 lambda: ops.rope_kv_write_fp4(qkv, lg, m, cs[:, :6], 4, 2, 64, sg), lambda: ops.rope_kv_write_fp4(qkv, lg, m, cs.double(), 4, 2, 64, sg),
                 lambda: ops.rope_kv_write_fp4(qkv, lg, m, cs, 2, 3, 64, sg), lambda: ops.rope_kv_write_fp4(qkv, lg, m, cs, 4, 2, 64, sg, torch.ones(64).cuda()),
                 lambda: ops.rope_kv_write_fp4(qkv, lg, m, cs, 4, 2, 64, sg, stage=torch.zeros(1, 2, 2, 16, 64).cuda(), stage_table=m.page_table),
                 lambda: ops.kv_evict(lg, w, m.page_table, m.past_len, m.page_table.cpu(), 4),
                 lambda: ops.kv_evict(lg.transpose(2, 3), w, m.page_table, m.past_len, m.page_table, 4)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("d", [64, 128, 256])
def test_commit_path_moves_codes_and_scales(d):
    g = torch.Generator().manual_seed(d)
    pool = torch.randint(0, 256, (3, 9, 2, 2, 32, d * 9 // 16), generator=g, dtype=torch.uint8)
    table = torch.tensor([[4, 1, 0], [2, 5, -1], [7, 8, 3]], dtype=torch.int32)
    past, path = torch.tensor([30, 3, 0]), torch.tensor([[0, 2, 5, 6], [0, 1, 4, 0], [0, 0, 0, 0]])
    plen = torch.tensor([4, 3, 1])
    got = pool.cuda()
    ops.kv_commit_path(got, table.cuda(), past.cuda(), path.int().cuda(), plen.int().cuda())
    ops.kv_commit_path(pool, table, past, path, plen)
    assert torch.equal(got.cpu(), pool)


@pytest.mark.parametrize("family", ["dense", "window"])
def test_model_with_four_bit_kv_eager_and_graph(family):
    """Chunked prompts, steps and captured steps on the GPU against the same model on the host, and tree steps against plain ones."""
    from tensorrt_edge_llm_b200 import AutoModel
    from tensorrt_edge_llm_b200.config import tiny_llama_config
    from tensorrt_edge_llm_b200.runtime.kv_cache import KVCacheManager
    from tensorrt_edge_llm_b200.runtime.runner import ModelRunner
    dev = torch.device("cuda", 0)
    cfg = tiny_llama_config(num_hidden_layers=3, vocab_size=512, dtype="bfloat16", head_dim=128, num_attention_heads=4, num_key_value_heads=2, hidden_size=512)
    if family == "window":
        cfg.sliding_window = 100
    model, host = AutoModel.from_config(cfg, device=dev, random_init=0), AutoModel.from_config(cfg, device="cpu", random_init=0)
    host.load_state_dict(model.state_dict())
    g = torch.Generator().manual_seed(5)
    prompts = torch.randint(0, cfg.vocab_size, (2, 300), generator=g).tolist()
    feed = torch.randint(0, cfg.vocab_size, (5, 2), generator=g).tolist()

    def run(m, device, kv_dtype, graphs=True):
        kv = KVCacheManager(cfg, num_pages=24, page_size=64, max_seats=2, max_pages_per_seq=10, device=device, kv_dtype=kv_dtype)
        r = ModelRunner(m, kv, max_num_tokens=256)
        r.use_cuda_graphs = graphs and device != "cpu"
        out = [r.prefill([0, 1], prompts).float()]
        for toks in feed:
            out.append(r.step([0, 1], [[t] for t in toks]).float())
        many = r.step([0, 1], [[3, 5, 7], [11, 13, 17]], logits_all=True).float()
        mask = torch.tensor([[1], [3], [7]] * 2, dtype=torch.int32, device=device)      # a chain as a tree: the same rows through the prompt kernels
        for s in (0, 1):
            kv.rewind(s, kv.lengths[s] - 3)
        tree = r.step([0, 1], [[3, 5, 7], [11, 13, 17]], logits_all=True, tree_mask=mask).float()
        toks = r.decode_greedy([0, 1], out[-1].argmax(-1).to(torch.int32), 12)
        return torch.stack(out).cpu(), many.cpu(), tree.cpu(), toks.cpu(), kv

    full = run(model, dev, "model")
    four, many, tree, toks, kv = run(model, dev, "nvfp4")
    assert kv.pool.dtype == torch.uint8
    want, many_h, _, _, _ = run(host, "cpu", "nvfp4")
    cos = lambda a, b: float(torch.nn.functional.cosine_similarity(a.flatten(1), b.flatten(1), dim=1).min())
    # bf16 layers: a code on a border may fall to either side of it, as in any two orders of the same sums
    assert cos(four, want) > 0.995 and cos(many, many_h) > 0.995 and cos(tree, many) > 0.995
    assert cos(full[0], four) > 0.95
    assert torch.equal(run(model, dev, "nvfp4", graphs=False)[3], toks)


@pytest.mark.parametrize("family", ["gemma", "hybrid"])
def test_other_stacks_over_four_bit_pages(family):
    """256-wide heads in sliding and full layers, and attention beside recurrent layers: near the 16-bit cache over prompts and steps."""
    from tensorrt_edge_llm_b200 import AutoModel
    from tensorrt_edge_llm_b200.config import GdnConfig, MambaConfig, ModelConfig, hybrid_nemotron_config
    from tensorrt_edge_llm_b200.runtime.kv_cache import KVCacheManager
    from tensorrt_edge_llm_b200.runtime.runner import ModelRunner
    if family == "gemma":
        cfg = ModelConfig.from_hf_dict(dict(model_type="gemma3_text", vocab_size=512, hidden_size=512, intermediate_size=1024, num_hidden_layers=3, num_attention_heads=4,
                                            num_key_value_heads=2, head_dim=256, sliding_window=96, query_pre_attn_scalar=256, max_position_embeddings=1024,
                                            layer_types=["sliding_attention", "full_attention", "sliding_attention"], dtype="bfloat16"))
    else:
        cfg = hybrid_nemotron_config(num_hidden_layers=8, vocab_size=512, hidden_size=256, intermediate_size=512, num_attention_heads=4, num_key_value_heads=2, head_dim=64,
                                     dtype="bfloat16", max_position_embeddings=512, mamba=MambaConfig(num_heads=8, head_dim=64, d_state=128, n_groups=2, conv_kernel=4),
                                     gdn=GdnConfig(num_k_heads=2, num_v_heads=4, head_k_dim=128, head_v_dim=128, conv_kernel=4))
    model = AutoModel.from_config(cfg, device=torch.device("cuda", 0), random_init=0)
    g = torch.Generator().manual_seed(3)
    prompts, feed = [torch.randint(0, 512, (n,), generator=g).tolist() for n in (200, 37)], torch.randint(0, 512, (4, 2), generator=g).tolist()

    def run(kv_dtype):
        kv = KVCacheManager(cfg, num_pages=16, page_size=64, max_seats=2, max_pages_per_seq=6, device="cuda", kv_dtype=kv_dtype)
        r = ModelRunner(model, kv)
        out = [r.prefill([0, 1], prompts)] + [r.step([0, 1], [[t] for t in row]) for row in feed]
        return torch.stack(out).float(), kv

    want, _ = run("model")
    got, kv = run("nvfp4")
    assert kv.kv_fp4
    # E2M1 with block scales is off by a tenth of a row's norm at most; a missing or misplaced row would leave no likeness
    assert float(torch.nn.functional.cosine_similarity(got.flatten(0, 1), want.flatten(0, 1), dim=1).min()) > 0.95
