"""Steps that are too long to read four-bit pages in place, on the host: tables with holes, trees and windows against a 64-bit oracle."""
from dataclasses import replace

import pytest
import torch

from fp4_expanded_cases import holey_step, oracle, poison_before_the_window
from fp4_kv_cases import make_step
from tensorrt_edge_llm_b200 import ops

# q_lens, past, page, missing logical pages of each sequence, window, tree
STEPS = [([40], [100], 64, [[0]], 0, False), ([40, 3], [100, 30], 16, [[1, 4], [0]], 0, False), ([7], [90], 32, [[1]], 0, True), ([5, 40], [60, 0], 16, [[0, 2], [1]], 0, True),
         ([20], [200], 32, [[3, 5]], 90, False), ([9], [64], 64, [[0, 1]], 0, False)]


@pytest.mark.parametrize("q_lens,past,page,missing,window,tree", STEPS)
@pytest.mark.parametrize("sunk", [False, True])
def test_holes_are_hidden_from_every_step(q_lens, past, page, missing, window, tree, sunk):
    hq, hkv, d = 6, 2, 64
    meta, layer, scales, g = holey_step(q_lens, past, page, hkv, d, missing, seed=sum(past), window=window, tree=tree)
    q = torch.randn(sum(q_lens), hq, d, generator=g) * 2
    sinks = torch.randn(hq, generator=g) if sunk else None
    want, top, kq = oracle(q, layer, meta, d ** -0.5, scales, window, sinks)
    got = ops.paged_attention_fp4(q, layer, meta, d ** -0.5, scales, sliding_window=window or None, sinks=sinks)
    # 32-bit: sums of 64 products (64 * 2^-24 of |q| |k|) make a probability off by that, sums of some 300 of them by 300 * 2^-24
    assert ((got.double() - want).abs() <= top * 2 ** -24 * (2 * 64 * kq + 600)).all()


def test_rows_that_a_window_hides_do_not_reach_the_outputs():
    for q_lens, past, window in (([1, 3], [90, 200], 37), ([40], [150], 65)):
        meta, layer, scales, g = make_step(q_lens, past, 16, 2, 64, seed=window)
        poison_before_the_window(meta, layer, window)
        q = torch.randn(sum(q_lens), 6, 64, generator=g)
        want, top, kq = oracle(q, layer, meta, 0.125, scales, window)
        got = ops.paged_attention_fp4(q, layer, meta, 0.125, scales, sliding_window=window)
        assert ((got.double() - want).abs() <= top * 2 ** -24 * (2 * 64 * kq + 600)).all()
        for new in (False, True):
            assert ops.kv_fp4_stage(layer, meta, scales, torch.bfloat16, window, new)[0].isfinite().all()


def test_copies_are_as_long_as_the_rows():
    q_lens, past = [1, 40, 0, 3, 128], [0, 300, 0, 126, 0]
    meta, layer, scales, _ = make_step(q_lens, past, 32, 1, 64)
    stage, staged = ops.kv_fp4_stage(layer, meta, scales, torch.float32, new_rows=True)
    assert stage.shape[0] == 2 * (1 + 3 + 1 + 2 + 1) + 1 and staged.page_table.shape == (5, 6)
    own = [int((row < stage.shape[0] - 1).sum()) for row in staged.page_table]
    assert own == [2, 6, 2, 4, 2] and sorted(staged.page_table[staged.page_table < 16].tolist()) == list(range(16)) and not stage[-1].any()
    whole, loose = ops.kv_fp4_stage(layer, replace(meta, host_lens=None, max_seq_len=500), scales, torch.float32, new_rows=True)
    assert whole.shape[0] == 5 * 8 and torch.equal(loose.page_table.flatten(), torch.arange(40, dtype=torch.int32))
    for s, (a, b) in enumerate(zip(q_lens, past)):
        for i in range((a + b + 63) // 64):
            assert torch.equal(stage[staged.page_table[s, i]], whole[loose.page_table[s, i]])
    same = make_step([4, 4], [60, 60], 32, 1, 64)
    assert ops.kv_fp4_stage(same[1], same[0], scales, torch.float32)[0].shape[0] == 4             # nobody shorter: no page of zeros


def test_clusters_follow_the_multiprocessors_of_the_device():
    ranks = ops.cuda_ops()._fp4_ranks
    assert ranks(8, 200) == 16 and ranks(9, 200) == 16 and ranks(10, 200) == 8
    assert ranks(8, 200, sms=120) == 8 and ranks(12, 200, sms=192) == 16        # 16 CTAs an item where each has a multiprocessor
    assert ranks(4, 4000) == 0 and ranks(9, 4000, sms=100) == 8                 # the line's merge pays for few items only


def test_commit_path_still_moves_rows_of_bytes():
    """Pages of one byte a feature, held as plain bytes, move as they did before there were four-bit pages."""
    g = torch.Generator().manual_seed(2)
    pool = torch.randint(0, 256, (2, 6, 2, 3, 16, 64), generator=g, dtype=torch.uint8)
    table, past = torch.tensor([[4, 1, 0], [2, 5, -1]], dtype=torch.int32), torch.tensor([14, 3])
    path, plen = torch.tensor([[0, 2, 5, 6], [0, 1, 4, 0]]), torch.tensor([4, 3])
    want = pool.view(torch.int8).clone()
    ops.kv_commit_path(want, table, past, path, plen)
    ops.kv_commit_path(pool, table, past, path, plen)
    assert torch.equal(pool, want.view(torch.uint8)) and not ops.ref.is_fp4_pages(pool)
