"""Steps that are too long to read four-bit pages in place, on the host: tables with holes, trees and windows against a 64-bit oracle."""
import pytest
import torch

from fp4_expanded_cases import holey_step, oracle
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
