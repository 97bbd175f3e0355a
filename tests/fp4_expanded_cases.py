"""Steps over four-bit pages that are expanded for the prompt kernels, and their 64-bit oracle: tables with holes, tree masks, windows.  Shared by the CPU
and GPU tests."""
import torch

from fp4_kv_cases import make_step, page_values


def mask_bits(ql, parents):
    """Ancestor words ``[ql, ceil(ql / 32)]`` of a tree whose row r hangs below ``parents[r]`` (-1: the root)."""
    rows = []
    for r in range(ql):
        seen, a = 0, r
        while a >= 0:
            seen |= 1 << a
            a = parents[a]
        rows.append([(seen >> (32 * w)) & 0xffffffff for w in range((ql + 31) // 32)])
    return torch.tensor([[w - (1 << 32) if w >= 1 << 31 else w for w in row] for row in rows], dtype=torch.int32)


def holey_step(q_lens, past, page, hkv, d, missing, seed=0, window=0, tree=False):
    """A step whose sequence s lacks the logical pages ``missing[s]``."""
    meta, layer, scales, g = make_step(q_lens, past, page, hkv, d, seed=seed, window=window)
    for s, pages in enumerate(missing):
        for lp in pages:
            meta.page_table[s, lp] = -1 if lp % 2 else layer.shape[0] + 3
    if tree:
        words = (max(q_lens) + 31) // 32
        rows = [torch.nn.functional.pad(mask_bits(q, [(r - 1) // 2 for r in range(q)]), (0, words - (q + 31) // 32)) for q in q_lens]
        meta.tree_mask = torch.cat(rows)
    return meta, layer, scales, g


def seen_keys(meta, s, page, pages, window=0):
    """``[q_len, past + q_len]``: which keys the rows of sequence s see."""
    r0, ql, past = int(meta.q_start[s]), int(meta.q_len[s]), int(meta.past_len[s])
    col, row = torch.arange(past + ql), torch.arange(ql)[:, None]
    seen = col <= past + row
    if meta.tree_mask is not None:
        words = meta.tree_mask[r0:r0 + ql].long()
        new = (col - past).clamp(min=0)
        seen = (col < past) | (((words[:, new // 32] >> (new % 32)) & 1) == 1)
    if window:
        seen = seen & (col > past + row - window)
    pg = meta.page_table[s].long()[col // page]
    return seen & (pg >= 0) & (pg < pages)


def oracle(q, layer, meta, scale, scales, window=0, sinks=None):
    """64-bit attention; values that no row of the step sees do not take part.  Returns ``(out, largest visible value, largest |q| |k| scale)``."""
    vals = page_values(layer, scales)
    hkv, p = layer.shape[2:4]
    hq, d = q.shape[1:]
    g = hq // hkv
    out = torch.zeros(q.shape, dtype=torch.float64)
    top = kq = 0.0
    for s in range(meta.num_seqs):
        r0, ql, past = int(meta.q_start[s]), int(meta.q_len[s]), int(meta.past_len[s])
        if ql == 0:
            continue
        seen = seen_keys(meta, s, p, layer.shape[0], window)
        col = torch.arange(past + ql)
        live = seen.any(0)
        pg = torch.where(live, meta.page_table[s].long()[col // p], 0)
        kv = vals[pg, :, :, col % p].masked_fill(~live[:, None, None, None], 0.0)          # [keys, 2, Hkv, D]
        qs = q[r0:r0 + ql].double().view(ql, hkv, g, d)
        z = torch.einsum("rhgd,khd->hgrk", qs, kv[:, 0]) * scale
        z = z.masked_fill(~seen, float("-inf"))
        if sinks is not None:
            z = torch.cat([z, sinks.double().view(hkv, g, 1, 1).expand(hkv, g, ql, 1)], -1)
        pr = torch.softmax(z, -1)[..., :past + ql].nan_to_num(0.0)
        out[r0:r0 + ql] = torch.einsum("hgrk,khd->rhgd", pr, kv[:, 1]).reshape(ql, hq, d)
        top = max(top, float(kv[:, 1].abs().max()))
        kq = max(kq, float(qs.norm(dim=-1).max() * kv[:, 0].norm(dim=-1).max()) * scale)
    return out, top, kq


def poison_before_the_window(meta, layer, window):
    """NaN block scales in all cached rows that no row of the step sees."""
    from tensorrt_edge_llm_b200.ops import reference as ref
    _, sf = ref.fp4_page_parts(layer)
    p = layer.shape[3]
    for s in range(meta.num_seqs):
        slot = torch.arange(max(0, int(meta.past_len[s]) + 1 - window))
        pg = meta.page_table[s].long()[slot // p]
        there = pg >= 0
        sf[pg[there], :, :, (slot % p)[there]] = 0x7f
    return layer
