"""Steps over four-bit pages and their 64-bit oracle, shared by the CPU and GPU tests of the four-bit cache."""
import math

import torch

from tensorrt_edge_llm_b200.ops import build_step_meta
from tensorrt_edge_llm_b200.ops import reference as ref

LEVELS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def e4m3(byte: torch.Tensor) -> torch.Tensor:
    """Values of E4M3 bytes from their fields (0x7f / 0xff: NaN)."""
    b = byte.long()
    e, m = (b >> 3) & 15, (b & 7).double()
    v = torch.where(e == 0, m * 2.0 ** -9, (1 + m / 8) * torch.exp2((e - 7).double()))
    v = torch.where((b & 127) == 127, torch.full_like(v, math.nan), v)
    return torch.where(b > 127, -v, v)


def page_values(layer: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """64-bit values ``[pages, 2, Hkv, P, D]`` of a four-bit layer, from its bytes."""
    n, _, h, p, width = layer.shape
    d = width * 16 // 9
    flat = layer.reshape(n, 2, h, -1)
    byte = flat[..., :p * d // 2].reshape(n, 2, h, p, d // 2).long()
    code = torch.stack([byte % 16, byte // 16], -1).reshape(n, 2, h, p, d)
    val = LEVELS[code % 8] * torch.where(code >= 8, -1.0, 1.0)
    sf = e4m3(flat[..., p * d // 2:].reshape(n, 2, h, p, d // 16))
    return val * sf.repeat_interleave(16, -1) * scales.double().view(1, 2, 1, 1, 1)


def random_layer(g, pages, hkv, p, d, scales):
    """Pages of normal features; the rows that no test writes hold arbitrary bytes, NaN block scales among them."""
    layer = torch.randint(0, 256, (pages, 2, hkv, p, d * 9 // 16), generator=g, dtype=torch.uint8)
    return layer


def fill_layer(layer, g, table, lengths, scales, spread=1.0):
    """Quantise normal rows into the slots ``[0, length)`` of every sequence."""
    p = layer.shape[3]
    d = ref.fp4_head_dim(layer)
    codes, sf = ref.fp4_page_parts(layer)
    for s, n in enumerate(lengths):
        slot = torch.arange(n)
        page = table[s].long()[slot // p]
        ok = page >= 0
        x = torch.randn(n, 2, layer.shape[2], d, generator=g) * spread
        c, f, _ = ref.fp4_encode_rows(x, scales.view(2, 1, 1))
        codes[page[ok], :, :, (slot % p)[ok]] = c[ok]
        sf[page[ok], :, :, (slot % p)[ok]] = f[ok]
    return layer


def make_step(q_lens, past, page=64, hkv=2, d=128, seed=0, window=0, spread=1.0, gaps=True):
    """``(meta, layer, scales, generator)``; with a window, the pages wholly before it are gone."""
    g = torch.Generator().manual_seed(seed)
    n = len(q_lens)
    total = [a + b for a, b in zip(q_lens, past)]
    wide = max((x + page - 1) // page for x in total) + (1 if gaps else 0)
    pages = n * wide + 2
    perm = torch.randperm(pages, generator=g).int()
    table, k = torch.full((n, wide), -1, dtype=torch.int32), 0
    for s in range(n):
        need = (total[s] + page - 1) // page
        table[s, :need] = perm[k:k + need]
        k += need
        if window:
            table[s, :max(0, past[s] + 1 - window) // 128 * 128 // page] = -1
    scales = torch.tensor([0.0021, 0.0034])
    layer = fill_layer(random_layer(g, pages, hkv, page, d, scales), g, table, total, scales, spread)
    return build_step_meta(q_lens, past, table, page), layer, scales, g


def oracle_attention(q, layer, meta, scale, scales, window=0, sinks=None, weights=None, decay=1.0):
    """64-bit attention; rows that see nothing give zeros.  Returns ``(out, weights)``."""
    vals = page_values(layer, scales)
    hkv, p = layer.shape[2:4]
    g = q.shape[1] // hkv
    out = torch.zeros(q.shape, dtype=torch.float64)
    w = None if weights is None else weights.double().clone()
    for s in range(meta.num_seqs):
        r0, ql, past = int(meta.q_start[s]), int(meta.q_len[s]), int(meta.past_len[s])
        given = torch.zeros(hkv, past + ql, dtype=torch.float64)
        touched = torch.zeros(past + ql, dtype=torch.bool)
        for r in range(ql):
            i = past + r
            keys = [j for j in range(max(0, i - window + 1) if window else 0, i + 1) if meta.page_table[s, j // p] >= 0]
            if not keys:
                continue
            keys = torch.tensor(keys)
            touched[keys] = True
            pg = meta.page_table[s].long()[keys // p]
            for h in range(q.shape[1]):
                k, v = vals[pg, 0, h // g, keys % p], vals[pg, 1, h // g, keys % p]
                z = k @ q[r0 + r, h].double() * scale
                if sinks is not None:
                    z = torch.cat([z, sinks[h].double().view(1)])
                pr = torch.softmax(z, 0)[:len(keys)]
                out[r0 + r, h] = pr @ v
                given[h // g, keys] += pr
        if w is not None:
            j = torch.arange(past + ql)[touched]
            pg = meta.page_table[s].long()[j // p]
            old = torch.where(j < past, 1.0, 0.0)[:, None] * w[pg, :, j % p] * decay
            w[pg, :, j % p] = old + given[:, touched].t()
    return out, w


def oracle_evict(weights, table, lengths, p, keep, first, recent):
    """Kept rows ``[sequences][head]`` by sorting."""
    out = []
    for s, n in enumerate(lengths):
        heads = []
        for h in range(weights.shape[1]):
            if n <= keep:
                heads.append(list(range(n)))
                continue
            mid = list(range(first, n - recent))
            w = [float(weights[table[s, j // p], h, j % p]) for j in mid]
            w = [math.inf if x != x else x for x in w]
            best = sorted(range(len(mid)), key=lambda a: (-w[a], a))[:keep - first - recent]
            heads.append(list(range(first)) + sorted(mid[b] for b in best) + list(range(n - recent, n)))
        out.append(heads)
    return out
