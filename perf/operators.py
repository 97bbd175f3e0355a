"""Four-bit key / value caches as measurable cases: writing them, attending over them, and shortening them.

A layer of such a cache is ``uint8 [pages, 2, Hkv, P, 9 D / 16]``.  The slab of a page, of its keys or its values and of one head holds the codes
``[P, D / 2]`` (E2M1, the even feature in the low nibble) and then the block scales ``[P, D / 16]`` (E4M3, one per 16 features); a value is
``code * block scale * scales[0 keys, 1 values]``.  A page table names the pages of every sequence (-1: no page).

Four kinds of case: ``write`` (norm, rotation, quantisation and paged write of a step's rows), ``attend`` (attention of a step's rows over the pages),
``scored`` (the same, which also adds up the attention weight that every cached row gets) and ``evict`` (keep the first, the latest and the heaviest
rows of every sequence and head, in other pages).
"""
from __future__ import annotations

import math
import zlib

import torch

own = False

EPS = 1e-6
THETA = 1e6
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
BORDERS = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)      # between two levels; a value on one takes the even code


def listed():
    full = dict(hq=32, hkv=8, d=128, page=64, dtype="bf16", window=0, sinks=False, norm=True, spread=0.0)
    return [
        # cache writes: a decode step of the headline benchmark's 64 users; one long prompt, whose rows also go out in 16 bits for its own attention
        dict(full, name="write_batch64", kind="write", seqs=64, past=1088, rows=1, spread=0.3),
        dict(full, name="write_prompt", kind="write", seqs=1, past=0, rows=8129),
        # one user's token a little into a conversation, where latency counts
        dict(full, name="attend_token", kind="attend", seqs=1, past=700, rows=1),
        # decode of 64 users, 1024 tokens and a bit each
        dict(full, name="attend_batch64", kind="attend", seqs=64, past=1088, rows=1, spread=0.1, dtype="fp16"),
        # many long conversations, lengths apart
        dict(full, name="attend_long", kind="attend", seqs=30, past=4000, rows=1, spread=0.6),
        # one user asks about a book; eight query heads share a KV head (the 30B-A3B shape)
        dict(full, name="attend_document", kind="attend", seqs=1, past=131000, rows=1, hkv=4),
        # verification of short drafts under a sliding window whose older pages are gone, learned sinks, small heads
        dict(full, name="attend_verify", kind="attend", seqs=4, past=2048, rows=5, hq=16, hkv=4, d=64, page=128, dtype="fp16", window=1024, sinks=True),
        # a portion of a new prompt behind what is cached of it
        dict(full, name="attend_prompt", kind="attend", seqs=1, past=7000, rows=983),
        # decode steps that keep account of the attention weights, before rows are dropped
        dict(full, name="scored_batch", kind="scored", seqs=16, past=8192, rows=1, spread=0.1),
        # the last 32 rows of two prompts vote on what of them stays
        dict(full, name="scored_window", kind="scored", seqs=2, past=4000, rows=32, dtype="fp16"),
        # a batch is cut to a quarter of its rows; a book to 8000 rows
        dict(full, name="evict_batch", kind="evict", seqs=16, past=8192, rows=0, keep=2048, spread=0.1),
        dict(full, name="evict_document", kind="evict", seqs=1, past=131000, rows=0, keep=8000, hkv=4),
    ]


def draw(rng):
    log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    kind = rng.choice(["write", "attend", "attend", "prompt", "scored", "evict"])
    hkv, group = rng.choice([(8, 4), (8, 1), (4, 8), (4, 7), (2, 8), (2, 5), (1, 16), (1, 8)])
    c = dict(hq=hkv * group, hkv=hkv, d=rng.choice([64, 128, 128, 128, 256]), page=rng.choice([32, 64, 64, 128]), dtype=rng.choice(["bf16", "fp16"]),
             window=0, sinks=False, norm=rng.random() < 0.5, spread=rng.choice([0.0, 0.3, 0.8]))
    width = hkv * c["d"]
    if kind == "write":
        if rng.random() < 0.5:
            c.update(kind="write", seqs=log(1, 200), past=log(1, 4000), rows=log(1, 6))
        else:
            c.update(kind="write", seqs=1, past=rng.choice([0, log(1, 3000)]), rows=max(1, min(log(10, 8000), 8000 * 48 * 128 // ((c["hq"] + 2 * hkv) * c["d"]))))
        return c
    if kind == "prompt":
        rows, past = log(20, 1500), rng.choice([0, log(10, 8000)])
        rows = max(17, min(rows, 983 * 7500 * 32 * 128 // (max(1, past + rows) * c["hq"] * c["d"])))
        c.update(kind="attend", seqs=1, past=past, rows=rows)
        return c
    most = 120_000_000 // width                             # cached rows of all sequences
    seqs = log(1, 64)
    past = log(1, max(2, min(131000, most // seqs)))
    if kind == "evict":
        past = max(past // 2, 64)
        c.update(kind="evict", seqs=seqs, past=past, rows=0, keep=max(36, log(36, max(37, past))))
        return c
    rows = rng.choice([1, 1, 1, 2, rng.randint(3, 8)])
    c.update(kind=kind, seqs=seqs, past=past, rows=rows, sinks=rng.random() < 0.3)
    if rng.random() < 0.3:
        c["window"] = log(1, 4000)
    return c


# ---- inputs ----------------------------------------------------------------------------------------------------------------------

FIRST, RECENT = 4, 32                                       # rows that an eviction never drops


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float16


def _lengths(case, seed):
    """Cached rows of every sequence: ``past``, some of them fewer by up to ``spread``."""
    g = torch.Generator().manual_seed(seed)
    cut = torch.rand(case["seqs"], generator=g) * case["spread"]
    cut[0] = 0.0
    return [max(0 if case["past"] == 0 else 1, int(case["past"] * (1.0 - float(x)))) for x in cut]


def _layer(g, pages, case, scales):
    """Random pages: normal features, some of the key's channels larger, in blocks of 16 over their largest."""
    hkv, p, d = case["hkv"], case["page"], case["d"]
    out = torch.empty(pages, 2, hkv, p * (d // 2 + d // 16), dtype=torch.uint8, device="cuda")
    size = torch.ones(2, hkv, 1, d, device="cuda")
    size[0] += 2.0 * (torch.rand(hkv, 1, d, generator=g, device="cuda") < 0.05)
    for a in range(0, pages, 256):
        n = min(256, pages - a)
        x = torch.randn(n, 2, hkv, p, d, generator=g, device="cuda") * size
        code, sf = _encode(x, scales.view(2, 1, 1, 1))
        out[a:a + n, ..., :p * d // 2] = (code[..., 0::2] | (code[..., 1::2] << 4)).flatten(-2)
        out[a:a + n, ..., p * d // 2:] = sf.view(torch.uint8).flatten(-2)
    return out.view(pages, 2, hkv, p, d // 2 + d // 16)


def prepare(case, seed):
    seed = zlib.crc32(repr(("four-bit", int(seed))).encode())
    g = torch.Generator(device="cuda").manual_seed(seed)
    n, rows, p, d, hq, hkv, dt = case["seqs"], case["rows"], case["page"], case["d"], case["hq"], case["hkv"], _dtype(case)
    past = _lengths(case, seed)
    total = [x + rows for x in past]
    need = [(x + p - 1) // p for x in total]
    wide = (case["past"] + rows + p - 1) // p + 1
    pages = n * (wide - 1) + 3
    ids = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))
    table = torch.full((n, wide), -1, dtype=torch.int32)
    at = 0
    for s in range(n):
        table[s, :need[s]] = ids[at:at + need[s]].int()
        at += need[s]
        if case["window"]:                                  # pages wholly before the window have been handed back
            table[s, :max(0, past[s] + 1 - case["window"]) // 128 * 128 // p] = -1
    i32 = dict(dtype=torch.int32, device="cuda")
    t = n * rows
    scales = (5.6 / 2688.0) * (0.8 + 0.4 * torch.rand(2, generator=g, device="cuda"))
    st = dict(case=dict(case), scales=scales, layer=_layer(g, pages, case, scales), table=table.cuda(), past=torch.tensor(past, **i32))
    if case["kind"] == "evict":
        w = torch.rand(pages, hkv, p, generator=g, device="cuda")
        w = torch.where(torch.rand(pages, hkv, p, generator=g, device="cuda") < 0.2, torch.zeros_like(w), (w * 12.0 - 12.0).exp())     # many rows nobody looks at
        keep = (case["keep"] + p - 1) // p
        st.update(weights=torch.cat([w, torch.zeros(n * keep, hkv, p, device="cuda")]),
                  layer=torch.cat([st["layer"], torch.zeros(n * keep, *st["layer"].shape[1:], dtype=torch.uint8, device="cuda")]),
                  to=(pages + torch.randperm(n * keep, generator=g, device="cuda")).int().view(n, keep))
        return st
    st.update(scale=d ** -0.5, step=dict(
        q_start=torch.arange(0, t + 1, rows, **i32), q_len=torch.full((n,), rows, **i32), past_len=st["past"],
        positions=(st["past"][:, None] + torch.arange(rows, **i32)).reshape(-1), seq_ids=torch.arange(n, **i32).repeat_interleave(rows), page_table=st["table"],
        slot_ids=torch.arange(n, **i32), logits_idx=torch.arange(rows - 1, t, rows, **i32), page_size=p, num_seqs=n, num_tokens=t, max_q_len=rows,
        max_seq_len=max(total), host_lens=tuple((rows, x) for x in past)))
    if case["kind"] == "write":
        inv = THETA ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)
        ang = torch.arange(max(total), dtype=torch.float64, device="cuda")[:, None] * inv
        st["cos_sin"] = torch.cat([ang.cos(), ang.sin()], dim=1).float()
        st["qkv"] = (torch.randn(t, (hq + 2 * hkv) * d, generator=g, device="cuda") * 1.5).to(dt)
        norm = lambda: (1.0 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(dt) if case["norm"] else None  # noqa: E731
        st["q_norm"], st["k_norm"] = norm(), norm()
        # 16-bit pages for the step's own rows: those that hold one of them
        first = torch.tensor([x // p for x in past])
        own_pages = (torch.tensor(total) - 1) // p - first + 1
        most = (rows + p - 2) // p + 1
        stage = torch.full((n, wide), -1, dtype=torch.int32)
        for s in range(n):
            stage[s, int(first[s]):int(first[s] + own_pages[s])] = torch.arange(int(own_pages[s]), dtype=torch.int32) + s * most
        st["stage_table"] = stage.cuda()
        st["stage"] = torch.zeros(n * most, 2, hkv, p, d, dtype=dt, device="cuda")
        return st
    st["q"] = (torch.randn(t, hq, d, generator=g, device="cuda") * 1.7).to(dt)
    st["sinks"] = torch.randn(hq, generator=g, device="cuda") * 2.0 if case["sinks"] else None
    if case["kind"] == "scored":
        st["before"] = torch.rand(pages, hkv, p, generator=g, device="cuda") * 0.1
    return st


# ---- one pass --------------------------------------------------------------------------------------------------------------------

def run(st):
    case = st["case"]
    if own:
        from tensorrt_edge_llm_b200 import ops
        if case["kind"] == "evict":
            kept = ops.kv_evict(st["layer"], st["weights"], st["table"], st["past"], st["to"], case["keep"], first=FIRST, recent=RECENT)
            return kept, st["layer"], st["weights"]
        meta = ops.StepMeta(**st["step"])
        if case["kind"] == "write":
            q = ops.rope_kv_write_fp4(st["qkv"], st["layer"], meta, st["cos_sin"], case["hq"], case["hkv"], case["d"], st["scales"], st["q_norm"],
                                      st["k_norm"], EPS, stage=st["stage"], stage_table=st["stage_table"])
            return q, st["stage"]
        w = None if case["kind"] == "attend" else st["before"].clone()
        o = ops.paged_attention_fp4(st["q"], st["layer"], meta, st["scale"], st["scales"], sliding_window=case["window"] or None, sinks=st["sinks"],
                                    weights=w)
        return o if w is None else (o, w)
    return {"write": _write, "attend": _attend, "scored": _attend, "evict": _evict}[case["kind"]](st)


# ---- plain forms -----------------------------------------------------------------------------------------------------------------

def _encode(x, scale):
    """Codes 0..15 of fp32 ``x`` and the E4M3 scales of its blocks of 16."""
    b = x.unflatten(-1, (-1, 16))
    sf = (b.abs().amax(-1) / 6.0 / scale).clamp(max=448.0).to(torch.float8_e4m3fn)
    step = (sf.float() * scale)[..., None]
    y = torch.where(step > 0, b / step, torch.zeros_like(b)).flatten(-2)
    a = y.abs()
    code = sum(((a >= m) if i % 2 else (a > m)).to(torch.uint8) for i, m in enumerate(BORDERS))
    return code | (torch.signbit(x).to(torch.uint8) << 3), sf


def _codes(layer):
    """Signed levels and block scales (fp32) of packed rows ``[..., P, 9 D / 16]``."""
    p, width = layer.shape[-2:]
    d = width * 16 // 9
    flat = layer.flatten(-2)
    byte = flat[..., :p * d // 2].unflatten(-1, (p, d // 2))
    code = torch.stack([byte & 15, byte >> 4], dim=-1).flatten(-2).long()
    level = torch.tensor(LEVELS + tuple(-x for x in LEVELS), device=layer.device)
    return level[code], flat[..., p * d // 2:].contiguous().view(torch.float8_e4m3fn).unflatten(-1, (p, d // 16)).float()


def _values(layer, scales):
    """fp32 values ``[..., 2, Hkv, P, D]`` of packed pages."""
    level, sf = _codes(layer)
    step = sf * scales.view(2, 1, 1, 1)
    return (level.unflatten(-1, (-1, 16)) * step[..., None]).flatten(-2)


def _write(st):
    case, step = st["case"], st["step"]
    hq, hkv, d, p, t = case["hq"], case["hkv"], case["d"], case["page"], step["num_tokens"]
    dt = st["qkv"].dtype
    x = st["qkv"].view(t, hq + 2 * hkv, d).float()
    q, k, v = x.split([hq, hkv, hkv], dim=1)

    def turn(y, w):
        if w is not None:                                   # a 64-bit sum: the rounding behind it is next to a border of the codes
            inv = (1.0 / torch.sqrt(y.double().square().mean(-1, keepdim=True) + EPS)).float()
            y = ((y * inv).to(dt).float() * w.float()).to(dt).float()
        c, s = st["cos_sin"][step["positions"].long()][:, None].chunk(2, dim=-1)
        a, b = y.chunk(2, dim=-1)
        return torch.cat([a * c - b * s, b * c + a * s], dim=-1).to(dt)

    q, k = turn(q, st["q_norm"]), turn(k, st["k_norm"])
    kv = torch.stack([k.float(), v], dim=1)                                     # [T, 2, Hkv, D]
    code, sf = _encode(kv, st["scales"].view(2, 1, 1))
    packed = torch.cat([code[..., 0::2] | (code[..., 1::2] << 4), sf.view(torch.uint8)], dim=-1)
    slot = step["positions"].long()
    page, at = st["table"].long()[step["seq_ids"].long(), slot // p], slot % p
    pages = st["layer"].shape[0]
    flat = st["layer"].view(pages, 2, hkv, -1)
    flat[..., :p * d // 2].view(pages, 2, hkv, p, d // 2)[page, :, :, at] = packed[..., :d // 2]
    flat[..., p * d // 2:].view(pages, 2, hkv, p, d // 16)[page, :, :, at] = packed[..., d // 2:]
    level = torch.tensor(LEVELS + tuple(-x for x in LEVELS), device=code.device)[code.long()]
    back = (level.unflatten(-1, (-1, 16)) * (sf.float() * st["scales"].view(2, 1, 1))[..., None]).flatten(-2)
    st["stage"][st["stage_table"].long()[step["seq_ids"].long(), slot // p], :, :, at] = back.to(dt)
    return q, st["stage"]


def _attend(st):
    case, step = st["case"], st["step"]
    n, rows, p, d, hq, hkv = case["seqs"], case["rows"], case["page"], case["d"], case["hq"], case["hkv"]
    g = hq // hkv
    table = st["table"].long()
    kv = _values(st["layer"][table.clamp(min=0)], st["scales"])                 # [N, pages, 2, Hkv, P, D]
    k, v = (kv[:, :, i].transpose(1, 2).flatten(2, 3) for i in (0, 1))          # [N, Hkv, keys, D]
    keys = torch.arange(k.shape[2], device="cuda")
    last = st["past"].long()[:, None] + torch.arange(rows, device="cuda")       # [N, rows]
    seen = (keys <= last[..., None]) & (table >= 0).repeat_interleave(p, dim=1)[:, None]
    if case["window"]:
        seen = seen & (keys > last[..., None] - case["window"])
    q = st["q"].view(n, rows, hkv, g, d).permute(0, 2, 3, 1, 4).float()         # [N, Hkv, g, rows, D]
    score = (q.flatten(2, 3) @ k.transpose(-1, -2)).unflatten(2, (g, rows)) * st["scale"]
    score.masked_fill_(~seen[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    if st["sinks"] is not None:
        sink = st["sinks"].view(1, hkv, g, 1, 1)
        top = torch.maximum(top, sink)
    w = torch.exp(score - top)
    total = w.sum(-1, keepdim=True)
    if st["sinks"] is not None:
        total = total + torch.exp(sink - top)
    w = w / total
    v = torch.where(seen.any(1)[:, None, :, None], v, torch.zeros_like(v))
    out = (w.flatten(2, 3) @ v).unflatten(2, (g, rows)).permute(0, 3, 1, 2, 4).reshape(n * rows, hq, d).to(st["q"].dtype)
    if case["kind"] == "attend":
        return out
    table_w = st["before"].clone()
    add = w.sum((2, 3)).unflatten(2, (-1, p)).transpose(1, 2)                   # [N, pages, Hkv, P]
    new = (keys >= st["past"][:, None]).view(n, -1, 1, p)                       # the step's own rows start from nothing
    some = seen.any(1).view(n, -1, 1, p)
    old = table_w[table.clamp(min=0)]
    changed = torch.where(some, torch.where(new, add, old + add), old)
    real = table >= 0
    table_w[table[real]] = changed[real]
    return out, table_w


def _evict(st):
    case = st["case"]
    n, p, hkv, keep = case["seqs"], case["page"], case["hkv"], case["keep"]
    table = st["table"].long()
    length = st["past"].long()[:, None]
    keys = torch.arange(table.shape[1] * p, device="cuda")
    w = st["weights"][table.clamp(min=0)].transpose(1, 2).flatten(2)            # [N, Hkv, keys]
    sure = ((keys < FIRST) | (keys >= length - RECENT)) & (keys < length)
    rank = torch.where(sure[:, None], torch.full_like(w, float("inf")), w).masked_fill((keys >= length)[:, None], float("-inf"))
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep]
    if order.shape[-1] < keep:
        order = torch.nn.functional.pad(order, (0, keep - order.shape[-1]), value=keys.numel())
    kept = torch.where(order < length[..., None], order, torch.full_like(order, 1 << 30)).sort(-1).values
    there = kept < (1 << 30)
    src = torch.where(there, kept, torch.zeros_like(kept))
    page, at = table[torch.arange(n, device="cuda")[:, None, None], src // p], src % p
    j = torch.arange(keep, device="cuda")
    to = st["to"].long()[:, None, j // p].expand(n, hkv, keep)
    to_at = (j % p).expand(n, hkv, keep)
    head = torch.arange(hkv, device="cuda")[None, :, None].expand(n, hkv, keep)
    pages, d = st["layer"].shape[0], case["d"]
    flat = st["layer"].view(pages, 2, hkv, -1)
    ok = there
    for part in (flat[..., :p * d // 2].view(pages, 2, hkv, p, d // 2), flat[..., p * d // 2:].view(pages, 2, hkv, p, d // 16)):
        part[to[ok], :, head[ok], to_at[ok]] = part[page[ok], :, head[ok], at[ok]]
    st["weights"][to[ok], head[ok], to_at[ok]] = st["weights"][page[ok], head[ok], at[ok]]
    return torch.where(there, kept, torch.full_like(kept, -1)).int(), st["layer"], st["weights"]


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------------

def work(case):
    n, rows, d, hq, hkv = case["seqs"], case["rows"], case["d"], case["hq"], case["hkv"]
    row = 2 * hkv * d * 9 / 16                                                  # a cached row's keys and values
    cached = sum(_lengths(dict(case), 0))
    t = n * rows
    if case["kind"] == "write":
        return {"bytes": t * ((hq + 2 * hkv) * d * 2 + hq * d * 2 + row + 2 * hkv * d * 2) + min(t, case["past"] + rows) * d * 4, "flops": t * (hq + 2 * hkv) * d * 8.0}
    if case["kind"] == "evict":
        kept = sum(min(x, case["keep"]) for x in _lengths(dict(case), 0))
        return {"bytes": cached * hkv * 4 + kept * (2 * row + hkv * 12), "flops": float(cached * hkv)}
    past = _lengths(dict(case), 0)
    w = case["window"] or 1 << 60
    seen = sum(min(x + 1 + r, w) for x in past for r in range(rows))
    read = sum(min(x + rows, w + rows - 1) for x in past)
    scored = case["kind"] == "scored"
    return {"bytes": read * row + t * hq * d * 4 + (read * hkv * 8 if scored else 0), "flops": 4.0 * seen * hq * d}


# ---- 64 bits ---------------------------------------------------------------------------------------------------------------------

def _bytes_to_e4m3(b):
    """The values of E4M3 bytes, from the fields."""
    b = b.long()
    e, m = (b >> 3) & 15, (b & 7).double()
    v = torch.where(e == 0, m * 2.0 ** -9, (1.0 + m / 8.0) * torch.exp2((e - 7).double()))
    return torch.where(b >= 128, -v, v)


def _rows64(st, pages, kv, head):
    """``[pages * P, D]`` of one head's keys or values."""
    case = st["case"]
    p, d = case["page"], case["d"]
    slab = st["layer"][pages, kv, head].flatten(1)
    byte = slab[:, :p * d // 2].reshape(-1, d // 2).long()
    sf = _bytes_to_e4m3(slab[:, p * d // 2:].reshape(-1, d // 16)) * st["scales"][kv].double()
    level = torch.tensor(LEVELS, dtype=torch.float64, device="cuda")
    out = torch.empty(byte.shape[0], d, dtype=torch.float64, device="cuda")
    for half, nib in enumerate((byte % 16, byte // 16)):
        out[:, half::2] = level[nib % 8] * (1.0 - 2.0 * (nib // 8).double())
    return out * sf.repeat_interleave(16, dim=1)


def _kept64(st):
    """The weights after an eviction: every kept row's in its new place."""
    case = st["case"]
    p, out, w = case["page"], st["weights"].double(), st["weights"].double()
    for s, total in enumerate(st["past"].tolist()):
        pos = torch.arange(total, device="cuda")
        page = st["table"][s].long()[pos // p]
        new = pos[:min(total, case["keep"])]
        for h in range(case["hkv"]):
            mine = w[page, h, pos % p]
            rank = mine.clone()
            rank[:FIRST] = math.inf
            rank[max(0, total - RECENT):] = math.inf
            best = torch.sort(-rank, stable=True).indices[:case["keep"]].sort().values
            out[st["to"][s].long()[new // p], h, new % p] = mine[best]
    return out


def exact(case, seed):
    st = prepare(case, seed)
    n, rows, p, d, hq, hkv = case["seqs"], case["rows"], case["page"], case["d"], case["hq"], case["hkv"]
    if case["kind"] == "evict":
        return None, None, _kept64(st)                      # whole numbers, and copied bytes
    past = _lengths(case, zlib.crc32(repr(("four-bit", int(seed))).encode()))
    if case["kind"] == "write":
        dt = _dtype(case)
        x = st["qkv"].double().view(-1, hq + 2 * hkv, d)
        q, k = x[:, :hq], x[:, hq:hq + hkv]
        ang = st["cos_sin"].double()[st["step"]["positions"].long()]

        def turn(y, w):
            if w is not None:
                y = (y * (y.pow(2).mean(-1, keepdim=True) + EPS) ** -0.5).to(dt).double()
                y = (y * w.double()).to(dt).double()
            z = torch.empty_like(y)
            c, s = ang[:, None, :d // 2], ang[:, None, d // 2:]
            z[..., :d // 2] = y[..., :d // 2] * c - y[..., d // 2:] * s
            z[..., d // 2:] = y[..., d // 2:] * c + y[..., :d // 2] * s
            return z

        return turn(q, st["q_norm"]), None                  # the rows behind: codes of four bits, chosen at borders
    g = hq // hkv
    out = torch.empty(n, rows, hq, d, dtype=torch.float64, device="cuda")
    table = st["before"].double() if case["kind"] == "scored" else None
    for s in range(n):
        total = past[s] + rows
        mine = st["table"][s, :(total + p - 1) // p].long()
        pos = torch.arange(total, device="cuda")
        i = past[s] + torch.arange(rows, device="cuda")[:, None]
        hide = (pos > i) | (pos <= i - (case["window"] or 1 << 40)) | (mine < 0).repeat_interleave(p)[:total]
        gone = hide.all(0)
        for h in range(hkv):
            k, v = (_rows64(st, mine.clamp(min=0), kv, h)[:total] for kv in (0, 1))
            v[gone] = 0.0
            given = torch.zeros(total, dtype=torch.float64, device="cuda")
            for j in range(h * g, h * g + g):
                z = st["q"].view(n, rows, hq, d)[s, :, j].double() @ k.T * st["scale"]
                z[hide] = -math.inf
                if st["sinks"] is not None:
                    z = torch.cat([z, st["sinks"][j].double().expand(rows, 1)], dim=1)
                z = torch.softmax(z, dim=1)[:, :total]
                out[s, :, j] = z @ v
                given += z.sum(0)
            if table is not None:
                flat = table[:, h].reshape(-1)
                at = (mine.clamp(min=0)[:, None] * p + torch.arange(p, device="cuda")).reshape(-1)[:total]
                flat[at[~gone]] = (torch.where(pos < past[s], flat[at], 0.0) + given)[~gone]
                table[:, h] = flat.view(-1, p)
    out = out.reshape(n * rows, hq, d)
    return out if table is None else (out, table)
