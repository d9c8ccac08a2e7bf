"""Measured cases of the paged, quantized KV cache: writing new tokens into its pages, reading them
back, and attention of a chunk of new tokens over them.

A page holds `page` tokens of one KV head; a page's K (and V) rows are stored 16 tokens at a time as
16 rows of codes followed by 16 rows of bf16 scales, one scale per (token, head, channel group):
pool uint8 [pages, heads, page / 16, 16 * (code bytes + 2 * groups)]. int4 codes hold two channels
per byte (code = q + 8, even channel low), int8 codes one (code = q + 128). A stored element stands
for q * scale. Sequences own pages through a block table; the new tokens of a sequence are its last
q_len ones.
"""
from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

D = 128
BLOCK = 16  # tokens of one storage block
EDGES = {
    "bands": (0, 44, 86, 128),
    "bands4": (0, 12, 24, 36, 44, 56, 68, 80, 86, 98, 110, 122, 128),
    "blind32": (0, 32, 64, 96, 128),
    "blind64": (0, 64, 128),
}


def _package():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "krea-realtime-bench_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from kvq import paged
    return paged


# ---------------------------------------------------------------- cases
def listed():
    return [
        # one new token for each of 24 running sequences (8 KV heads): the write of a decode step
        dict(name="append_decode", op="append", seqs=24, q=1, q_spread=0.0, kv=4097, kv_spread=0.9, heads=8, group=1,
             k_bits=4, v_bits=4, mode="blind32", page=16),
        # prompts of 1 to 1531 tokens written side by side, int8 K and V
        dict(name="append_ragged", op="append", seqs=9, q=1531, q_spread=0.97, kv=1531, kv_spread=0.97, heads=10,
             group=1, k_bits=8, v_bits=8, mode="blind64", page=32),
        # one 3-frame block of 4680 tokens, 40 heads, at the end of a window of 21 frames
        dict(name="append_block", op="append", seqs=1, q=4680, q_spread=0.0, kv=32760, kv_spread=0.0, heads=40,
             group=1, k_bits=4, v_bits=4, mode="bands4", page=64),
        # a short context with an odd length read back
        dict(name="read_short", op="read", seqs=3, q=1, q_spread=0.0, kv=777, kv_spread=0.5, heads=5, group=1,
             k_bits=8, v_bits=4, mode="bands", page=16),
        # the whole window of 21 frames of one layer read back
        dict(name="read_window", op="read", seqs=1, q=1, q_spread=0.0, kv=32760, kv_spread=0.0, heads=40, group=1,
             k_bits=4, v_bits=4, mode="bands4", page=64),
        # one token of one sequence: the latency of a single decode step
        dict(name="decode_one", op="attention", seqs=1, q=1, q_spread=0.0, kv=1561, kv_spread=0.0, heads=8, group=4,
             causal=True, window=0, sink=0, k_bits=4, v_bits=4, mode="blind32", page=16),
        # a running batch of sequences of very different lengths
        dict(name="decode_batch", op="attention", seqs=64, q=1, q_spread=0.0, kv=16384, kv_spread=0.95, heads=8,
             group=5, causal=True, window=0, sink=0, k_bits=4, v_bits=4, mode="blind32", page=16),
        # a few very long contexts, int8 keys, one KV head per query head, rotary-band groups
        dict(name="decode_long", op="attention", seqs=2, q=1, q_spread=0.0, kv=131071, kv_spread=0.3, heads=10,
             group=1, causal=True, window=0, sink=0, k_bits=8, v_bits=4, mode="bands4", page=64),
        # several drafted tokens per sequence verified at once
        dict(name="verify_drafts", op="attention", seqs=12, q=6, q_spread=0.5, kv=6240, kv_spread=0.6, heads=4,
             group=8, causal=True, window=0, sink=0, k_bits=8, v_bits=8, mode="blind64", page=32),
        # chunks of prompts and single tokens in one step, a sliding window behind a kept first frame
        dict(name="mixed_step", op="attention", seqs=6, q=1021, q_spread=1.0, kv=9360, kv_spread=0.7, heads=8, group=4,
             causal=True, window=4680, sink=1560, k_bits=4, v_bits=4, mode="bands", page=32),
        # a 2000-token chunk of a long prompt, grouped heads, causal
        dict(name="prompt_chunk", op="attention", seqs=1, q=2000, q_spread=0.0, kv=18720, kv_spread=0.0, heads=8,
             group=5, causal=True, window=0, sink=0, k_bits=4, v_bits=4, mode="blind32", page=16),
        # a denoising block of 4680 queries over the window of 21 frames, 40 heads, every query sees all of it
        dict(name="block_window", op="attention", seqs=1, q=4680, q_spread=0.0, kv=32760, kv_spread=0.0, heads=40,
             group=1, causal=False, window=0, sink=0, k_bits=4, v_bits=4, mode="bands4", page=64),
    ]


def _between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("append", "read", "decode", "decode", "chunk", "chunk"))
    k_bits, v_bits = rng.choice(((4, 4), (4, 4), (8, 4), (8, 8)))
    c = dict(op=op, q_spread=round(rng.uniform(0.0, 0.9), 3), kv_spread=round(rng.uniform(0.0, 0.9), 3), group=1,
             k_bits=k_bits, v_bits=v_bits, mode=rng.choice(tuple(EDGES)), page=rng.choice((16, 32, 64, 128)))
    if op in ("append", "read"):
        c["heads"] = rng.choice((1, 4, 5, 8, 10, 20, 40))
        most = (4680 if op == "append" else 32760) * 40 // c["heads"]
        tokens = _between(rng, 1, min(most, 60000))
        c["seqs"] = min(_between(rng, 1, 64), tokens)
        c["q"] = tokens // c["seqs"] if op == "append" else 1
        c["kv"] = c["q"] + rng.randrange(0, 3000) if op == "append" else tokens // c["seqs"]
        return c
    c["op"] = "attention"
    c["heads"] = rng.choice((1, 2, 4, 5, 8, 10))
    c["group"] = rng.choice((1, 2, 4, 5, 7, 8))
    c["window"], c["sink"] = rng.choice(((0, 0), (0, 0), (rng.randrange(100, 5000), rng.randrange(0, 1600))))
    if op == "decode":
        c["causal"] = True
        c["seqs"] = _between(rng, 1, 64)
        c["q"] = rng.choice((1, 1, 1, 2, 3, 5, 8))
        c["kv"] = _between(rng, 16, max(17, min(131072, 64 * 16384 * 8 // (c["seqs"] * c["heads"]))))
        c["q"] = min(c["q"], c["kv"])
    else:
        c["causal"] = rng.random() < 0.75
        c["seqs"] = rng.choice((1, 1, 2, 3, 6))
        c["q"] = _between(rng, 16, 4680)
        heads = c["heads"] * c["group"]
        most = min(32760, 4680 * 32760 * 40 // (4 * c["seqs"] * c["q"] * heads))
        c["kv"] = max(c["q"], _between(rng, 64, max(65, most)))
    return c


def _lens(case):
    """(kv lengths, new-token counts) of the case's sequences: the first has the full length, the others
    spread below it."""
    b = np.arange(case["seqs"], dtype=np.float64)
    kv = np.maximum(1, np.rint(case["kv"] * (1.0 - case["kv_spread"] * np.mod(b * 0.6180339887, 1.0)))).astype(np.int64)
    q = np.maximum(1, np.rint(case["q"] * (1.0 - case["q_spread"] * np.mod(b * 0.7548776662, 1.0)))).astype(np.int64)
    return kv, np.minimum(q, kv)


# ---------------------------------------------------------------- storage in plain torch
def _gid(case, device):
    e = EDGES[case["mode"]]
    return torch.from_numpy(np.repeat(np.arange(len(e) - 1), np.diff(e))).to(device)


def _rows(x, gid, bits):
    """x fp32 [..., 128] -> (codes uint8 [..., code bytes], scales bf16 [..., groups])."""
    qmax = float((1 << (bits - 1)) - 1)
    groups = int(gid[-1]) + 1
    amax = torch.zeros(x.shape[:-1] + (groups,), dtype=torch.float32, device=x.device)
    amax.scatter_reduce_(-1, gid.expand(x.shape), x.abs(), "amax")
    s = amax / torch.full_like(amax, qmax)  # a tensor: by a number torch multiplies with its reciprocal
    s = torch.where(s > 0, s, torch.ones_like(s))
    c = torch.round(x / s[..., gid]).clamp_(-qmax, qmax).add_(qmax + 1).to(torch.uint8)
    if bits == 4:
        c = c[..., 0::2] | (c[..., 1::2] << 4)
    return c, s.to(torch.bfloat16)


def _values(codes, scales, gid, bits):
    """The values that codes and scales stand for, fp32 [..., 128]."""
    if bits == 4:
        q = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2).float() - 8.0
    else:
        q = codes.float() - 128.0
    return q * scales.float()[..., gid]


def _parts(pool, page, bits):
    """(codes, scales) views of a pool, [pages, heads, page / 16, 16, ...]."""
    n, h, nb, size = pool.shape
    cw = D // 2 if bits == 4 else D
    codes = pool[..., : BLOCK * cw].unflatten(-1, (BLOCK, cw))
    scales = pool[..., BLOCK * cw:].view(torch.bfloat16).unflatten(-1, (BLOCK, (size // BLOCK - cw) // 2))
    return codes, scales


def _places(table, tokens, page):
    """(page id, block, row) of token positions [B, n] through a block table [B, most pages]."""
    ids = torch.gather(table, 1, torch.div(tokens, page, rounding_mode="floor"))
    off = tokens % page
    return ids, torch.div(off, BLOCK, rounding_mode="floor"), off % BLOCK


def _fetch(pool, places, gid, page, bits):
    """Values [..., heads, 128] fp32 of the tokens at `places`."""
    codes, scales = _parts(pool, page, bits)
    ids, blk, row = places
    return _values(codes[ids, :, blk, row], scales[ids, :, blk, row], gid, bits)


# ---------------------------------------------------------------- inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    kv, q = _lens(case)
    page, heads = case["page"], case["heads"]
    pages = -(-kv // page)
    n_pages = int(pages.sum()) + 3
    perm = torch.randperm(n_pages, generator=g, device=dev).cpu().numpy()
    table = np.zeros((len(kv), int(pages.max())), dtype=np.int32)
    first = np.concatenate(([0], np.cumsum(pages)))
    for b in range(len(kv)):
        table[b, : pages[b]] = perm[first[b]: first[b + 1]]
    gid = _gid(case, dev)
    groups = len(EDGES[case["mode"]]) - 1
    # keys with channel outliers, values without
    chan = torch.exp(0.5 * torch.randn(heads, 1, 1, D, generator=g, device=dev))

    def pool(bits, factor):
        size = BLOCK * ((D // 2 if bits == 4 else D) + 2 * groups)
        p = torch.zeros((n_pages, heads, page // BLOCK, size), dtype=torch.uint8, device=dev)
        if case["op"] == "append":
            return p
        codes, scales = _parts(p, page, bits)
        step = max(1, (1 << 26) // (heads * page * D))
        for i in range(0, n_pages, step):
            n = min(step, n_pages - i)
            x = torch.randn(n, heads, page // BLOCK, BLOCK, D, generator=g, device=dev)
            c, s = _rows((x * factor).bfloat16().float(), gid, bits)
            codes[i: i + n] = c
            scales[i: i + n] = s
        return p

    s = dict(case=case, k_pool=pool(case["k_bits"], chan), v_pool=pool(case["v_bits"], 1.0),
             table=torch.from_numpy(table).long().to(dev), gid=gid, kv=torch.from_numpy(kv).to(dev),
             q_len=torch.from_numpy(q).to(dev), kv_host=kv, q_host=q, table_host=table)
    total = int(q.sum())
    if case["op"] == "append":
        s["k"] = (torch.randn(total, heads, D, generator=g, device=dev) * chan[:, 0, 0]).bfloat16()
        s["v"] = torch.randn(total, heads, D, generator=g, device=dev).bfloat16()
    elif case["op"] == "attention":
        s["q"] = torch.randn(total, heads * case["group"], D, generator=g, device=dev).bfloat16()
    if own:
        paged = _package()
        cache = paged.PagedKVCache(n_pages, page, heads, D, k_bits=case["k_bits"], v_bits=case["v_bits"],
                                   group_mode=case["mode"], device=dev)
        cache.k_pages.copy_(s["k_pool"])
        cache.v_pages.copy_(s["v_pool"])
        s["k_pool"] = s["v_pool"] = None
        s["cache"] = cache
        s["batch"] = paged.PagedBatch(table, kv, q, page, device=dev)
    return s


# ---------------------------------------------------------------- one pass
def _new_tokens(s):
    """(sequence, position) of every new token, in order."""
    ends = torch.cumsum(s["q_len"], 0)
    i = torch.arange(int(s["q_host"].sum()), device=ends.device)
    b = torch.searchsorted(ends, i, right=True)
    return b, i - (ends - s["q_len"])[b] + (s["kv"] - s["q_len"])[b]


def _plain_append(s):
    case = s["case"]
    b, pos = _new_tokens(s)
    ids, blk, row = _places(s["table"][b], pos[:, None], case["page"])
    at = ids[:, 0], blk[:, 0], row[:, 0]
    out = []
    for x, pool, bits in ((s["k"], s["k_pool"], case["k_bits"]), (s["v"], s["v_pool"], case["v_bits"])):
        codes, scales = _parts(pool, case["page"], bits)
        c, sc = _rows(x.float(), s["gid"], bits)
        codes[at[0], :, at[1], at[2]] = c
        scales[at[0], :, at[1], at[2]] = sc
        out.append(_fetch(pool, at, s["gid"], case["page"], bits).bfloat16())
    return tuple(out)


def _plain_read(s):
    case = s["case"]
    t = torch.arange(int(s["kv_host"].max()), device=s["table"].device)
    at = _places(s["table"], t.expand(case["seqs"], -1), case["page"])
    live = t < s["kv"][:, None]
    at = tuple(x[live] for x in at)
    return tuple(_fetch(pool, at, s["gid"], case["page"], bits).bfloat16()
                 for pool, bits in ((s["k_pool"], case["k_bits"]), (s["v_pool"], case["v_bits"])))


def _plain_attention(s):
    case = s["case"]
    dev = s["table"].device
    n, heads, group = case["seqs"], case["heads"], case["group"]
    most_q, most_kv = int(s["q_host"].max()), int(s["kv_host"].max())
    t = torch.arange(most_kv, device=dev)
    at = _places(s["table"], t.expand(n, -1), case["page"])
    k = _fetch(s["k_pool"], at, s["gid"], case["page"], case["k_bits"])
    v = _fetch(s["v_pool"], at, s["gid"], case["page"], case["v_bits"])
    # queries padded to the longest sequence: [n, heads, group * most_q, 128]
    i = torch.arange(most_q, device=dev)
    live = i < s["q_len"][:, None]
    q = torch.zeros((n, most_q, heads * group, D), dtype=torch.float32, device=dev)
    q[live] = s["q"].float()
    q = q.unflatten(2, (heads, group)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    logits = torch.matmul(q, k.permute(0, 2, 3, 1)).mul_(1.0 / math.sqrt(D))
    del k
    pos = (s["kv"] - s["q_len"])[:, None] + i
    seen = (t < s["kv"][:, None])[:, None, :].expand(n, most_q, most_kv)
    if case["causal"]:
        seen = seen & (t <= pos[:, :, None])
    if case["window"]:
        seen = seen & ((t > pos[:, :, None] - case["window"]) | (t < case["sink"]))
    logits = logits.view(n, heads, group, most_q, most_kv).masked_fill_(~seen[:, None, None], -math.inf)
    top = logits.amax(-1, keepdim=True).clamp_(min=-1e30)
    p = logits.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(n, heads, group * most_q, most_kv), v.permute(0, 2, 1, 3))
    o = o.view(n, heads, group, most_q, D) / total.clamp_(min=1e-30)
    o = o.permute(0, 3, 1, 2, 4).flatten(2, 3)
    return o[live].bfloat16()


def run(state):
    case = state["case"]
    if own:
        cache, batch = state["cache"], state["batch"]
        if case["op"] == "append":
            cache.append(state["k"], state["v"], batch)
            return cache.read(batch, new_only=True)
        if case["op"] == "read":
            return cache.read(batch)
        return _package().attention(state["q"], cache, batch, causal=case["causal"], window=case["window"],
                                    sink=case["sink"])
    return {"append": _plain_append, "read": _plain_read, "attention": _plain_attention}[case["op"]](state)


# ---------------------------------------------------------------- what a pass cannot do without
def _visible(case):
    """(query-token pairs, tokens that some query sees), summed over the sequences."""
    kv, q = _lens(case)
    pairs = tokens = 0
    for n, m in zip(kv.tolist(), q.tolist()):
        pos = np.arange(n - m, n)
        hi = pos + 1 if case["causal"] else np.full(m, n)
        lo = np.maximum(0, pos + 1 - case["window"]) if case["window"] else np.zeros(m, dtype=np.int64)
        kept = np.minimum(case["sink"], lo) if case["window"] else np.zeros(m, dtype=np.int64)
        pairs += int((hi - lo + kept).sum())
        tokens += int(hi.max() - lo.min() + kept.min())
    return pairs, tokens


def work(case):
    kv, q = _lens(case)
    groups = len(EDGES[case["mode"]]) - 1
    row = sum((D // 2 if b == 4 else D) + 2 * groups for b in (case["k_bits"], case["v_bits"]))
    table = 4 * int((-(-kv // case["page"])).sum())
    if case["op"] == "append":
        # new rows in, codes and scales out, the values read back out
        n = int(q.sum()) * case["heads"]
        return {"bytes": n * (2 * 2 * D + row + 2 * 2 * D) + table, "flops": n * 2 * D * 6}
    if case["op"] == "read":
        n = int(kv.sum()) * case["heads"]
        return {"bytes": n * (row + 2 * 2 * D) + table, "flops": n * 2 * D}
    pairs, tokens = _visible(case)
    rows = int(q.sum()) * case["heads"] * case["group"]
    return {"bytes": tokens * case["heads"] * row + rows * D * 4 + table,
            "flops": pairs * case["heads"] * case["group"] * 4 * D}


# ---------------------------------------------------------------- the definition in 64 bits
def _exact_rows(pool, ids, n, page, bits, edges):
    """Stored values of n tokens of one sequence, fp64 [n, heads, 128], block by block."""
    cw = D // 2 if bits == 4 else D
    raw = pool[ids].flatten(2, 2).permute(0, 2, 1, 3).flatten(0, 1)  # [blocks, heads, bytes]
    groups = len(edges) - 1
    c = raw[..., : BLOCK * cw].reshape(raw.shape[0], raw.shape[1], BLOCK, cw)
    sc = raw[..., BLOCK * cw:].contiguous().view(torch.bfloat16).double()
    sc = sc.reshape(raw.shape[0], raw.shape[1], BLOCK, groups)
    out = torch.empty(c.shape[:3] + (D,), dtype=torch.float64, device=pool.device)
    if bits == 4:
        out[..., 0::2] = (c % 16).double() - 8
        out[..., 1::2] = torch.div(c, 16, rounding_mode="floor").double() - 8
    else:
        out[...] = c.double() - 128
    for j in range(groups):
        out[..., edges[j]: edges[j + 1]] *= sc[..., j: j + 1]
    return out.permute(0, 2, 1, 3).flatten(0, 1)[:n]


def exact(case, seed):
    s = prepare(case, seed)
    edges, page = EDGES[case["mode"]], case["page"]
    kv, q = _lens(case)
    if case["op"] == "append":
        out = []
        for x, bits in ((s["k"].double(), case["k_bits"]), (s["v"].double(), case["v_bits"])):
            qmax = (1 << (bits - 1)) - 1
            y = torch.empty_like(x)
            for a, b in zip(edges[:-1], edges[1:]):
                # by the storage format the scale is a 32-bit number, and the code rounds the 32-bit quotient
                scale = (x[..., a:b].abs().max(-1, keepdim=True).values / qmax).float().double()
                scale = torch.where(scale > 0, scale, 1.0)
                y[..., a:b] = torch.round((x[..., a:b] / scale).float()).double() * scale.bfloat16().double()
            out.append(y)
        return tuple(out)
    table = [s["table"][b, : -(-int(kv[b]) // page)] for b in range(len(kv))]
    if case["op"] == "read":
        return tuple(torch.cat([_exact_rows(pool, table[b], int(kv[b]), page, bits, edges) for b in range(len(kv))])
                     for pool, bits in ((s["k_pool"], case["k_bits"]), (s["v_pool"], case["v_bits"])))
    out, first, group = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda"), 0, case["group"]
    for b in range(len(kv)):
        n, m = int(kv[b]), int(q[b])
        k = _exact_rows(s["k_pool"], table[b], n, page, case["k_bits"], edges)
        v = _exact_rows(s["v_pool"], table[b], n, page, case["v_bits"], edges)
        j = torch.arange(n, device="cuda")
        for i in range(0, m, 2048):
            rows = min(2048, m - i)
            pos = torch.arange(n - m + i, n - m + i + rows, device="cuda")[:, None]
            hidden = (j > pos) if case["causal"] else torch.zeros((rows, n), dtype=torch.bool, device="cuda")
            if case["window"]:
                hidden = hidden | ((pos - j >= case["window"]) & (j >= case["sink"]))
            for h in range(case["heads"] * group):
                x = s["q"][first + i: first + i + rows, h].double() @ k[:, h // group].T / math.sqrt(D)
                w = torch.softmax(x.masked_fill(hidden, -math.inf), -1)
                out[first + i: first + i + rows, h] = w @ v[:, h // group]
        first += m
    return out
