"""Refusals and argument checks of the paged cache that run on the host (no GPU)."""
import ctypes

import numpy as np
import pytest
import torch

from kvq import _lib, paged

DEV = "cuda:0"


def test_batch_refuses_what_does_not_fit():
    ok = dict(block_table=[[0, 1], [2, 3]], kv_lens=[20, 17], q_lens=[1, 17], page_size=16)

    def bad(match, exc=ValueError, **kw):
        with pytest.raises(exc, match=match):
            paged.PagedBatch(**{**ok, **kw}, device=DEV)

    bad("page_size", page_size=24)
    bad("2, 2 and 1 sequences", q_lens=[1])
    bad(">= 0", kv_lens=[20, -1])
    bad("needs 3 pages", kv_lens=[20, 33])
    bad("not a page", block_table=[[0, -1], [2, 3]])
    bad("whole numbers", kv_lens=[20.0, 17.0])
    bad("2-D", block_table=[0, 1])
    bad("fewer than 2\\^31", kv_lens=[2 ** 30, 2 ** 30])
    with pytest.raises(RuntimeError, match="no CPU path"):
        paged.PagedBatch(**ok, device="cpu")


def test_cache_refuses_unsupported_formats():
    for kw, match in ((dict(head_dim=64), "head_dim"), (dict(k_bits=4, v_bits=8), "bits"), (dict(page_size=48), "page_size"),
                      (dict(group_mode="blind16"), "group modes"), (dict(n_pages=0), "n_pages")):
        args = dict(n_pages=4, page_size=16, n_heads=2, head_dim=128, device=DEV)
        with pytest.raises(ValueError, match=match):
            paged.PagedKVCache(**{**args, **kw})
    with pytest.raises(RuntimeError, match="no CPU path"):
        paged.PagedKVCache(4, 16, 2, device="cpu")


def test_c_entry_points_refuse_bad_arguments(libkvq):
    cb = np.repeat(np.arange(4, dtype=np.int32), 32)
    p = 4096

    def cache(**kw):
        c = dict(k_pages=p, v_pages=p, n_pages=8, page_size=16, n_heads=2, head_dim=128, k_bits=4, v_bits=4, n_groups=4,
                 chan_band=cb.ctypes.data)
        return ctypes.byref(_lib.PagedCacheArgs(**{**c, **kw}))

    def batch(**kw):
        b = dict(table=p, table_stride=2, seqs=p, n_new=2, n_tokens=20, n_new_blocks=2, n_blocks=3, n_seqs=2)
        return ctypes.byref(_lib.PagedBatchArgs(**{**b, **kw}))

    def append(c, b, k=p, ks=256):
        return libkvq.kvq_paged_append(k, ks, p, 256, c, b, None)

    assert append(None, batch()) == -1 and append(cache(), None) == -1
    assert append(cache(head_dim=64), batch()) == -2
    assert append(cache(k_bits=4, v_bits=8), batch()) == -2 and b"bits" in libkvq.kvq_last_error()
    assert append(cache(page_size=20), batch()) == -2
    assert append(cache(n_pages=0), batch()) == -1
    assert append(cache(n_pages=1 << 31), batch()) == -1
    assert append(cache(k_pages=p + 8), batch()) == -4
    assert append(cache(v_pages=0), batch()) == -1
    blind16 = np.repeat(np.arange(8, dtype=np.int32), 16)
    assert append(cache(chan_band=blind16.ctypes.data, n_groups=8), batch()) == -2
    assert append(cache(), batch(n_new=-1)) == -1
    assert append(cache(), batch(seqs=p + 4)) == -4
    assert append(cache(), batch(table=0)) == -1
    assert append(cache(), batch(), ks=255) == -1
    assert append(cache(), batch(), ks=260) == -4
    assert append(cache(), batch(), k=p + 2) == -4
    assert append(cache(), batch(), k=0) == -1
    assert append(cache(), batch(n_new=0)) == 0
    assert libkvq.kvq_paged_read(cache(), batch(), 0, 0, 256, p, 256, None) == -1
    assert libkvq.kvq_paged_read(cache(), batch(n_tokens=0), 0, p, 256, p, 256, None) == 0


def format_args(n_heads=2, k_bits=4, v_bits=4):
    cb = np.repeat(np.arange(4, dtype=np.int32), 32)
    return _lib.PagedCacheArgs(4096, 4096, 8, 16, n_heads, 128, k_bits, v_bits, 4, cb.ctypes.data), cb


def plan_of(lib, kv, q, n_heads=2, group=1, causal=1, window=0, sink=0, n_sms=148, capacity=None):
    """(status, info, items [n, 16] of the kernel for few rows, of the one for many, cta_first)."""
    c, keep = format_args(n_heads)
    kv, q = np.asarray(kv, dtype=np.int32), np.asarray(q, dtype=np.int32)
    info = _lib.PagedPlanInfo()
    args = (ctypes.byref(c), kv.ctypes.data, q.ctypes.data, len(kv), n_heads * group, causal, window, sink, n_sms)
    assert lib.kvq_paged_plan(*args, None, 0, ctypes.byref(info)) == 0
    words = np.full(info.words + 8, 77, dtype=np.int32)
    rc = lib.kvq_paged_plan(*args, words.ctypes.data, info.words if capacity is None else capacity, ctypes.byref(info))
    assert (words[info.words:] == 77).all()  # nothing past its length
    a, b = info.n_row_items * 16, (info.n_row_items + info.n_tile_items) * 16
    return rc, info, words[:a].reshape(-1, 16), words[a:b].reshape(-1, 16), words[b:info.words]


BATCHES = [
    ([1], [1]), ([0, 0], [0, 0]), ([0, 5], [3, 0]), ([16], [16]), ([700, 33, 200, 0, 1], [1, 1, 1, 1, 1]),
    ([100000], [1]), ([100000, 7], [1, 7]), ([5000] * 64, [1] * 64), ([3000, 40, 2000], [9, 40, 600]), ([4680], [4680]),
    ([20000, 100], [300, 4]), ([257], [300]),
]


@pytest.mark.parametrize("kv,q", BATCHES)
@pytest.mark.parametrize("group", [1, 5, 8])
@pytest.mark.parametrize("causal,window,sink", [(1, 0, 0), (0, 0, 0), (1, 100, 20), (0, 33, 7), (1, 10 ** 6, 5)])
@pytest.mark.parametrize("n_sms", [1, 148])
def test_plan_covers_every_row_and_block_once(libkvq, kv, q, group, causal, window, sink, n_sms):
    heads = 2
    rc, info, few, many, cta_first = plan_of(libkvq, kv, q, heads, group, causal, window, sink, n_sms)
    assert rc == 0
    if info.n_row_items == info.n_row_ctas:
        assert len(cta_first) in (0, info.n_row_ctas + 1 if info.n_row_ctas else 0)
    else:  # each block of threads has its share of the items, in order
        assert len(cta_first) == info.n_row_ctas + 1 and cta_first[0] == 0 and cta_first[-1] == info.n_row_items
        assert (np.diff(cta_first) >= 1).all()
    q_first = np.concatenate(([0], np.cumsum(q)))
    slots = {0: [], 1: []}
    units = []
    seen = {(s, h): np.zeros(q[s] * group, dtype=int) for s in range(len(kv)) for h in range(heads)}
    for kind, items, most in ((0, few, info.row_tile), (1, many, 256)):
        by_unit = {}
        for it in items:
            s, h, row0, n_rows, n_sink, first, jb, je, part, parts, unit, slot, kv_len, start, qf, _ = (int(x) for x in it)
            assert 1 <= n_rows <= most and kv_len == kv[s] and start == kv[s] - q[s] and qf == q_first[s]
            assert kind == 0 if q[s] * group <= 16 else q[s] * group <= 64 or kind == 1
            by_unit.setdefault((s, h, row0, n_rows), []).append((part, parts, jb, je, n_sink, first, unit, slot))
        for (s, h, row0, n_rows), parts in by_unit.items():
            seen[s, h][row0:row0 + n_rows] += 1
            n = parts[0][1]
            assert sorted(p[0] for p in parts) == list(range(n)) and len({p[1:2] + p[4:] for p in parts}) == 1
            parts.sort()
            _, _, _, end, n_sink, first, unit, slot = parts[-1]
            assert parts[0][2] == 0 and all(a[3] == b[2] for a, b in zip(parts, parts[1:]))
            if kind == 1:  # parts begin on tiles of four storage blocks
                assert all(p[2] % 4 == 0 for p in parts)
            if n > 1:
                units.append(unit)
                slots[kind] += range(slot, slot + n)
            # the blocks listed are those some row of the unit sees, each once
            p = start_of(kv[s], q[s]) + (row0 + np.arange(n_rows)) // group
            j = np.arange(kv[s])
            vis = np.ones((n_rows, kv[s]), dtype=bool)
            if causal:
                vis &= j[None] <= p[:, None]
            if window:
                vis &= (j[None] > p[:, None] - window) | (j[None] < sink)
            need = set((np.flatnonzero(vis.any(0)) // 16).tolist())
            listed = list(range(n_sink)) + list(range(first, first + end - n_sink))
            assert len(listed) == len(set(listed)) and need <= set(listed)
            assert all(0 <= b < -(-kv[s] // 16) for b in listed)
            assert len(listed) <= len(need) + 1  # a kept block may lie past what a causal row sees
    assert all((x == 1).all() for x in seen.values())
    assert sorted(units) == list(range(info.n_units))
    for kind in slots:
        assert sorted(slots[kind]) == list(range(len(slots[kind])))
    assert info.tile_workspace_offset >= len(slots[0]) * info.row_tile * 130 * 4
    assert info.workspace_bytes == info.tile_workspace_offset + len(slots[1]) * 2 * 33 * 128 * 16


def start_of(kv, q):
    return kv - q


def test_plan_shares_the_work(libkvq):
    """A long sequence with one row is shared by about as many blocks of threads as there
    are SMs, and a ragged batch gives each the same number of storage blocks."""
    _, info, few, _, cta_first = plan_of(libkvq, [200000], [1], n_heads=1)
    assert info.n_row_ctas >= 100 and len(few) == info.n_row_ctas
    lens = (np.arange(1, 200) * 977) % 9000 + 1
    _, info, few, _, cta_first = plan_of(libkvq, lens, [1] * len(lens), n_heads=2)
    work = np.add.reduceat(few[:, 7] - few[:, 6], cta_first[:-1])
    assert info.n_row_ctas > 148 and work[:-1].max() - work[:-1].min() <= 1


def test_plan_refuses(libkvq):
    rc, info, *_ = plan_of(libkvq, [500, 20], [1, 1], capacity=15)
    assert rc == -1 and info.words > 15 and b"words" in libkvq.kvq_last_error()
    c, keep = format_args()
    kv = np.array([4, 4], dtype=np.int32)
    info = _lib.PagedPlanInfo()

    def plan(cache=c, kv=kv, q=kv, n=2, heads=2, window=0, sink=0, sms=148, out=info):
        return libkvq.kvq_paged_plan(ctypes.byref(cache), None if kv is None else kv.ctypes.data, q.ctypes.data, n, heads, 1,
                                     window, sink, sms, None, 0, None if out is None else ctypes.byref(out))

    assert plan() == 0 and plan(n=0, kv=None) == 0
    assert plan(kv=None) == -1 and plan(n=-1) == -1 and plan(sms=0) == -1 and plan(out=None) == -1
    assert plan(heads=3) == -1 and plan(heads=0) == -1 and plan(heads=65536) == -1
    assert plan(window=-1) == -1 and plan(sink=-1) == -1
    assert plan(kv=np.array([4, -1], dtype=np.int32)) == -1 and b"sequence 1" in libkvq.kvq_last_error()
    assert plan(cache=format_args(k_bits=4, v_bits=8)[0]) == -2


def test_attention_entry_refuses_bad_arguments(libkvq):
    cb = np.repeat(np.arange(4, dtype=np.int32), 32)
    p = 4096
    c = _lib.PagedCacheArgs(p, p, 8, 16, 2, 128, 4, 4, 4, cb.ctypes.data)
    b = _lib.PagedBatchArgs(p, 2, p, 2, 20, 2, 3, 2, 0)
    plan = _lib.PagedPlanInfo(n_row_items=2, n_row_ctas=1, n_units=1, words=34, workspace_bytes=256)

    def attend(q=p, qs=512, cache=c, batch=b, out=p, os_=512, lse=None, heads=4, window=0, sink=0, scale=0.0, info=plan,
               items=p, ws=p, ctr=p):
        ref = lambda x: None if x is None else ctypes.byref(x)
        return libkvq.kvq_paged_attention(q, qs, ref(cache), ref(batch), out, os_, lse, heads, 1, window, sink, scale,
                                          ref(info), items, ws, ctr, None)

    assert attend(cache=None) == -1 and attend(batch=None) == -1
    assert attend(heads=3) == -1 and attend(heads=0) == -1
    assert attend(window=-1) == -1 and attend(sink=-1) == -1
    assert attend(scale=float("nan")) == -1 and attend(scale=float("inf")) == -1 and attend(scale=2e38) == -1
    assert attend(q=None) == -1 and attend(out=None) == -1 and attend(qs=511) == -1 and attend(os_=504) == -1
    assert attend(q=p + 8) == -4 and attend(out=p + 2) == -4 and attend(qs=516) == -4 and attend(lse=p + 2) == -4
    assert attend(info=None) == -1 and attend(items=None) == -1 and attend(items=p + 4) == -4
    assert attend(ws=None) == -1 and attend(ctr=None) == -1 and attend(ws=p + 128) == -4
    assert attend(batch=_lib.PagedBatchArgs(p, 2, p, 0, 20, 0, 3, 2, 0)) == 0  # no new tokens


def test_plan_and_entries_refuse_sizes_before_they_work_on_them(libkvq):
    """More rows than a launch has are refused before their work list is made (it would fill the
    host's memory), and block counts beyond a grid before they are cut to 32 bits."""
    c, keep = format_args(n_heads=1)
    q = np.full(3, (2 ** 31 - 1) // 65535, dtype=np.int32)
    info = _lib.PagedPlanInfo()
    assert libkvq.kvq_paged_plan(ctypes.byref(c), q.ctypes.data, q.ctypes.data, 3, 65535, 1, 0, 0, 148, None, 0,
                                 ctypes.byref(info)) == -1
    assert b"too many rows" in libkvq.kvq_last_error()
    p = 4096
    for kw in (dict(n_new_blocks=1 << 32), dict(n_blocks=(1 << 32) + 3)):
        b = dict(table=p, table_stride=2, seqs=p, n_new=2, n_tokens=20, n_new_blocks=2, n_blocks=3, n_seqs=2)
        b = ctypes.byref(_lib.PagedBatchArgs(**{**b, **kw}))
        c2 = ctypes.byref(format_args()[0])
        assert libkvq.kvq_paged_append(p, 256, p, 256, c2, b, None) == -1
        assert libkvq.kvq_paged_read(c2, b, 0, p, 256, p, 256, None) == -1
