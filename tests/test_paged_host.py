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
