"""What a captured call of the paged cache needs at its replays outlives the caller's names."""
import gc
import weakref

import pytest
import torch

from kvq import paged
from test_paged_gpu import fill, make, rows_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q", [1, 130])
def test_a_captured_batch_is_kept_until_it_is_released(q):
    n = 3000
    cache, batch, table = make([n], [q], heads=1)
    fill(cache, table, [n])
    x, k = rows_of(q, 2, 9).cuda(), rows_of(q, 1, 10).cuda()

    def step():
        cache.append(k, k, batch)
        return paged.attention(x, cache, batch), *cache.read(batch, new_only=True)

    want = step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    alive = weakref.ref(batch)
    del batch, step
    gc.collect()
    assert alive() is not None, "its memory would be read after it was freed"  # and nothing is replayed
    junk = [torch.full((m,), -1, dtype=torch.int32, device="cuda") for m in (8, 64, 200, 1000, 5000) for _ in range(8)]
    for _ in range(2):
        for t in got:
            t.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    del g, junk
    cache.release_captured()
    gc.collect()
    assert alive() is None


@pytest.mark.parametrize("kind", ["append", "read", "attention"])
def test_each_kind_of_call_keeps_its_batch(kind):
    cache, _, table = make([40], [2], heads=1)
    fill(cache, table, [40])
    x, k = rows_of(2, 1, 1).cuda(), rows_of(2, 1, 2).cuda()

    def call(batch):
        if kind == "append":
            cache.append(k, k, batch)
        elif kind == "read":
            cache.read(batch)
        else:
            paged.attention(x, cache, batch)

    for captured in (False, True):
        batch = paged.PagedBatch(table, [40], [2], 16, device="cuda:0")
        call(batch)
        torch.cuda.synchronize()
        if captured:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                call(batch)
        alive = weakref.ref(batch)
        del batch
        gc.collect()
        assert (alive() is not None) == captured  # an eager call keeps nothing
    del g
    cache.release_captured()
    gc.collect()
    assert alive() is None
