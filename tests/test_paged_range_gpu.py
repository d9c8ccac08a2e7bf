"""Paged attention on the GPU where fp16 operands are short of range: channel groups of
different magnitude inside a token. Against its definition in 64 bits, with the tolerances of
test_paged_gpu.py, which hold every K and V value to fp16's relative rounding."""
import numpy as np
import pytest
import torch

from kvq import paged
from test_paged_gpu import FORMATS, check, make, rows_of, stored

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _seed():
    torch.manual_seed(4321)


def append(cache, table, kk, vv):
    n = kk.shape[0]
    cache.append(kk.cuda(), vv.cuda(), paged.PagedBatch(table, [n], [n], cache.page_size, device="cuda:0"))
    return stored(kk, cache.k_bits, cache.bands), stored(vv, cache.v_bits, cache.bands)


@pytest.mark.parametrize("q", [1, 12, 150])
@pytest.mark.parametrize("k_bits,v_bits", FORMATS)
@pytest.mark.parametrize("mode", ["bands", "bands4", "blind32", "blind64"])
@pytest.mark.parametrize("ratio", [1e-3, 2.0 ** -15, 1e-6])
def test_groups_of_different_magnitude(q, k_bits, v_bits, mode, ratio):
    """Every second group is smaller by a ratio, in keys and values; queries are larger there,
    so that each group has its share of the logits. One of them in its range otherwise, and
    tokens beyond it."""
    n = 217
    cache, batch, table = make([n], [q], heads=2, page=32, k_bits=k_bits, v_bits=v_bits, mode=mode)
    small = torch.ones(128)
    for lo, hi in cache.bands[1::2]:
        small[lo:hi] = ratio
    for ks, vs in ((1.0, 1.0), (0.05, 3.0), (1e5, 1e6), (1e-6, 1e-5)):
        kk, vv = ((rows_of(n, 2, s).float() * small * x).bfloat16() for s, x in ((3, ks), (4, vs)))
        kk[::3] *= 0.125
        x = (torch.randn(q, 4, 128) / small).bfloat16()
        k, v = append(cache, table, kk, vv)
        out = check(x.cuda(), cache, batch, k, v, scale=0.09 / ks)
        assert (out.abs() > 0).all()  # no group vanished


@pytest.mark.parametrize("q", [1, 12, 150])
@pytest.mark.parametrize("k_bits,v_bits", FORMATS)
@pytest.mark.parametrize("mode", ["bands", "bands4", "blind32", "blind64"])
@pytest.mark.parametrize("size", [1e-6, 1e-8, 1e-20])
def test_groups_of_zeros_beside_small_ones(q, k_bits, v_bits, mode, size):
    """A group of zeros is stored with the scale 1: it does not hide the others."""
    n = 217
    cache, batch, table = make([n], [q], heads=2, page=32, k_bits=k_bits, v_bits=v_bits, mode=mode)
    kk, vv = (rows_of(n, 2, s, size) for s in (3, 4))
    for i, (lo, hi) in enumerate(cache.bands):
        kk[i::2 * len(cache.bands), :, lo:hi] = 0
        vv[i::len(cache.bands) + 1, :, lo:hi] = 0
    lo, hi = cache.bands[-1]
    kk[:, :, lo:hi] = 0
    kk[17] = vv[18] = 0
    k, v = append(cache, table, kk, vv)
    check(torch.randn(q, 4, 128).bfloat16().cuda(), cache, batch, k, v, scale=0.09 / size)
