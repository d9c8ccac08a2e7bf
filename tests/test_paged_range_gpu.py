"""Paged cache on the GPU where fp16 operands are short of range (channel groups of different
magnitude inside a token, small weights, values and scales near fp32's ends), and what
test_paged_gpu.py holds loosely. Against definitions in 64 bits, with its tolerances where no
other is derived: they hold every K and V value to fp16's relative rounding."""
import numpy as np
import pytest
import torch

from kvq import paged
from oracle import c_oracle
from test_paged_gpu import FORMATS, check, fill, make, rows_of, stored, u16

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


@pytest.mark.parametrize("q", [1, 70])
@pytest.mark.parametrize("k_bits,v_bits", [(4, 4), (8, 8)])
@pytest.mark.parametrize("n,lead", [(200, 5.0), (200, 13.0), (200, 16.5), (200, 17.2), (131072, 16.5), (131072, 17.2)])
def test_weights_under_one_dominating_token(q, k_bits, v_bits, n, lead):
    """The first token leads by `lead` nats and has the value zero: the output is the sum of the
    others' small weights. 200 tokens in one part, 131072 in many.

    Bound per element: the output's rounding (2^-8), and of each weight either fp16's relative
    rounding (2^-11) or, below its normal range, 2^-32 of the row's largest (fp16 ends at 2^-24,
    and the largest is stored as 2^7 at least), a value's rounding (2^-11) and a logit's by
    those of the keys (twice d)."""
    cache, batch, table = make([n], [q], heads=1, page=128, k_bits=k_bits, v_bits=v_bits, mode="blind64", garbage=False)
    kk = torch.randn(n, 1, 128) * 0.03
    vv = 1 + 0.3 * torch.randn(n, 1, 128)
    kk[:, 0, 0] = 0
    kk[0] = vv[0] = 0
    kk[0, 0, 0] = lead
    x = torch.randn(q, 1, 128)
    x[:, :, 0] = 1
    x = x.bfloat16()
    k, v = append(cache, table, kk.bfloat16(), vv.bfloat16())
    out, lse = paged.attention(x.cuda(), cache, batch, causal=False, softmax_scale=1.0, return_lse=True)
    k, v, xd = k[:, 0], v[:, 0], x[:, 0].double()
    logits = xd @ k.T
    w = torch.softmax(logits, 1)
    ref = w @ v
    d = (2.0 ** -11 * (xd.abs() @ k.abs().T)).amax(1, keepdim=True)
    most = w.amax(1, keepdim=True)
    bound = 2.0 ** -8 * ref.abs() + (2 * 2.0 ** -11 + 2 * d + 2e-5) * (w @ v.abs()) + 2.0 ** -32 * most * v.abs().sum(0)
    assert ((out[:, 0].double().cpu() - ref).abs() <= bound).all()
    assert ((lse[:, 0].double().cpu() - torch.logsumexp(logits, 1)).abs() <= d[:, 0] + 2e-5).all()


def test_slots_that_were_never_written_cost_nothing():
    """A decode step over pages as append leaves them, zeros past the sequence's end, takes
    as long as one over pages that were full: rows past the end do not send a step through the
    exact conversion. One attempt of five has to show it (2.1 times as long otherwise)."""
    n, heads = 1561, 8
    table = np.arange(100)[None]
    caches = [paged.PagedKVCache(100, 16, heads, group_mode="blind32", device="cuda:0") for _ in range(2)]
    k = rows_of(n, heads, 1).cuda()
    for cache, m in zip(caches, (n, 1600)):
        full = torch.cat((k, k))[:m]
        cache.append(full, full, paged.PagedBatch(table, [m], [m], 16, device="cuda:0"))
    x = torch.randn(1, 4 * heads, 128).bfloat16().cuda()
    batch = paged.PagedBatch(table, [n], [1], 16, device="cuda:0")
    assert torch.equal(*(paged.attention(x, cache, batch) for cache in caches))
    graphs = []
    for cache in caches:
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            for _ in range(50):
                paged.attention(x, cache, batch)
        graphs.append(g)

    def fastest():
        times = [[], []]
        for _ in range(8):
            for g, t in zip(graphs, times):
                a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
                g.replay()
                a.record()
                g.replay()
                b.record()
                b.synchronize()
                t.append(a.elapsed_time(b))
        return [min(t) for t in times]

    ratios = [t[0] / t[1] for t in (fastest() for _ in range(5))]
    assert min(ratios) < 1.07, ratios


@pytest.mark.parametrize("q", [1, 12, 150])
@pytest.mark.parametrize("scale,size", [(1e-20, 1e-30), (1e-38, 1e-25), (1e-38, 1.0), (1e-30, 1e-6)])
def test_tiny_scale_and_queries(q, scale, size):
    """Logits of no size: the mean of the values that a row sees, where the product of the
    softmax scale and the power of two taken out of a query is below fp32's range too."""
    n = 217
    cache, batch, table = make([n], [q], heads=2, page=32)
    k, v = append(cache, table, rows_of(n, 2, 3), rows_of(n, 2, 4))
    x = (torch.randn(q, 4, 128) * size).bfloat16()
    check(x.cuda(), cache, batch, k, v, scale=scale)
    check(x.cuda(), cache, batch, k, v, scale=scale, window=50, sink=7)


@pytest.mark.parametrize("q", [1, 12, 40, 150])
@pytest.mark.parametrize("k_bits,v_bits,mode", [(4, 4, "blind32"), (8, 8, "bands4")])
@pytest.mark.parametrize("n", [217, 9000])
def test_values_near_the_end_of_fp32(q, k_bits, v_bits, mode, n):
    """The mean of values is in range where their sum is not."""
    cache, batch, table = make([n], [q], heads=2, page=32, k_bits=k_bits, v_bits=v_bits, mode=mode)
    kk, vv = rows_of(n, 2, 3), (1e38 * (1 + 0.2 * torch.randn(n, 2, 128))).bfloat16()
    vv[5::7] *= 1e-30
    k, v = append(cache, table, kk, vv)
    x = torch.randn(q, 4, 128).bfloat16()
    check(x.cuda(), cache, batch, k, v)
    check(x.cuda(), cache, batch, k, v, window=150, sink=20)
    # an infinity is stored as 3e38: rows that see it are finite
    vv = rows_of(n, 2, 4)
    vv[n - 3 * q // 4 - 1, 1, 77] = float("inf")
    cache.append(kk.cuda(), vv.cuda(), paged.PagedBatch(table, [n], [n], 32, device="cuda:0"))
    out = paged.attention(x.cuda(), cache, batch).float()
    assert torch.isfinite(out).all() and out[-1, 2:, 77].min() > 1e30


@pytest.mark.parametrize("q", [1, 12, 40, 150])
@pytest.mark.parametrize("k_bits,v_bits,mode", [(4, 4, "blind32"), (8, 8, "bands4")])
@pytest.mark.parametrize("n", [600, 5000])
@pytest.mark.parametrize("size,other", [(1e-20, 1.0), (1e-30, 1e-9), (1.0, 1e18)])
def test_small_values_behind_large_ones_of_no_weight(q, k_bits, v_bits, mode, n, size, other):
    """The first half's values are 1e18 to 1e21 times as large as the second half's, and their
    weights 1e-26 times: the row's power of two follows the maximum down.

    Bound per element: roundings as above, of each weight; below fp16's normal range 2^-32 of
    the largest product of a weight and its value."""
    cache, batch, table = make([n], [q], heads=1, page=32, k_bits=k_bits, v_bits=v_bits, mode=mode)
    kk, vv = 0.03 * torch.randn(n, 1, 128), 1 + 0.2 * torch.randn(n, 1, 128)
    kk[:, 0, 0] = 0
    kk[n // 2:, 0, 0] = 60
    vv[: n // 2] *= other
    vv[n // 2:] *= size
    x = torch.randn(q, 4, 128)
    x[:, :, 0] = 1
    k, v = append(cache, table, kk.bfloat16(), vv.bfloat16())
    out = paged.attention(x.bfloat16().cuda(), cache, batch, causal=False, softmax_scale=1.0)[:, 0].double().cpu()
    k, v, xd = k[:, 0], v[:, 0], x[:, 0].bfloat16().double()
    w = torch.softmax(xd @ k.T, 1)
    ref = w @ v
    d = (2.0 ** -11 * (xd.abs() @ k.abs().T)).amax(1, keepdim=True)
    most = (w * v.abs().amax(1)).amax(1, keepdim=True)
    bound = 2.0 ** -8 * ref.abs() + (2 * 2.0 ** -11 + 2 * d + 2e-5) * (w @ v.abs()) + 2.0 ** -32 * n * most
    assert ((out - ref).abs() <= bound).all()


@pytest.mark.parametrize("q", [1, 12, 40, 150])
@pytest.mark.parametrize("k_bits,v_bits", FORMATS)
@pytest.mark.parametrize("mode", ["bands", "blind32"])
@pytest.mark.parametrize("ratio", [1e3, 2.0 ** 15, 1e6])
@pytest.mark.parametrize("size", [1.0, 2e-3, 1e-9])
def test_queries_with_groups_of_different_magnitude(q, k_bits, v_bits, mode, ratio, size):
    """Queries that are small in the channels where keys are large: each group has its share of
    the logits."""
    n = 217
    cache, batch, table = make([n], [q], heads=2, page=32, k_bits=k_bits, v_bits=v_bits, mode=mode)
    large = torch.ones(128)
    for lo, hi in cache.bands[1::2]:
        large[lo:hi] = ratio
    k, v = append(cache, table, (rows_of(n, 2, 3).float() * large).bfloat16(), rows_of(n, 2, 4))
    x = (torch.randn(q, 4, 128) / large * size).bfloat16()
    check(x.cuda(), cache, batch, k, v, scale=0.09 / size)


@pytest.mark.parametrize("q", [1, 150])
def test_windows_longer_than_any_sequence(q):
    """Whole numbers of any size are windows and sinks."""
    cache, batch, table = make([200], [q], heads=1)
    append(cache, table, rows_of(200, 1, 3), rows_of(200, 1, 4))
    x = torch.randn(q, 2, 128).bfloat16().cuda()
    want = paged.attention(x, cache, batch)
    for window, sink in ((2 ** 31, 0), (2 ** 63 - 1, 2 ** 63 - 1), (2 ** 63, 0), (2 ** 64 + 5, 2 ** 64), (9, 2 ** 64 + 3)):
        assert torch.equal(paged.attention(x, cache, batch, window=window, sink=sink), want), (window, sink)


@pytest.mark.parametrize("q", [1, 12, 150])
@pytest.mark.parametrize("most", [1e4, 1e6, 3e7, 1e8])
def test_logits_up_to_1e8(q, most):
    """One token of a row leads by 20 nats and by far more than logits' spacing in fp32: its value,
    and 300 e^-20 of others at most."""
    n = 300
    cache, batch, table = make([n], [q], heads=1, page=32)
    k, v = append(cache, table, rows_of(n, 1, 3), rows_of(n, 1, 4))
    x = torch.randn(q, 2, 128).bfloat16()
    logits = (x.double().flatten(0, 1) @ k[:, 0].T)
    scale = most / float(logits.abs().max())
    first, second = (logits * scale).topk(2, -1).values.T
    out = paged.attention(x.cuda(), cache, batch, causal=False, softmax_scale=scale).double().cpu().flatten(0, 1)
    assert torch.isfinite(out).all()
    clear = first - second > max(20.0, 100 * most * 2.0 ** -23)
    assert clear.float().mean() > 0.8
    want = v[logits.argmax(-1), 0]
    assert ((out - want).abs() <= 2.0 ** -8 * want.abs() + n * 2.1e-9 * 2 * v.abs().max())[clear].all()


@pytest.mark.parametrize("q", [1, 12, 150])
@pytest.mark.parametrize("k_bits,v_bits,mode", [(4, 4, "blind32"), (8, 4, "bands4"), (8, 8, "bands2")])
def test_log_sum_exp(q, k_bits, v_bits, mode):
    """To the error that the keys' roundings allow (d per logit; none for int4) and fp32's."""
    kv = [700, 9001]
    cache, batch, table = make(kv, [q, q], heads=2, page=32, k_bits=k_bits, v_bits=v_bits, mode=mode)
    k, v = fill(cache, table, kv)
    x = torch.randn(2 * q, 4, 128).bfloat16()
    for window, sink in ((0, 0), (200, 30)):
        _, lse = paged.attention(x.cuda(), cache, batch, window=window, sink=sink, return_lse=True)
        first = token = 0
        for n in kv:
            p, j = torch.arange(n - q, n)[:, None], torch.arange(n)[None]
            see = (j <= p) & ((j > p - window) | (j < sink)) if window else j <= p
            for h in range(4):
                xh, kh = x[first:first + q, h].double(), k[token:token + n, h // 2]
                want = torch.logsumexp((xh @ kh.T / 128 ** 0.5).masked_fill(~see, -np.inf), 1)
                mass = xh.abs() @ kh.abs().T / 128 ** 0.5
                d = (2.0 ** -11 * (k_bits == 8) + 2.0 ** -22) * mass.masked_fill(~see, 0).amax(1)
                err = (lse[first:first + q, h].double().cpu() - want).abs()
                assert (err <= d + 1e-5).all(), float((err - d).max())
            first, token = first + q, token + n


@pytest.mark.parametrize("heads", [7, 9, 12, 16, 17, 40])
@pytest.mark.parametrize("k_bits,v_bits", FORMATS)
def test_append_and_read_of_more_heads_than_a_tile(heads, k_bits, v_bits):
    kv, q = [50, 33], [19, 33]
    cache, batch, table = make(kv, q, heads=heads, page=16, k_bits=k_bits, v_bits=v_bits, mode="bands4")
    k, v = rows_of(52, heads, 1), rows_of(52, heads, 2)
    cache.append(k.cuda(), v.cuda(), batch)
    rk, rv = cache.read(batch, new_only=True)
    assert torch.equal(rk.cpu(), stored(k, k_bits, cache.bands).bfloat16())
    assert torch.equal(rv.cpu(), stored(v, v_bits, cache.bands).bfloat16())


@pytest.mark.parametrize("mode", ["bands", "blind64"])
def test_append_extreme_rows_int8(mode):
    """All-zero, tiny and huge rows as the oracle stores them; non-finite ones finite."""
    cache, batch, table = make([8], [8], heads=1, k_bits=8, v_bits=8, mode=mode)
    x = torch.randn(8, 1, 128).bfloat16()
    x[0] = 0
    x[1] *= 1e-38
    x[2] *= 2.0 ** -120
    x[3] *= 1e37
    cache.append(x.cuda(), x.cuda(), batch)
    rc, rs = c_oracle.quantize(u16(x), cache.bands, 8)
    at = (int(table[0, 0]), 0, 0, slice(0, 8))
    for codes, scales in ((cache.k_codes, cache.k_scales), (cache.v_codes, cache.v_scales)):
        assert np.array_equal(codes[at].cpu().numpy(), rc[:, 0]) and np.array_equal(u16(scales[at]), rs[:, 0])
    x[4, 0, 3], x[5, 0, 50], x[6, 0, 127], x[7] = np.nan, np.inf, -np.inf, np.nan
    cache.append(x.cuda(), x.cuda(), batch)
    k, v = (t.float().cpu()[:, 0] for t in cache.read(batch))
    assert torch.isfinite(k).all() and torch.equal(k, v)
    assert k[4, 3] == 0 and (k[7] == 0).all() and k[5, 50] > 2.9e38 and k[6, 127] < -2.9e38


@pytest.mark.parametrize("q", [1, 12, 150])
@pytest.mark.parametrize("k_bits,v_bits", FORMATS)
@pytest.mark.parametrize("ks,qs", [(1e34, 1e-30), (1e36, 1.0), (1e-35, 1e30), (1e-30, 1e34)])
def test_huge_keys_and_tiny_queries(q, k_bits, v_bits, ks, qs):
    """Products in range of factors near both ends of it."""
    n = 217
    cache, batch, table = make([n], [q], heads=2, page=32, k_bits=k_bits, v_bits=v_bits, mode="bands")
    k, v = append(cache, table, rows_of(n, 2, 3, ks), rows_of(n, 2, 4))
    x = (torch.randn(q, 4, 128) * qs).bfloat16()
    check(x.cuda(), cache, batch, k, v, scale=max(0.09 / (ks * qs), 2e-38))


@pytest.mark.parametrize("q", [1, 70])
@pytest.mark.parametrize("k_bits,v_bits", [(4, 4), (8, 8)])
@pytest.mark.parametrize("size", [1.0, 1e-3, 1e-4, 1e-5, 3e-6, 1e-6])
def test_small_weights_of_small_values(q, k_bits, v_bits, size):
    """As under a dominating token (17 nats), whose value lies in the other channels, with
    values of any size: their power of two leaves the weights as much room as there is."""
    n = 200
    cache, batch, table = make([n], [q], heads=1, page=128, k_bits=k_bits, v_bits=v_bits, mode="blind64", garbage=False)
    kk = torch.randn(n, 1, 128) * 0.03
    vv = (1 + 0.3 * torch.randn(n, 1, 128)) * size
    kk[:, 0, 0] = 0
    kk[0] = 0
    kk[0, 0, 0] = 17.0
    vv[0, :, 64:] = 0
    vv[1:, :, :64] = 0
    x = torch.randn(q, 1, 128)
    x[:, :, 0] = 1
    x = x.bfloat16()
    k, v = append(cache, table, kk.bfloat16(), vv.bfloat16())
    out = paged.attention(x.cuda(), cache, batch, causal=False, softmax_scale=1.0)
    k, v, xd = k[:, 0], v[:, 0], x[:, 0].double()
    w = torch.softmax(xd @ k.T, 1)
    ref = w @ v
    d = (2.0 ** -11 * (xd.abs() @ k.abs().T)).amax(1, keepdim=True)
    bound = 2.0 ** -8 * ref.abs() + (2 * 2.0 ** -11 + 2 * d + 2e-5) * (w @ v.abs())
    bound += 2.0 ** -32 * w.amax(1, keepdim=True) * v.abs().sum(0)
    assert ((out[:, 0].double().cpu() - ref).abs() <= bound).all()


@pytest.mark.parametrize("q", [1, 12, 150])
@pytest.mark.parametrize("bits", [1, 2, 0x7F, 0x80])
def test_queries_of_the_smallest_numbers(q, bits):
    """Zeros beside bf16's smallest magnitudes, in every second channel, in both orders: logits of
    no size."""
    n = 217
    cache, batch, table = make([n], [q], heads=2, page=32)
    k, v = append(cache, table, rows_of(n, 2, 3), rows_of(n, 2, 4))
    for first in (0, 1):
        x = torch.zeros(q, 4, 128, dtype=torch.int16)
        x[..., first::2] = bits
        x[:, 1, :64] = 0
        x[:, 2, 8:] = 0
        check(x.view(torch.bfloat16).cuda(), cache, batch, k, v)
