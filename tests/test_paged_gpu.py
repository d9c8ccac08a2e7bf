"""Paged quantized cache (kvq.paged) on the GPU against plain forms: append bit-exact to
the storage oracle, read exact, attention against its definition in 64 bits.

Tolerances of the attention, derived from its roundings: the output to bf16 (relative
U = 2^-8, half a step at the bottom of a binade), each K and V value and each softmax weight to
fp16 (u = 2^-11; a weight below fp16's normal range, of which the largest is at least 1,
absolutely 2^-25). A K rounding moves a logit by at most d = scale * u * sum_c |q_c K_c|, a
weight by a factor exp(+-2 d). So per output element, with L = sum_j exp(x_j - max x)
  |err| <= U |o| + (2 u + 2 d_max + 2e-5) * sum_j w_j |V_j| + 2^-25 sum_j |V_j| / L
(2e-5: fp32 sums and exp) always. As the roundings are independent, with a standard
deviation of at most a bound / sqrt(3) each, the error's expected square is, per element,
  U^2/3 o^2 + u^2/3 sum_j w_j^2 (2 V_j^2 + (V_j - o)^2 scale^2 sum_c (q_c K_jc)^2)
and the 2-norm of a case's error is held to three times the root of their sum (and the
absolute parts above): a case has at least 128 elements, but one row's weights are shared by
them and may rest on a few tokens. A single wrongly seen or missed token exceeds that at every
length used here.
"""
import numpy as np
import pytest
import torch

from kvq import paged
from oracle import c_oracle
from quant_kv import _band_edges

pytestmark = pytest.mark.gpu

U, UH = 2.0 ** -8, 2.0 ** -11
FORMATS = [(4, 4), (8, 4), (8, 8)]
MODES = ["bands", "bands2", "bands4", "blind32", "blind64"]


@pytest.fixture(autouse=True)
def _seed():
    torch.manual_seed(1234)


def u16(t):
    return t.detach().cpu().contiguous().view(torch.int16).numpy().view(np.uint16)


def make(kv, q, heads=2, page=16, k_bits=4, v_bits=4, mode="blind32", seed=0, spare=3, garbage=True):
    """A cache whose pages hold garbage, and a batch with its pages in random order."""
    rng = np.random.default_rng(seed)
    kv, q = np.asarray(kv), np.asarray(q)
    pages = -(-kv // page)
    n = int(pages.sum()) + spare
    ids = rng.permutation(n)
    table = np.full((len(kv), int(pages.max()) + 1 if len(kv) else 1), -7)
    at = 0
    for b, m in enumerate(pages):
        table[b, :m] = ids[at:at + m]
        at += m
    cache = paged.PagedKVCache(n, page, heads, k_bits=k_bits, v_bits=v_bits, group_mode=mode, device="cuda:0")
    if garbage:
        g = torch.Generator(device="cuda").manual_seed(seed)
        for p in (cache.k_pages, cache.v_pages):
            p.copy_(torch.randint(0, 256, p.shape, dtype=torch.uint8, device="cuda", generator=g))
    return cache, paged.PagedBatch(table, kv, q, page, device="cuda:0"), table


def rows_of(n, heads, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    chan = torch.exp(0.5 * torch.randn(heads, 128, generator=g))
    return (torch.randn(n, heads, 128, generator=g) * chan * scale).bfloat16()


def fill(cache, table, kv, seed=5):
    """Writes every sequence whole; returns the stored values in 64 bits, per sequence."""
    kv = np.asarray(kv)
    b = paged.PagedBatch(table, kv, kv, cache.page_size, device="cuda:0")
    k, v = (rows_of(int(kv.sum()), cache.n_heads, seed + i) for i in (0, 1))
    cache.append(k.cuda(), v.cuda(), b)
    return [stored(x, bits, cache.bands) for x, bits in ((k, cache.k_bits), (v, cache.v_bits))]


def stored(x, bits, bands):
    """The values code * bf16 scale of quantized rows x, fp64, from the C oracle's codes."""
    codes, scales = c_oracle.quantize(u16(x), bands, bits)
    if bits == 4:
        q = np.stack((codes & 15, codes >> 4), -1).reshape(x.shape).astype(np.float64) - 8
    else:
        q = codes.reshape(x.shape).astype(np.float64) - 128
    s = torch.from_numpy(scales.view(np.int16)).view(torch.bfloat16).double().numpy()
    for g, (lo, hi) in enumerate(bands):
        q[..., lo:hi] *= s[..., g:g + 1]
    return torch.from_numpy(q)


def reference(q, k, v, kv, ql, heads, causal, window, sink, scale=None):
    """(out, lse, worst-case bound, expected square of the error) in 64 bits; k, v: all sequences'
    stored values in a row."""
    q = q.double().cpu()
    group = q.shape[1] // heads
    scale = 1 / np.sqrt(128) if scale is None else scale
    out, lse, bound = torch.zeros_like(q), torch.full(q.shape[:2], -np.inf).double(), torch.zeros_like(q)
    var = torch.zeros_like(q)
    f, t = 0, 0
    for n, m in zip(kv, ql):
        kb, vb = k[t:t + n], v[t:t + n]
        pos = torch.arange(n - m, n)[:, None]
        j = torch.arange(n)[None]
        see = torch.ones((m, n), dtype=torch.bool)
        if causal:
            see &= j <= pos
        if window:
            see &= (j > pos - window) | (j < sink)
        for h in range(q.shape[1]):
            x = (q[f:f + m, h] @ kb[:, h // group].T) * scale
            d = scale * UH * (q[f:f + m, h].abs() @ kb[:, h // group].abs().T)
            x = x.masked_fill(~see, -np.inf)
            some = see.any(1)
            w = torch.where(some[:, None], torch.softmax(x, 1), torch.zeros(()).double())
            out[f:f + m, h] = w @ vb[:, h // group]
            lse[f:f + m, h] = torch.where(some, torch.logsumexp(x, 1), torch.tensor(-np.inf).double())
            dm = torch.where(see, d, torch.zeros(()).double()).amax(1, keepdim=True) if n else torch.zeros(m, 1)
            rel = torch.where(see, torch.exp(x - x.amax(1, keepdim=True)), torch.zeros(()).double()) if n else x
            small = 2.0 ** -25 * (see.double() @ vb[:, h // group].abs()) / rel.sum(1, keepdim=True).clamp(min=1)
            floor = 2e-5 * (w @ vb[:, h // group].abs()) + small
            bound[f:f + m, h] = U * out[f:f + m, h].abs() + (2 * UH + 2 * dm) * (w @ vb[:, h // group].abs()) + floor
            vh, oh, w2 = vb[:, h // group], out[f:f + m, h], w * w
            ws = w2 * scale * scale * (q[f:f + m, h].square() @ kb[:, h // group].square().T)
            var[f:f + m, h] = U * U / 3 * oh.square() + floor.square() + UH * UH / 3 * (
                2 * (w2 @ vh.square()) + ws @ vh.square() - 2 * oh * (ws @ vh) + oh.square() * ws.sum(1, keepdim=True))
        f, t = f + m, t + n
    return out, lse, bound, var


def check(q, cache, batch, k, v, causal=True, window=0, sink=0, scale=None):
    out, lse = paged.attention(q, cache, batch, causal=causal, window=window, sink=sink, softmax_scale=scale,
                               return_lse=True)
    ref, ref_lse, bound, var = reference(q, k, v, batch.kv_lens.tolist(), batch.q_lens.tolist(), cache.n_heads, causal,
                                    window, sink, scale)
    out, lse = out.double().cpu(), lse.double().cpu()
    assert torch.isfinite(out).all()
    assert ((out - ref).abs() <= bound + 1e-30).all(), float(((out - ref).abs() - bound).max())
    assert (out - ref).norm() <= 3 * var.sum().sqrt() + 1e-30
    none = torch.isinf(ref_lse)
    assert torch.equal(none, torch.isinf(lse)) and (lse[none] < 0).all()
    # |lse error| <= max logit error (bounded through `bound`'s d) + fp32
    assert (lse[~none] - ref_lse[~none]).abs().max() < 0.05 if (~none).any() else True
    assert (out[none] == 0).all()
    return out


# ---------------------------------------------------------------- append and read
@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("k_bits,v_bits", FORMATS)
def test_append_is_the_storage_oracle_and_read_is_exact(mode, k_bits, v_bits):
    kv, q = [37, 16, 5, 120, 1], [37, 3, 0, 55, 1]
    cache, batch, table = make(kv, q, heads=3, page=32, k_bits=k_bits, v_bits=v_bits, mode=mode)
    before = cache.k_pages.clone(), cache.v_pages.clone()
    k, v = rows_of(96, 3, 1), rows_of(96, 3, 2)
    cache.append(k.cuda(), v.cuda(), batch)
    touched = [torch.zeros_like(c, dtype=torch.bool) for c in (cache.k_codes[..., 0], cache.v_codes[..., 0])]
    for x, bits, codes, scales, seen in ((k, k_bits, cache.k_codes, cache.k_scales, touched[0]),
                                         (v, v_bits, cache.v_codes, cache.v_scales, touched[1])):
        rc, rs = c_oracle.quantize(u16(x), cache.bands, bits)
        i = 0
        for b in range(len(kv)):
            for p in range(kv[b] - q[b], kv[b]):
                at = (table[b, p // 32], slice(None), p % 32 // 16, p % 16)
                assert np.array_equal(codes[at].cpu().numpy(), rc[i]) and np.array_equal(u16(scales[at]), rs[i])
                seen[at] = True
                i += 1
    # nothing else was written
    for pages, old, seen, codes in ((cache.k_pages, before[0], touched[0], cache._codes(before[0], k_bits)),
                                    (cache.v_pages, before[1], touched[1], cache._codes(before[1], v_bits))):
        now = cache._codes(pages, k_bits if pages is cache.k_pages else v_bits)
        assert torch.equal(now[~seen], codes[~seen])
    rk, rv = cache.read(batch, new_only=True)
    assert torch.equal(rk.double().cpu(), stored(k, k_bits, cache.bands).bfloat16().double())
    assert torch.equal(rv.double().cpu(), stored(v, v_bits, cache.bands).bfloat16().double())


@pytest.mark.parametrize("page", paged.PAGE_SIZES)
@pytest.mark.parametrize("kv", [[1], [0, 17, 0], [16], [128, 129, 127], [1561, 4, 33]])
def test_read_whole_sequences(page, kv):
    cache, batch, table = make(kv, [min(1, n) for n in kv], heads=5, page=page, k_bits=8, mode="bands4")
    k, v = fill(cache, table, kv)
    rk, rv = cache.read(batch)
    assert torch.equal(rk.cpu(), k.bfloat16()) and torch.equal(rv.cpu(), v.bfloat16())


def test_append_strides_and_order():
    """Rows of a fused projection (a token stride larger than the row) and transposed heads."""
    kv = [33, 7]
    cache, batch, table = make(kv, kv, heads=4)
    x = torch.randn(40, 3, 4, 128).bfloat16().cuda()
    cache.append(x[:, 1], x[:, 2], batch)
    k, v = cache.read(batch)
    assert torch.equal(k.cpu(), stored(x[:, 1].cpu(), 4, cache.bands).bfloat16())
    y = torch.randn(4, 40, 128).bfloat16().cuda()
    cache.append(y.transpose(0, 1), x[:, 0], batch)
    k, v = cache.read(batch)
    assert torch.equal(k.cpu(), stored(y.transpose(0, 1).contiguous().cpu(), 4, cache.bands).bfloat16())
    assert torch.equal(v.cpu(), stored(x[:, 0].contiguous().cpu(), 4, cache.bands).bfloat16())


def test_append_extreme_rows():
    """All-zero, tiny, huge and non-finite rows: what the oracle stores where it is defined,
    finite values elsewhere."""
    cache, batch, table = make([8], [8], heads=1, mode="bands4")
    x = torch.randn(8, 1, 128).bfloat16()
    x[0] = 0
    x[1] *= 1e-38
    x[2] *= 2.0 ** -120
    x[3] *= 1e37
    cache.append(x.cuda(), x.cuda(), batch)
    rc, rs = c_oracle.quantize(u16(x), cache.bands, 4)
    at = (int(table[0, 0]), 0, 0, slice(0, 8))
    assert np.array_equal(cache.k_codes[at].cpu().numpy(), rc[:, 0]) and np.array_equal(u16(cache.k_scales[at]), rs[:, 0])
    x[4, 0, 3], x[5, 0, 50], x[6, 0, 127], x[7] = np.nan, np.inf, -np.inf, np.nan
    cache.append(x.cuda(), x.cuda(), batch)
    k, v = (t.float().cpu()[:, 0] for t in cache.read(batch))
    assert torch.isfinite(k).all() and torch.equal(k, v)
    assert k[4, 3] == 0 and (k[7] == 0).all() and k[5, 50] > 2.9e38 and k[6, 127] < -2.9e38
    good = torch.ones(128, dtype=torch.bool)
    good[0:12] = False  # the group of the NaN
    ref = stored(x.nan_to_num(0.0, 0.0, 0.0), 4, cache.bands).bfloat16().float()[:, 0]
    assert torch.equal(k[4], ref[4])  # NaN counts as 0
    assert torch.equal(k[5][68:], ref[5][68:]) and torch.equal(k[6][:110], ref[6][:110])  # other groups untouched


# ---------------------------------------------------------------- attention
@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("k_bits,v_bits", FORMATS)
@pytest.mark.parametrize("q", [1, 3, 70])
def test_formats(mode, k_bits, v_bits, q):
    kv = [200, 70, 131]
    cache, batch, table = make(kv, [q, q, q], heads=2, page=16, k_bits=k_bits, v_bits=v_bits, mode=mode)
    k, v = fill(cache, table, kv)
    check(torch.randn(3 * q, 8, 128).bfloat16().cuda(), cache, batch, k, v)


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 257, 1000])
@pytest.mark.parametrize("q", [1, 9, 1000])
@pytest.mark.parametrize("causal", [True, False])
def test_lengths(n, q, causal):
    q = min(q, n)
    cache, batch, table = make([n], [q], heads=1, page=32)
    k, v = fill(cache, table, [n])
    check(torch.randn(q, 2, 128).bfloat16().cuda(), cache, batch, k, v, causal=causal)


@pytest.mark.parametrize("group", [1, 2, 3, 5, 7, 8, 16, 33])
@pytest.mark.parametrize("q", [1, 2, 41])
def test_grouped_heads(group, q):
    kv = [150, 41, 300]
    cache, batch, table = make(kv, [q] * 3, heads=2, page=64, mode="bands4")
    k, v = fill(cache, table, kv)
    check(torch.randn(3 * q, 2 * group, 128).bfloat16().cuda(), cache, batch, k, v)


@pytest.mark.parametrize("page", paged.PAGE_SIZES)
@pytest.mark.parametrize("window,sink", [(1, 0), (16, 0), (50, 7), (64, 64), (100, 130), (400, 16), (1, 1), (5000, 9)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("q", [1, 5, 260])
def test_window_and_sink(page, window, sink, causal, q):
    kv = [520, 333, 260]
    cache, batch, table = make(kv, [q] * 3, heads=1, page=page, mode="bands")
    k, v = fill(cache, table, kv)
    check(torch.randn(3 * q, 3, 128).bfloat16().cuda(), cache, batch, k, v, causal=causal, window=window, sink=sink)


@pytest.mark.parametrize("causal", [True, False])
def test_rows_that_see_nothing_and_empty_sequences(causal):
    kv, q = [0, 5, 0, 40, 3], [0, 9, 4, 300, 1]
    cache, batch, table = make(kv, q, heads=2)
    k, v = fill(cache, table, kv)
    check(torch.randn(sum(q), 4, 128).bfloat16().cuda(), cache, batch, k, v, causal=causal)
    check(torch.randn(sum(q), 4, 128).bfloat16().cuda(), cache, batch, k, v, causal=causal, window=3)


def test_ragged_mix():
    """Chunks, single tokens and idle sequences in one step."""
    kv, q = [900, 1, 257, 1300, 64, 2000], [300, 1, 1, 129, 0, 1]
    cache, batch, table = make(kv, q, heads=2, page=16, mode="bands4", k_bits=8)
    k, v = fill(cache, table, kv)
    x = torch.randn(sum(q), 8, 128).bfloat16().cuda()
    check(x, cache, batch, k, v)
    check(x, cache, batch, k, v, window=200, sink=33)


@pytest.mark.parametrize("n,q,heads,group", [(20000, 1, 1, 1), (9001, 4, 2, 4), (5000, 130, 1, 2)])
def test_long_context_is_split_and_joined(n, q, heads, group):
    cache, batch, table = make([n], [q], heads=heads, page=64, mode="blind64", k_bits=8, v_bits=8)
    k, v = fill(cache, table, [n])
    a = check(torch.randn(q, heads * group, 128, generator=torch.Generator().manual_seed(1)).bfloat16().cuda(), cache,
              batch, k, v)
    b = check(torch.randn(q, heads * group, 128, generator=torch.Generator().manual_seed(1)).bfloat16().cuda(), cache,
              batch, k, v)
    assert torch.equal(a, b)  # joined in a fixed order


@pytest.mark.parametrize("q", [1, 200])
def test_large_logits_and_scale(q):
    """One token holds nearly all the weight, at the start, the end and in the middle; and a
    softmax_scale of its own."""
    n = 300
    cache, batch, table = make([n], [q], heads=1)
    k, v = fill(cache, table, [n])
    x = torch.randn(q, 1, 128).bfloat16()
    for j in (0, n - q, 77):
        y = (k[j, 0] * 3).bfloat16().expand(q, 1, 128).contiguous()
        out = paged.attention(y.cuda(), cache, batch, causal=False).double().cpu()
        ref, _, bound, _ = reference(y, k, v, [n], [q], 1, False, 0, 0)
        assert ((out - ref).abs() <= bound).all()
    check(x.cuda(), cache, batch, k, v, scale=0.031)
    check(x.cuda(), cache, batch, k, v, scale=1e-6)


@pytest.mark.parametrize("q", [1, 150])
def test_unseen_tokens_have_no_effect(q):
    """Whatever lies in masked places and in pages past the end (non-finite scales among it)."""
    n = 217
    cache, batch, table = make([n], [q], heads=2, page=64)
    k, v = fill(cache, table, [n])
    x = torch.randn(q, 4, 128).bfloat16().cuda()
    a = paged.attention(x, cache, batch)
    for s in (cache.k_scales, cache.v_scales):
        s[int(table[0, 3]), :, 1, 9:] = float("nan")  # positions 217.. of the last page
        s[int(table[0, 3]), :, 2:] = float("inf")
        used = torch.zeros(cache.n_pages, dtype=torch.bool)
        used[torch.from_numpy(table[0, :4])] = True
        s[~used] = float("nan")
    assert torch.equal(paged.attention(x, cache, batch), a)
    # new tokens with infinities: earlier queries do not see them
    if q > 1:
        nk, nv = (rows_of(q, 2, 70 + i) for i in (0, 1))
        cache.append(nk.cuda(), nv.cuda(), batch)
        a = paged.attention(x, cache, batch)
        nk[100:, :, 5], nv[100:, :, 6] = float("inf"), float("nan")
        cache.append(nk.cuda(), nv.cuda(), batch)
        assert torch.equal(paged.attention(x, cache, batch)[:100], a[:100])


def test_non_finite_queries_stay_in_their_rows():
    cache, batch, table = make([100, 64], [30, 30], heads=1)
    k, v = fill(cache, table, [100, 64])
    x = torch.randn(60, 4, 128).bfloat16().cuda()
    a = paged.attention(x, cache, batch)
    x[17, 2] = float("nan")
    x[44, 0, 0] = float("inf")
    b = paged.attention(x, cache, batch)
    same = torch.ones(60, 4, dtype=torch.bool)
    same[17, 2] = same[44, 0] = False
    assert torch.equal(a[same], b[same]) and torch.isnan(b[17, 2]).all()


def test_strided_q_and_out():
    kv, q = [90, 200], [20, 1]
    cache, batch, table = make(kv, q, heads=2)
    fill(cache, table, kv)
    big = torch.randn(21, 3, 4, 128).bfloat16().cuda()
    a = paged.attention(big[:, 1].contiguous(), cache, batch)
    assert torch.equal(paged.attention(big[:, 1], cache, batch), a)
    out = torch.full((21, 6, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    got = paged.attention(big[:, 1], cache, batch, out=out[:, :4])
    assert got.data_ptr() == out.data_ptr() and torch.equal(out[:, :4], a) and (out[:, 4:] == 7).all()


def test_shared_prefix_and_dropped_pages():
    """Two sequences over the same first pages; a sequence whose middle pages were dropped."""
    cache, batch, table = make([96, 64], [1, 1], heads=2)
    k, v = fill(cache, table, [96, 64])
    t = np.stack((table[0, :6], np.concatenate((table[0, :3], table[1, 3:4], [0, 0]))))
    b = paged.PagedBatch(t, [96, 60], [1, 1], 16, device="cuda:0")
    x = torch.randn(2, 4, 128).bfloat16().cuda()
    kk = torch.cat((k[:96], k[:48], k[96 + 48:96 + 60]))
    vv = torch.cat((v[:96], v[:48], v[96 + 48:96 + 60]))
    check(x, cache, b, kk, vv)
    shared = paged.PagedBatch(np.stack((table[0, :6], table[0, :6])), [90, 90], [1, 1], 16, device="cuda:0")
    with pytest.raises(ValueError, match="more than once"):
        cache.append(torch.zeros(2, 2, 128).bfloat16().cuda(), torch.zeros(2, 2, 128).bfloat16().cuda(), shared)


def test_offsets_past_32_bits():
    """Pages beyond 4 GB of a pool."""
    page, heads = 128, 40
    rec = 16 * (128 + 24) * 8 * heads
    n = (1 << 32) // rec + 6
    cache = paged.PagedKVCache(n, page, heads, k_bits=8, v_bits=4, group_mode="bands4", device="cuda:0")
    kv = [300, 200]
    table = np.array([[n - 1, 0, n - 3], [n - 2, 1, 0]])
    k, v = fill(cache, table, kv)
    rk, rv = cache.read(paged.PagedBatch(table, kv, [1, 1], page, device="cuda:0"))
    assert torch.equal(rk.cpu(), k.bfloat16()) and torch.equal(rv.cpu(), v.bfloat16())
    for q in (1, 150):
        b = paged.PagedBatch(table, kv, [q, q], page, device="cuda:0")
        check(torch.randn(2 * q, heads, 128).bfloat16().cuda(), cache, b, k, v)


def test_another_stream():
    kv, q = [500, 90], [40, 1]
    cache, batch, table = make(kv, q, heads=2)
    fill(cache, table, kv)
    x = torch.randn(41, 8, 128).bfloat16().cuda()
    a = paged.attention(x, cache, batch)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        got = [paged.attention(x, cache, batch) for _ in range(3)]
        fresh = paged.PagedBatch(table, kv, q, 16, device="cuda:0")
    torch.cuda.current_stream().wait_stream(st)
    got.append(paged.attention(x, cache, fresh))
    torch.cuda.synchronize()
    assert all(torch.equal(a, g) for g in got)


def test_cuda_graph():
    """append + attention of one step captured once and replayed on new inputs."""
    kv, q = [700, 33, 200], [1, 1, 1]
    cache, batch, table = make(kv, q, heads=2)
    fill(cache, table, kv)
    k, v, x = (torch.zeros(3, h, 128, dtype=torch.bfloat16, device="cuda") for h in (2, 2, 8))
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        cache.append(k, v, batch)
        paged.attention(x, cache, batch)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cache.append(k, v, batch)
        out = paged.attention(x, cache, batch)
    for seed in (1, 2):
        torch.manual_seed(seed)
        for t in (k, v, x):
            t.copy_(torch.randn(t.shape).bfloat16())
        g.replay()
        a = out.clone()
        cache.append(k, v, batch)
        assert torch.equal(paged.attention(x, cache, batch), a)


@pytest.mark.parametrize("q", [1, 12, 150])
@pytest.mark.parametrize("k_bits,v_bits,mode", [(4, 4, "blind32"), (8, 8, "bands4")])
def test_magnitudes_beyond_half_precision(q, k_bits, v_bits, mode):
    """Keys, values and queries whose magnitudes pass 65504 or are tiny, in some tokens and
    rows and not in others; logits stay moderate through softmax_scale."""
    n = 300
    cache, batch, table = make([n], [q], heads=1, page=32, k_bits=k_bits, v_bits=v_bits, mode=mode)
    whole = paged.PagedBatch(table, [n], [n], 32, device="cuda:0")
    for ks, vs, qs in ((1e6, 1.0, 1e-6), (1.0, 1e7, 1.0), (1e-5, 1e-6, 1e5), (1e12, 1e-3, 1e-12), (1e-3, 1e30, 1e6)):
        kk, vv = rows_of(n, 1, 3, ks), rows_of(n, 1, 4, vs)
        kk[::3] *= 1e-3
        vv[1::4] *= 1e-3
        x = (torch.randn(q, 4, 128) * qs).bfloat16()
        x[::2] *= 0.25
        cache.append(kk.cuda(), vv.cuda(), whole)
        k, v = stored(kk, k_bits, cache.bands), stored(vv, v_bits, cache.bands)
        check(x.cuda(), cache, batch, k, v, scale=0.09 / (ks * qs))


def test_huge_tokens_do_not_touch_rows_that_do_not_see_them():
    """Tokens past the range of half precision, between others of the same storage block."""
    n, q = 200, 150
    cache, batch, table = make([n], [q], heads=1)
    whole = paged.PagedBatch(table, [n], [n], 16, device="cuda:0")
    kk, vv = rows_of(n, 1, 3), rows_of(n, 1, 4)
    x = torch.randn(q, 4, 128).bfloat16().cuda()
    cache.append(kk.cuda(), vv.cuda(), whole)
    a = paged.attention(x, cache, batch)
    kk[120] *= 1e6
    vv[123] *= 1e9
    cache.append(kk.cuda(), vv.cuda(), whole)
    b = paged.attention(x, cache, batch)
    assert torch.equal(a[:70], b[:70])  # positions 50..119
    k, v = stored(kk, 4, cache.bands), stored(vv, 4, cache.bands)
    check(x, cache, batch, k, v, scale=0.09e-6)


@pytest.mark.parametrize("q", [1, 130])
def test_graph_captured_on_a_stream_that_is_used_outside_of_it(q):
    """Split units: launches outside a graph, on the stream it was captured on and before
    its first replay, and replays agree with a launch on another stream."""
    n = 5000
    cache, batch, table = make([n], [q], heads=1)
    fill(cache, table, [n])
    x = rows_of(q, 1, 9).cuda()
    want = paged.attention(x, cache, batch)
    torch.cuda.synchronize()
    st, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        a = paged.attention(x, cache, batch)
        b = paged.attention(x, cache, batch)
    with torch.cuda.stream(st):
        c = paged.attention(x, cache, batch)
    torch.cuda.synchronize()
    assert torch.equal(c, want)
    for _ in range(2):
        a.zero_(), b.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(a, want) and torch.equal(b, want)
    assert torch.equal(paged.attention(x, cache, batch), want)


def test_refusals():
    cache, batch, table = make([40, 20], [3, 2], heads=2)
    q, k = rows_of(5, 4, 1).cuda(), rows_of(5, 2, 2).cuda()

    def refuses(match, fn, *args, exc=ValueError, **kw):
        with pytest.raises(exc, match=match):
            fn(*args, **kw)

    refuses("not a multiple", paged.attention, q[:, :3], cache, batch)
    refuses("q must be", paged.attention, q[:4], cache, batch)
    refuses("q must be", paged.attention, q[0], cache, batch, exc=TypeError)
    refuses("bfloat16", paged.attention, q.float(), cache, batch, exc=TypeError)
    refuses("CPU|cuda", paged.attention, q.cpu(), cache, batch, exc=(RuntimeError, ValueError))
    refuses("PagedKVCache", paged.attention, q, batch, cache, exc=TypeError)
    refuses("PagedBatch", cache.append, k, k, table, exc=TypeError)
    refuses(">= 0", paged.attention, q, cache, batch, window=-1)
    refuses("window too", paged.attention, q, cache, batch, sink=4)
    for scale in (0.0, -1.0, float("nan"), float("inf"), 1e-50, 1e39):
        refuses("softmax_scale", paged.attention, q, cache, batch, softmax_scale=scale)
    refuses("out must have", paged.attention, q, cache, batch, out=torch.empty(5, 4, 256, device="cuda", dtype=torch.bfloat16)[..., ::2])
    refuses("k must be", cache.append, k[:4], k, batch)
    refuses("v must be", cache.append, k, q, batch)
    other = paged.PagedBatch(table, [40, 20], [3, 2], 32, device="cuda:0")
    refuses("pages of 32", cache.read, other)
    far = paged.PagedBatch([[1000, 3, 4], [5, 6, 0]], [40, 20], [3, 2], 16, device="cuda:0")
    refuses("names page 1000", cache.read, far)
    early = paged.PagedBatch(table, [40, 20], [41, 2], 16, device="cuda:0")
    refuses("every new token has a position", cache.append, rows_of(43, 2, 3).cuda(), rows_of(43, 2, 3).cuda(), early)
    refuses("every new token has a position", cache.read, early, new_only=True)
    twice = paged.PagedBatch([[0, 1, 2], [3, 2, 0]], [40, 20], [3, 2], 16, device="cuda:0")
    refuses("more than once", cache.append, k, k, twice)
    with pytest.raises(ValueError):
        batch.kv_lens[0] = 7
    g = torch.cuda.CUDAGraph()
    fresh = paged.PagedBatch(table, [40, 20], [3, 2], 16, device="cuda:0")
    torch.cuda.synchronize()
    with torch.cuda.graph(g):  # a first use in a capture cannot upload its plan
        with pytest.raises(RuntimeError, match="before the capture"):
            paged.attention(q, cache, fresh)
        y = q + 1
    assert y.shape == q.shape


@pytest.mark.parametrize("group", [5, 8, 11, 21])
@pytest.mark.parametrize("kv", [[300, 17, 1000, 0, 3], [2500, 4000, 90, 1, 64], [40000, 30000, 35000, 38000, 2]])
@pytest.mark.parametrize("k_bits,v_bits,mode", [(4, 4, "blind32"), (8, 8, "bands")])
def test_rows_between_the_two_kernels(group, kv, k_bits, v_bits, mode):
    """10 to 63 rows per KV head beside sequences with none and with one query: tiles of 16
    rows or of 128, by the lengths, whole and in parts."""
    q = [2, 3, 3, 0, 1]
    cache, batch, table = make(kv, q, heads=1 if kv[0] > 10000 else 2, page=32, k_bits=k_bits, v_bits=v_bits, mode=mode)
    k, v = fill(cache, table, kv)
    x = torch.randn(sum(q), cache.n_heads * group, 128).bfloat16().cuda()
    check(x, cache, batch, k, v)
    check(x, cache, batch, k, v, window=333, sink=40)


@pytest.mark.parametrize("rows", [17, 64, 65, 127, 128, 129])
@pytest.mark.parametrize("n", [64, 65, 128, 129, 192, 640, 9000])
def test_one_q_tile_takes_turns(rows, n):
    """Few and many key tiles, odd and even, whole and in parts; more sequences than the kernel
    for few rows takes at the longer ones."""
    seqs = 24 if n == 9000 else 3
    kv = [n] * seqs
    cache, batch, table = make(kv, [rows] * seqs, heads=1, page=64, mode="bands2", k_bits=8)
    k, v = fill(cache, table, kv)
    check(torch.randn(rows * seqs, 1, 128).bfloat16().cuda(), cache, batch, k, v)
