"""Paged, quantized KV cache for batches of sequences of different lengths.

    cache = PagedKVCache(n_pages, page_size, n_kv_heads, k_bits=4, v_bits=4, group_mode="bands4", device="cuda")
    batch = PagedBatch(block_table, kv_lens, q_lens, page_size, device="cuda")   # once per step, for all layers
    cache.append(k, v, batch)                  # quantize the step's new tokens into their pages
    out = attention(q, cache, batch)           # their queries over everything cached, causal
    k, v = cache.read(batch)                   # bf16 values of the sequences' tokens

One layer's K and V live in pages of 16 to 128 tokens; a sequence owns pages through
its row of the block table, so sequences grow, share a prefix, or drop their oldest
pages (an eviction that moves and requantizes nothing) by editing that row. Rows are
stored as QuantKVTensor stores them: int4 or int8 codes with one bf16 scale per
(token, head, channel group). There is no CPU path.
"""
from __future__ import annotations

import ctypes

import numpy as np
import torch

import quant_kv_kernels as _kern

from . import _lib
from .ops import _require_cuda

BLOCK = 16  # tokens of one storage block
PAGE_SIZES = (16, 32, 64, 128)
HEAD_DIM = 128
_FAR = 2 ** 32  # a window or sink beyond all positions


# the current stream of a device as an integer, and the current device: what the public
# calls return, without making a Stream object at every launch
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice
_capturing = torch._C._cuda_isCurrentStreamCapturing


def _launch(cache: "PagedKVCache", batch: "PagedBatch", raw: int, fn, what: str, *args) -> None:
    """One C call on the cache's device and its stream `raw`. A captured one holds addresses
    of the batch's uploads, so the cache, whose pages it holds too, keeps the batch."""
    if _current_device() == cache.device.index:
        rc = fn(*args, raw)
        captured = raw and _capturing()  # the legacy default stream, 0, cannot be captured
    else:
        with torch.cuda.device(cache.device):
            rc = fn(*args, raw)
            captured = raw and _capturing()
    if captured:
        cache._captured.add(batch)
    if rc:
        _lib.check(rc, what)


def _cuda_device(device) -> torch.device:
    dev = torch.device(device)
    if dev.type != "cuda":
        raise RuntimeError(f"the paged cache needs a CUDA (sm_100) device, got {device}; "
                           "the B200 build has no CPU path")
    return torch.device("cuda", torch.cuda.current_device()) if dev.index is None else dev


def _host_ints(x, name: str, ndim: int) -> np.ndarray:
    if isinstance(x, torch.Tensor):
        if x.device.type != "cpu":
            raise TypeError(f"{name} must be host data (a list, a numpy array or a CPU tensor): the step is planned "
                            "on the host")
        x = x.numpy()
    a = np.asarray(x)
    if a.size == 0:
        a = a.astype(np.int64)
    if a.ndim != ndim or a.dtype.kind not in "iu":
        raise ValueError(f"{name} must be a {ndim}-D array of whole numbers")
    return a.astype(np.int64)


class PagedBatch:
    """The sequences of one step: which pages they own, how many tokens they hold
    (new ones included) and how many of those are new. Shared by all layers and by
    append, read and attention. block_table [B, most pages], kv_lens [B] and q_lens
    [B] are host data; row b's first ceil(kv_lens[b] / page_size) entries are used.
    Tensors with one row per new token are ordered sequence after sequence.

    A CUDA graph into which a call was captured keeps this batch's lengths, table and work
    list, whose memory belongs to the batch: the cache holds the batch until its
    release_captured(), so only the cache has to be kept as long as the graph."""

    def __init__(self, block_table, kv_lens, q_lens, page_size: int, device="cuda"):
        dev = _cuda_device(device)
        if page_size not in PAGE_SIZES:
            raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {page_size}")
        kv, ql = _host_ints(kv_lens, "kv_lens", 1), _host_ints(q_lens, "q_lens", 1)
        table = _host_ints(block_table, "block_table", 2)
        n = len(kv)
        if len(ql) != n or table.shape[0] != n:
            raise ValueError(f"block_table, kv_lens and q_lens describe {table.shape[0]}, {n} and {len(ql)} sequences")
        if n and (kv.min() < 0 or ql.min() < 0):
            raise ValueError("kv_lens and q_lens must be >= 0")
        if kv.sum() >= 2 ** 31 - 256 or ql.sum() >= 2 ** 31 - 256:
            raise ValueError("a batch holds fewer than 2^31 tokens")
        pages = -(-kv // page_size)
        if n and pages.max() > table.shape[1]:
            raise ValueError(f"a sequence of {int(kv[pages.argmax()])} tokens needs {int(pages.max())} pages, "
                             f"block_table has {table.shape[1]} per sequence")
        used = np.arange(table.shape[1])[None] < pages[:, None]
        ids = table[used]
        if ids.size and (ids.min() < 0 or ids.max() >= 2 ** 31):
            raise ValueError("block_table has a page id that is not a page of any pool")
        self.device, self.page_size, self.n_seqs = dev, int(page_size), n
        self._plans = {}
        kv.setflags(write=False)
        ql.setflags(write=False)
        self.kv_lens, self.q_lens = kv, ql
        self.n_new, self.n_tokens = int(ql.sum()), int(kv.sum())
        self.n_pages_needed = int(ids.max()) + 1 if ids.size else 0
        # append: every new token has a position, and its page is written by it alone
        start = kv - ql
        self._append_error = None
        if n and start.min() < 0:
            self._append_error = "append needs q_lens <= kv_lens: every new token has a position"
        else:
            col = np.arange(table.shape[1])[None]
            fresh = used & (col >= (start // page_size)[:, None]) & (ql > 0)[:, None]
            written = table[fresh]
            listed = np.sort(ids)
            times = np.searchsorted(listed, written, side="right") - np.searchsorted(listed, written, side="left")
            if times.size and times.max() > 1:
                self._append_error = "append would write a page that the block table lists more than once"
        new_blocks = np.where(ql > 0, -(-kv // BLOCK) - np.maximum(start, 0) // BLOCK, 0)
        blocks = -(-kv // BLOCK)
        seqs = np.zeros((n, 8), dtype=np.int32)
        for col, x in enumerate((kv, ql)):
            seqs[:, col] = x
        for col, x in enumerate((ql, kv, new_blocks, blocks)):
            seqs[1:, 2 + col] = np.cumsum(x)[:-1]
        self.n_new_blocks, self.n_blocks = int(new_blocks.sum()), int(blocks.sum())
        # unused entries point at page 0, which any pool has
        width = int(pages.max()) if n else 0
        rows = np.where(used, table, 0)[:, :width].astype(np.int32)
        self._upload(seqs, rows)

    def _plan(self, cache: "PagedKVCache", n_q_heads: int, causal: bool, window: int, sink: int) -> "_Plan":
        """The work list of attention with this cache format, heads and masks, made at its
        first use in the step and shared by the step's layers."""
        key = (cache._format, n_q_heads, causal, window, sink)
        plan = self._plans.get(key)
        if plan is None:
            plan = self._plans[key] = _Plan(self, cache, n_q_heads, causal, window, sink)
        return plan

    def _upload(self, seqs: np.ndarray, rows: np.ndarray) -> None:
        self._dev = _Uploaded(np.concatenate((seqs.ravel(), rows.ravel())), self.device)
        base = self._dev.data.data_ptr()
        self._args = _lib.PagedBatchArgs(base + seqs.size * 4, rows.shape[1], base, self.n_new, self.n_tokens,
                                         self.n_new_blocks, self.n_blocks, self.n_seqs, 0)
        self._ref = ctypes.byref(self._args)

    def _use(self) -> int:
        """The current stream, on which the uploaded arguments are now safe to read."""
        raw = _raw_stream(self.device.index)
        if raw != self._dev.stream:
            self._dev.use()
        return raw


class _Uploaded:
    """int32 data copied to the device on the stream that is current when it is made."""

    def __init__(self, flat: np.ndarray, device: torch.device):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("call this once before the capture: its upload cannot be replayed")
        self.data = torch.empty(max(flat.size, 8), dtype=torch.int32, device=device)
        if flat.size:
            self.data[:flat.size].copy_(torch.from_numpy(flat).pin_memory(), non_blocking=True)
        self._event = torch.cuda.Event()
        self.stream = _raw_stream(device.index)
        self._event.record(torch.cuda.current_stream(device))

    def use(self) -> None:
        """Makes the data safe to read on the current stream, another one than that which
        uploaded it: waits for the upload, and tells the allocator. A capture begins
        with a synchronization, so an upload before it has completed."""
        if not torch.cuda.is_current_stream_capturing():
            stream = torch.cuda.current_stream(self.data.device)
            stream.wait_event(self._event)
            self.data.record_stream(stream)


class _Plan:
    """kvq_paged_plan of a batch: the work list on the device, and per stream a workspace
    and counters, so that launches on different streams may overlap."""

    def __init__(self, batch: PagedBatch, cache: "PagedKVCache", n_q_heads: int, causal: bool, window: int, sink: int):
        kv, ql = batch.kv_lens.astype(np.int32), batch.q_lens.astype(np.int32)
        self.info = _lib.PagedPlanInfo()
        sms = torch.cuda.get_device_properties(batch.device).multi_processor_count
        lib = _lib.load()
        words = np.empty(1 << 15, dtype=np.int32)
        for _ in range(2):  # again with more room where the plan is longer
            rc = lib.kvq_paged_plan(cache._ref, kv.ctypes.data, ql.ctypes.data, len(kv), n_q_heads, causal, window, sink,
                                    sms, words.ctypes.data, words.size, ctypes.byref(self.info))
            if self.info.words <= words.size:
                break
            words = np.empty(self.info.words, dtype=np.int32)
        _lib.check(rc, "kvq_paged_plan")
        self.device = batch.device
        self.items = _Uploaded(words[:self.info.words], batch.device)
        self._work, self._keep = {}, []

    def args(self, raw: int):
        """(info, plan, workspace, counters) for a launch on the current stream, raw."""
        # A captured launch gets a workspace of its graph's own (and counters that each replay
        # clears): the graph may be replayed beside launches of this stream, and memory that is
        # cleared in a graph is not cleared for a launch outside of it.
        capturing = self.info.n_units > 0 and torch.cuda.is_current_stream_capturing()
        got = None if capturing else self._work.get(raw)
        if got is None:
            n, c = self.info.workspace_bytes, self.info.n_units
            # counters count up to a unit's parts and are set back by the last one
            ws = torch.empty(max(n, 1), dtype=torch.uint8, device=self.device)
            counters = torch.zeros(max(c, 1), dtype=torch.int32, device=self.device)
            got = ctypes.byref(self.info), self.items.data.data_ptr(), ws.data_ptr(), counters.data_ptr()
            if not capturing:
                self._keep.append((ws, counters))
                self._work[raw] = got
        if raw != self.items.stream:
            self.items.use()
        return got


class PagedKVCache:
    """One layer's pool of pages. k_pages / v_pages: uint8 [n_pages, n_heads,
    page_size / 16, 16 * (code bytes + 2 * groups)], a block of 16 tokens of one head
    being its 16 rows of codes and then its 16 rows of bf16 scales; k_codes, k_scales,
    v_codes, v_scales are views of them."""

    def __init__(self, n_pages: int, page_size: int, n_heads: int, head_dim: int = HEAD_DIM, k_bits: int = 4,
                 v_bits: int = 4, group_mode: str = "bands", device="cuda"):
        from quant_kv import _band_edges
        dev = _cuda_device(device)
        if head_dim != HEAD_DIM:
            raise ValueError(f"the paged cache supports head_dim {HEAD_DIM}, got {head_dim}")
        if (k_bits, v_bits) not in ((4, 4), (8, 4), (8, 8)):
            raise ValueError(f"the paged cache holds K/V in 4/4, 8/4 or 8/8 bits, got {k_bits}/{v_bits}")
        if page_size not in PAGE_SIZES:
            raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {page_size}")
        if group_mode not in ("bands", "bands1", "bands2", "bands4", "blind32", "blind64"):
            raise ValueError("the paged cache supports the bands, bands2, bands4, blind32 and blind64 group modes, "
                             f"got {group_mode}")
        if n_pages < 1 or n_heads < 1:
            raise ValueError("n_pages and n_heads must be >= 1")
        self.device, self.n_pages, self.page_size = dev, int(n_pages), int(page_size)
        self.n_heads, self.head_dim = int(n_heads), int(head_dim)
        self.k_bits, self.v_bits, self.group_mode = int(k_bits), int(v_bits), group_mode
        self.bands = _band_edges(head_dim, group_mode)
        self._map = np.ascontiguousarray(_kern.host_chan_band(_kern.build_chan_band(self.bands, head_dim, "cpu")),
                                         dtype=np.int32)
        self._k_pages, self._v_pages = (
            torch.zeros((n_pages, n_heads, page_size // BLOCK, BLOCK * self._row_bytes(b)), dtype=torch.uint8,
                        device=dev) for b in (k_bits, v_bits))
        self._c = _lib.PagedCacheArgs(self._k_pages.data_ptr(), self._v_pages.data_ptr(), self.n_pages, self.page_size,
                                      self.n_heads, self.head_dim, self.k_bits, self.v_bits, len(self.bands),
                                      self._map.ctypes.data)
        self._ref = ctypes.byref(self._c)
        self._format = (self.n_heads, self.k_bits, self.v_bits, group_mode)
        self._captured = set()

    def _row_bytes(self, bits: int) -> int:
        return self._code_bytes(bits) + 2 * len(self.bands)

    def _code_bytes(self, bits: int) -> int:
        return self.head_dim // 2 if bits == 4 else self.head_dim

    def _codes(self, pages, bits):
        return pages[..., :BLOCK * self._code_bytes(bits)].unflatten(-1, (BLOCK, self._code_bytes(bits)))

    def _scales(self, pages, bits):
        return pages[..., BLOCK * self._code_bytes(bits):].view(torch.bfloat16).unflatten(-1, (BLOCK, len(self.bands)))

    # written in place by append and by whoever loads saved pages; never rebound
    k_pages = property(lambda self: self._k_pages)
    v_pages = property(lambda self: self._v_pages)
    # [n_pages, n_heads, page_size / 16, 16, code bytes or groups]
    k_codes = property(lambda self: self._codes(self.k_pages, self.k_bits))
    v_codes = property(lambda self: self._codes(self.v_pages, self.v_bits))
    k_scales = property(lambda self: self._scales(self.k_pages, self.k_bits))
    v_scales = property(lambda self: self._scales(self.v_pages, self.v_bits))

    def storage_bytes(self) -> int:
        return self._k_pages.numel() + self._v_pages.numel()

    def release_captured(self) -> None:
        """Drops the batches that were kept for CUDA graphs: a graph into which a call was
        captured reads the batch's table, lengths and plan at every replay. Call it when no
        such graph will be replayed again; the cache itself has to outlive them."""
        self._captured.clear()

    def _check(self, batch: PagedBatch) -> None:
        if not isinstance(batch, PagedBatch):
            raise TypeError(f"expected a PagedBatch, got {type(batch).__name__}")
        if batch.device != self.device:
            raise ValueError(f"the batch is on {batch.device}, the cache on {self.device}")
        if batch.page_size != self.page_size:
            raise ValueError(f"the batch has pages of {batch.page_size} tokens, the cache of {self.page_size}")
        if batch.n_pages_needed > self.n_pages:
            raise ValueError(f"the block table names page {batch.n_pages_needed - 1}, the cache has {self.n_pages}")

    def append(self, k: torch.Tensor, v: torch.Tensor, batch: PagedBatch) -> None:
        """Quantize the step's new tokens, k and v [n_new, n_heads, 128] bf16, into
        their pages (kvq_paged_append): codes and scales are those of QuantKVTensor's
        slice write; NaN is stored as 0 and infinities as the group's largest value."""
        self._check(batch)
        if batch._append_error:
            raise ValueError(batch._append_error)
        shape = (batch.n_new, self.n_heads, self.head_dim)
        k, ks = _rows(k, shape, self.device, "k")
        v, vs = _rows(v, shape, self.device, "v")
        _launch(self, batch, batch._use(), _lib.load().kvq_paged_append, "kvq_paged_append", k.data_ptr(), ks,
                v.data_ptr(), vs, self._ref, batch._ref)

    def read(self, batch: PagedBatch, new_only: bool = False):
        """(k, v) bf16 [n, n_heads, 128]: the values held for the sequences' tokens, or
        for their new tokens only, sequence after sequence (kvq_paged_read)."""
        self._check(batch)
        if new_only and batch._append_error and (batch.q_lens > batch.kv_lens).any():
            raise ValueError("new_only needs q_lens <= kv_lens: every new token has a position")
        n = batch.n_new if new_only else batch.n_tokens
        shape, row = (n, self.n_heads, self.head_dim), self.n_heads * self.head_dim
        k = torch.empty(shape, dtype=torch.bfloat16, device=self.device)
        v = torch.empty_like(k)
        _launch(self, batch, batch._use(), _lib.load().kvq_paged_read, "kvq_paged_read", self._ref, batch._ref,
                1 if new_only else 0, k.data_ptr(), row, v.data_ptr(), row)
        return k, v

    def __repr__(self):
        return (f"<PagedKVCache {self.n_pages} pages of {self.page_size} tokens, {self.n_heads} heads, "
                f"int{self.k_bits}/int{self.v_bits} groups={self.group_mode} ({len(self.bands)}) on {self.device}: "
                f"{self.storage_bytes() / 2**30:.2f} GiB resident>")


def _rows(t, shape, device, name: str):
    """(t, or a contiguous copy where its rows are not 16-byte aligned blocks; token stride)."""
    if not isinstance(t, torch.Tensor) or t.device != device:
        if _require_cuda(t) != device:
            raise ValueError(f"{name} is on {t.device}, the cache on {device}")
    if t.dtype is not torch.bfloat16:
        raise TypeError(f"{name} must be bfloat16, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} must be {tuple(shape)}, got {tuple(t.shape)}")
    row = shape[1] * shape[2]
    if t.data_ptr() % 16 == 0:
        if t.is_contiguous():
            return t, row
        s0, s1, s2 = t.stride()
        if s2 == 1 and (s1 == shape[2] or shape[1] == 1) and (shape[0] == 1 or (s0 % 8 == 0 and s0 >= row)):
            return t, (row if shape[0] == 1 else s0)
    return t.clone(memory_format=torch.contiguous_format), row


def attention(q: torch.Tensor, cache: PagedKVCache, batch: PagedBatch, causal: bool = True, window: int = 0,
              sink: int = 0, softmax_scale: float | None = None, out: torch.Tensor | None = None,
              return_lse: bool = False):
    """Attention of the new tokens' queries, q [n_new, n_q_heads, 128] bf16, over their
    sequences' cached tokens (append the step's k and v first): bf16 like q, and with
    return_lse also fp32 [n_new, n_q_heads], the natural log of the sum of exponentials.

    Query i of a sequence stands at position p = kv_len - q_len + i. It sees tokens j <= p
    if causal (else all); with a window, of those only j > p - window, and the first `sink`
    (so without causal a window bounds how far a query looks back, and all later tokens are
    seen). A query that sees nothing gives 0, and -inf. Query head h reads KV head
    h / (n_q_heads / n_heads); softmax_scale defaults to 1 / sqrt(128). Logits beyond 1e8 in
    magnitude, where fp32 no longer tells neighbours apart, may give NaN or 0, and so may
    products q . K_j beyond fp32's range before the scale."""
    if not isinstance(cache, PagedKVCache):
        raise TypeError(f"expected a PagedKVCache, got {type(cache).__name__}")
    cache._check(batch)
    if not isinstance(q, torch.Tensor) or q.dim() != 3:
        raise TypeError("q must be a [n_new, n_q_heads, 128] bfloat16 tensor")
    heads = q.shape[1]
    if heads < 1 or heads % cache.n_heads:
        raise ValueError(f"{heads} query heads are not a multiple of {cache.n_heads} KV heads")
    window, sink = int(window), int(sink)
    if window < 0 or sink < 0:
        raise ValueError("window and sink must be >= 0")
    if sink and not window:
        raise ValueError("sink keeps the first tokens of a window: give window too")
    window, sink = min(window, _FAR), min(sink, _FAR)
    scale = 0.0 if softmax_scale is None else float(softmax_scale)
    # least: the kernels hold it in fp32, where a smaller one is 0
    if softmax_scale is not None and not 1e-38 <= scale <= 1e38:
        raise ValueError(f"softmax_scale must be between 1e-38 and 1e38, got {softmax_scale}")
    shape, device = (batch.n_new, heads, cache.head_dim), cache.device
    q, qs = _rows(q, shape, device, "q")
    if out is None:
        out, os_ = torch.empty(shape, dtype=torch.bfloat16, device=device), heads * cache.head_dim
    else:
        rows, os_ = _rows(out, shape, device, "out")
        if rows is not out:
            raise ValueError("out must have contiguous [heads, channels] blocks, 16-byte aligned rows")
    lse = torch.empty(shape[:2], dtype=torch.float32, device=device) if return_lse else None
    plan = batch._plan(cache, heads, bool(causal), window, sink)
    raw = batch._use()
    _launch(cache, batch, raw, _lib.load().kvq_paged_attention, "kvq_paged_attention", q.data_ptr(), qs, cache._ref,
            batch._ref, out.data_ptr(), os_, lse.data_ptr() if return_lse else None, heads, 1 if causal else 0, window, sink,
            scale, *plan.args(raw))
    return (out, lse) if return_lse else out
