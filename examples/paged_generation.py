"""Generation with a paged, quantized KV cache: requests of different lengths in one batch.

    python examples/paged_generation.py                 # tokens per second
    python examples/paged_generation.py --check         # each attention against a dense one

A small decoder with random weights (there is no checkpoint here) serves a queue of
requests. Every step takes one token of each running request and fills up with chunks of
waiting prompts; per layer it appends the step's keys and values to the pages and attends
over them. Requests begin with the same instructions, whose full pages they share, grow
page by page, give back the pages that a sliding window has left, and all others when they
end. The window keeps the first tokens.
"""
import argparse
import os
import sys
import time

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "krea-realtime-bench_b200"))
from kvq import paged  # noqa: E402


class Pool:
    """Free pages and how many requests use each."""

    def __init__(self, n_pages):
        self.free, self.users = list(range(n_pages))[::-1], [0] * n_pages

    def take(self):
        page = self.free.pop()
        self.users[page] = 1
        return page

    def give_back(self, page):
        self.users[page] -= 1
        if self.users[page] == 0:
            self.free.append(page)


class Request:
    def __init__(self, tokens, n_out):
        self.tokens, self.n_prompt, self.n_out = list(tokens), len(tokens), n_out
        self.pages, self.held, self.released = [], 0, 0  # held: tokens in the cache

    def grow(self, pool, n_tokens, page_size):
        while len(self.pages) * page_size < n_tokens:
            self.pages.append(pool.take())

    def share(self, other, n_tokens, page_size):
        """Takes the full pages of other's first n_tokens, which both begin with."""
        n = min(n_tokens, other.held) // page_size
        if n and not other.released:
            self.pages, self.held = other.pages[:n], n * page_size

    def release(self, pool, window, sink, page_size):
        """Gives back pages that no later token sees. Their entries name the first page."""
        last = max(0, self.held + 1 - window) // page_size
        for i in range(max(self.released, -(-sink // page_size), 1), last):
            pool.give_back(self.pages[i])
            self.pages[i] = self.pages[0]
            self.released = i + 1

    def end(self, pool, sink, page_size):
        kept = max(-(-sink // page_size), 1)
        for i, page in enumerate(self.pages):
            if i < kept or i >= self.released:
                pool.give_back(page)


class Decoder:
    """Attention layers with random weights; greedy next tokens."""

    def __init__(self, a, device):
        g = torch.Generator(device=device).manual_seed(0)
        d = a.heads * a.group * 128
        rand = lambda *s: (torch.randn(s, generator=g, device=device) * s[-1] ** -0.5).bfloat16()
        self.a, self.emb = a, rand(a.vocab, d) * d ** 0.5
        self.qkv = [rand(d + 2 * a.heads * 128, d) for _ in range(a.layers)]
        self.proj = [rand(d, d) for _ in range(a.layers)]
        self.caches = [paged.PagedKVCache(a.pages, a.page, a.heads, k_bits=a.k_bits, v_bits=a.v_bits,
                                          group_mode=a.group_mode, device=device) for _ in range(a.layers)]
        self.worst = 0.0

    def step(self, tokens, batch):
        """The next token after each sequence's last new one."""
        a, hq = self.a, self.a.heads * self.a.group
        x = self.emb[torch.from_numpy(tokens).to(batch.device)]
        for qkv, proj, cache in zip(self.qkv, self.proj, self.caches):
            y = torch.nn.functional.rms_norm(x, x.shape[-1:]) @ qkv.T
            q, k, v = (t.unflatten(-1, (-1, 128)) for t in y.split((hq * 128, a.heads * 128, a.heads * 128), dim=-1))
            cache.append(k, v, batch)
            o = paged.attention(q, cache, batch, window=a.window, sink=a.sink)
            if a.check:
                self.worst = max(self.worst, difference(q, o, cache, batch, a))
            x = x + o.flatten(1) @ proj.T
        ends = torch.from_numpy(np.cumsum(batch.q_lens) - 1).to(batch.device)
        return (torch.nn.functional.rms_norm(x[ends], x.shape[-1:]) @ self.emb.T).argmax(-1).tolist()


def difference(q, o, cache, batch, a):
    """Relative error (2-norm) of the step's attention against a dense one in fp32 over the
    values read back."""
    k, v = (t.float() for t in cache.read(batch))
    want, q0, k0 = [], 0, 0
    for n, m in zip(batch.kv_lens.tolist(), batch.q_lens.tolist()):
        p = torch.arange(n - m, n, device=q.device)[:, None]
        j = torch.arange(n, device=q.device)[None]
        see = (j <= p) & ((j > p - a.window) | (j < a.sink)) if a.window else j <= p
        ks, vs = (t[k0:k0 + n].repeat_interleave(a.group, 1) for t in (k, v))
        s = torch.einsum("qhd,khd->hqk", q[q0:q0 + m].float(), ks) * 128 ** -0.5
        want.append(torch.einsum("hqk,khd->qhd", s.masked_fill(~see, -torch.inf).softmax(-1), vs))
        q0, k0 = q0 + m, k0 + n
    want = torch.cat(want)
    return float((o.float() - want).norm() / want.norm())


def generate(a, device="cuda:0"):
    rng = np.random.default_rng(0)
    torch.cuda.set_device(device)
    model, pool = Decoder(a, device), Pool(a.pages)
    common = rng.integers(0, a.vocab, a.common)
    waiting = [Request(np.concatenate((common, rng.integers(0, a.vocab, rng.integers(1, a.prompt + 1)))),
                       int(rng.integers(1, a.out + 1))) for _ in range(a.requests)]
    running, done, n_steps, n_tokens = [], [], 0, 0
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    while waiting or running:
        # one token of each running request, then chunks of prompts
        budget, takes = a.step_tokens, []
        for r in running:
            n = min(len(r.tokens) - r.held, budget)
            takes.append(n)
            budget -= n
        room = lambda r: len(pool.free) - sum(-(-x.n_prompt // a.page) - len(x.pages) for x in running if x.held < x.n_prompt) > \
            (len(r.tokens) + r.n_out) // a.page + len(running) + 1
        while waiting and budget > 0 and len(running) < a.batch and room(waiting[0]):
            r = waiting.pop(0)
            if running:
                r.share(running[0], a.common, a.page)
                for page in r.pages:
                    pool.users[page] += 1
            n = min(len(r.tokens) - r.held, budget)
            running.append(r)
            takes.append(n)
            budget -= n
        if not running:
            raise RuntimeError("the pool is too small for the next request")
        for r, n in zip(running, takes):
            r.grow(pool, r.held + n, a.page)
            r.held += n
        width = max(len(r.pages) for r in running)
        table = np.zeros((len(running), width), dtype=np.int64)
        for i, r in enumerate(running):
            table[i, :len(r.pages)] = r.pages
        batch = paged.PagedBatch(table, [r.held for r in running], takes, a.page, device)
        tokens = np.concatenate([r.tokens[r.held - n:r.held] for r, n in zip(running, takes)]).astype(np.int64)
        following = model.step(tokens, batch)
        n_steps, n_tokens = n_steps + 1, n_tokens + len(tokens)
        for r, n, token in zip(list(running), takes, following):
            if n and r.held == len(r.tokens):
                r.tokens.append(token)
                if len(r.tokens) - r.n_prompt == r.n_out:
                    r.end(pool, a.sink if a.window else 0, a.page)
                    running.remove(r)
                    done.append(r)
                    continue
            if a.window:
                r.release(pool, a.window, a.sink, a.page)
    torch.cuda.synchronize()
    seconds = time.perf_counter() - t0
    assert len(pool.free) == a.pages, "every page was given back"
    return dict(requests=len(done), steps=n_steps, tokens=n_tokens, seconds=seconds, worst=model.worst,
                generated=sum(r.n_out for r in done), outputs=[r.tokens[r.n_prompt:] for r in done])


def parse(argv=None):
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value, text in (("layers", 4, "attention layers"), ("heads", 4, "KV heads"), ("group", 4, "query heads per KV head"),
                              ("vocab", 1000, "tokens of the vocabulary"), ("requests", 40, "requests"),
                              ("batch", 24, "most requests at a time"), ("prompt", 900, "longest own prompt"),
                              ("common", 200, "instructions that all begin with"), ("out", 60, "most tokens to generate"),
                              ("page", 16, "tokens of a page"), ("pages", 4000, "pages of the pool"),
                              ("step-tokens", 512, "most tokens of a step"), ("window", 512, "sliding window (0: none)"),
                              ("sink", 64, "first tokens that the window keeps"), ("k-bits", 4, "bits of a key"),
                              ("v-bits", 4, "bits of a value")):
        p.add_argument("--" + name, type=int, default=value, help=f"{text} ({value})")
    p.add_argument("--group-mode", default="blind32", help="groups of channels that share a scale (blind32)")
    p.add_argument("--check", action="store_true", help="compare each attention with a dense one")
    a = p.parse_args(argv)
    if not a.window:
        a.sink = 0
    return a


def main(argv=None):
    a = parse(argv)
    r = generate(a)
    print(f"{r['requests']} requests, {r['steps']} steps, {r['tokens']} tokens through {a.layers} layers, "
          f"{r['generated']} generated: {r['seconds']:.2f} s, {r['tokens'] / r['seconds']:.0f} tokens/s")
    if a.check:
        print(f"largest relative error of an attention: {r['worst']:.1e}")
        # the output's and the weights' roundings (2^-9, 2^-11 and less) averaged over elements
        return 0 if r["worst"] < 2.0 ** -8 else 1
    return 0


if __name__ == "__main__":
    sys.exit(main())
