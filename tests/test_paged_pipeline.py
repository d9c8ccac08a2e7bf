"""A model of the barriers between the warps of the paged attention kernel for many rows
(kvq_paged_tiles.cu), run under many orders of its warps: no tile is multiplied before both
of its tensors are converted, no stage or exponent slot is written while it is still read, and
every order ends. The stage and barrier counts are those of the source."""
import os
import random
import re

import pytest

SOURCE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "krea-realtime-bench_b200", "csrc",
                      "kvq_paged_tiles.cu")


def geometry(v_bits):
    src = open(SOURCE).read()
    nk, nv8, nv4 = map(int, re.search(r"NK = (\d+), NV = VB == 8 \? (\d+) : (\d+);", src).groups())
    ready = int(re.search(r"kReady = (\d+);", src).group(1))
    exp_k, exp_v = map(int, re.search(r"kExpK = (\d+), kExpV = (\d+);", src).groups())
    assert "NV1 = NV + kQTile / kKVTile;" in src  # 32 KB, 16 KB
    nv = nv8 if v_bits == 8 else nv4
    return nk, nv, nv + 2, ready, exp_k, exp_v


class Barrier:
    """An mbarrier: a wait for a parity passes while the current phase has the other one."""

    def __init__(self, count):
        self.count, self.pending, self.phase = count, count, 0

    def arrive(self):
        self.pending -= 1
        if self.pending == 0:
            self.phase, self.pending = self.phase + 1, self.count

    def passed(self, parity):
        return self.phase & 1 != parity & 1


def run(n_tiles, shared, geo, rng):
    """One order of the warps; returns after the last tile or raises AssertionError."""
    nk, nv, nv1, n_ready, exp_k, exp_v = geo
    if shared:
        nv = nv1
    ready = [Barrier(4) for _ in range(n_ready)]
    empty = {t: [Barrier(1 if shared else 2) for _ in range(n)] for t, n in (("K", nk), ("V", nv))}
    s_full = [[Barrier(1), Barrier(1)] for _ in range(2)]
    p_full = [[Barrier(1), Barrier(1)] for _ in range(2)]
    tile = (lambda x, i: 2 * i + x) if shared else (lambda x, i: i)
    mine = [(n_tiles - x + 1) // 2 if shared else n_tiles for x in (0, 1)]
    users = (lambda j: [j & 1]) if shared else (lambda j: [0, 1])
    index = (lambda j: j // 2) if shared else (lambda j: j)
    stages, slots = {"K": nk, "V": nv}, {"K": exp_k, "V": exp_v}
    converted = {t: [0] * n_tiles for t in "KV"}
    at = {(t, w): 0 for t in "KV" for w in (0, 1)}  # next tile of a converter warp
    s_issued, pv_issued, s_done, pv_done, steps = ([0, 0] for _ in range(5))
    s_looked = [0, 0]  # S found complete, the arrivals made
    queue = [[], []]   # products under way, in order

    def convert(t, w):
        j, n = at[t, w], stages[t]
        if j == n_tiles or (j >= n and not empty[t][j % n].passed(j // n - 1)):
            return None

        def go():
            if j >= n:
                for x in users(j - n):
                    done = s_done if t == "K" else pv_done
                    assert done[x] > index(j - n), f"{t}({j}) overwrites {t}({j - n}), which is still read"
            if j >= slots[t]:
                for x in users(j - slots[t]):
                    assert steps[x] > index(j - slots[t]), f"exponents of {t}({j - slots[t]}) are still read"
            converted[t][j] += 1
            at[t, w] = j + 1
            ready[j % n_ready].arrive()
        return go

    def issue(x):
        """The next product of MMA thread x: S(0), S(1), PV(0), S(2), PV(1), ..."""
        i, p = s_issued[x], pv_issued[x]
        if i < mine[x] and i - p < 2:
            j = tile(x, i)
            if not ready[j % n_ready].passed(j // n_ready):
                return None

            def go():
                assert converted["K"][j] == 2, f"S({j}) before K({j}) is converted"
                assert converted["V"][j] == 2, f"S({j}) before the exponents of V({j}) are written"
                s_issued[x] += 1
                queue[x].append(("S", i))
            return go
        if p < mine[x] and p_full[x][p & 1].passed(p >> 1):
            def go():
                pv_issued[x] += 1
                queue[x].append(("PV", p))
            return go
        return None

    def complete(x):
        if not queue[x]:
            return None

        def go():
            kind, i = queue[x].pop(0)
            if kind == "S":
                s_done[x] += 1
                s_full[x][i & 1].arrive()
            else:
                pv_done[x] += 1
        return go

    def look(x):
        """Softmax set x finds S of its next tile complete and gives back what that frees."""
        i = s_looked[x]
        if i == mine[x] or steps[x] < i or not s_full[x][i & 1].passed(i >> 1):
            return None

        def go():
            assert s_done[x] > i
            s_looked[x] += 1
            empty["K"][tile(x, i) % nk].arrive()
            if i >= 2:
                empty["V"][tile(x, i - 2) % nv].arrive()
        return go

    def step(x):
        i = steps[x]
        if s_looked[x] <= i:
            return None

        def go():
            steps[x] += 1
            p_full[x][i & 1].arrive()
        return go

    actors = [(convert, t, w) for t in "KV" for w in (0, 1)] + [(f, x) for f in (issue, complete, look, step) for x in (0, 1)]
    # some warps are much slower than others, now and then for a while
    pace = {a: rng.choice((1.0, 1.0, 0.1, 1e-4)) for a in actors}
    while any(d < m for d, m in zip(pv_done, mine)):
        if rng.random() < 0.02:
            pace[rng.choice(actors)] = rng.choice((1.0, 0.1, 1e-4))
        able = [(a, g) for a in actors if (g := a[0](*a[1:])) is not None]
        assert able, "the warps wait for each other"
        rng.choices([g for _, g in able], [pace[a] for a, _ in able])[0]()


@pytest.mark.parametrize("v_bits", [4, 8])
@pytest.mark.parametrize("shared", [False, True])
def test_no_order_of_the_warps_reads_early_or_overwrites(v_bits, shared):
    geo = geometry(v_bits)
    for seed in range(300):
        run(random.Random(seed).choice((1, 2, 3, 5, 9, 24)), shared, geo, random.Random(seed))
