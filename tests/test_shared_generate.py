"""Shared attention, accumulated weights and eviction together, as
examples/paged_generate.py uses them, against a dense model in 64 bits
(test_paged_generate.py, whose tolerances hold here: an eviction rounds the keys
that move once more, as a drop does).

Weights: a score is off by about 2^-11 of scores of order 1, through the keys'
rounding and through the queries', per layer: 8 x 2^-11 of their norm, as the
logits.
"""
import importlib.util
import os
import types

import numpy as np
import pytest

from conftest import ROOT
from test_paged_generate import Dense, example, logits_of  # noqa: F401  (a fixture)


class Weighed(Dense):
    """A conversation that keeps the weight of each of its tokens."""

    def __init__(self, model):
        super().__init__(model)
        self.mass = np.empty(0)

    def add(self, tokens):
        held, n, (d, kv, H) = len(self.k[0]), len(tokens), (self.m.cfg[x] for x in ("d", "kv", "heads"))
        out = super().add(tokens)
        self.mass = np.concatenate([self.mass, np.zeros(n)])
        # the same once more for the weights: the layers' queries from their inputs
        norm = lambda x: x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6)  # noqa: E731
        x = self.embed[np.array(tokens)]
        for i, w in enumerate(self.w):
            y = (norm(x) @ w["qkv"].T).reshape(n, -1, d)
            q, k = self.turn(y[:, :H], held), self.turn(self.k[i], 0)
            a = np.empty((n, H, d))
            for t in range(n):
                for j in range(H):
                    s = k[:held + t + 1, j * kv // H] @ q[t, j] / np.sqrt(d)
                    e = np.exp(s - s.max())
                    self.mass[:held + t + 1] += e / e.sum()
                    a[t, j] = e / e.sum() @ self.v[i][:held + t + 1, j * kv // H]
            x = x + a.reshape(n, -1) @ w["o"].T
            y = norm(x)
            g = y @ w["gate"].T
            x = x + (g / (1 + np.exp(-g)) * (y @ w["up"].T)) @ w["down"].T
        return out

    def copy(self):
        c = Weighed(self.m)
        c.k, c.v, c.mass = [x.copy() for x in self.k], [x.copy() for x in self.v], self.mass.copy()
        return c

    def keep(self, src):
        self.k, self.v = ([x[src] for x in y] for y in (self.k, self.v))
        self.mass = self.mass[src]


def near(got, want, n):
    return np.linalg.norm(got - want) <= n * 2.0 ** -11 * np.linalg.norm(want)


@pytest.mark.gpu
def test_answers_over_one_budget(example, torch):  # noqa: F811
    """Prompts, forks, tokens of families, evictions of rows that share pages and
    of rows that own theirs, and tokens after them."""
    rng = np.random.default_rng(6)
    m = example.PagedModel(example.SMALL, 8, 90)
    words, cache, mass = example.words, m.cache, m.cache.mass()
    seqs = [rng.integers(0, 4096, k).tolist() for k in (120, 50)]
    dense = [Weighed(m) for _ in seqs]
    for x, s in zip(dense, seqs):
        x.add(s)
    cache.extend(words([120, 50]), rows=words([0, 1]))
    m.forward(words(sum(seqs, [])), words([0, 1]), words([0, 120, 170]), 120, mass=mass)
    for r, x in enumerate(dense):
        assert near(mass[r, :len(x.mass)].double().cpu().numpy(), x.mass, 8)
        assert not mass[r, len(x.mass):].any()
    src, kids = words([0, 0, 0, 1, 1]), words([2, 3, 4, 5, 6])
    cache.fork(src, kids)
    mass[kids.long()] = mass[src.long()]
    rows = [dense[0].copy(), dense[0].copy(), dense[0].copy(), dense[1].copy(), dense[1].copy()]
    families = words([0, 3, 5])

    def tokens(steps, n):
        for _ in range(steps):
            new = rng.integers(0, 4096, 5).tolist()
            cache.extend(1, rows=kids)
            got = logits_of(m, m.forward(words(new), kids, families=families, mass=mass), torch)
            for i, (x, t) in enumerate(zip(rows, new)):
                assert near(got[i], x.add([t]), n)
                assert near(mass[2 + i, :len(x.mass)].double().cpu().numpy(), x.mass, n)

    def cut(of, budget, first, recent):
        before, lens = mass.double().cpu().numpy(), cache.len.cpu().tolist()
        cache.evict(mass, budget, words([2 + i for i in of]), first=first, recent=recent, rope=m.rope)
        for i in of:
            w, n = before[2 + i], lens[2 + i]
            if n <= budget:
                continue
            middle = sorted(range(first, n - recent), key=lambda t: (-w[t], t))[:budget - first - recent]
            stays = list(range(first)) + sorted(middle) + list(range(n - recent, n))
            rows[i].keep(stays)
            assert np.array_equal(mass[2 + i, :budget].double().cpu().numpy(), w[stays])
        assert cache.len.cpu().tolist()[2:7] == [len(x.mass) for x in rows]

    tokens(3, 8)
    cut([1, 3], 45, 4, 12)                                         # pages that other rows hold too: those are as before
    tokens(2, 16)
    cut([0, 1, 2, 3, 4], 40, 2, 9)                                 # some rows' pages are their own by now
    tokens(2, 16)
    # the prompts' own rows still hold all of their tokens
    cache.extend(1, rows=words([0, 1]))
    got = logits_of(m, m.forward(words([7, 8]), words([0, 1])), torch)
    for g, x, t in zip(got, dense, (7, 8)):
        assert near(g, x.add([t]), 8)


@pytest.mark.gpu
def test_generate(example, torch):  # noqa: F811
    """Rows that fill up are cut to the budget and go on; the pages are accounted
    for, and the same call gives the same tokens."""
    rng = np.random.default_rng(4)
    prompts = [rng.integers(0, 4096, k) for k in (150, 190, 5)]
    runs = []
    for _ in range(2):
        m = example.PagedModel(example.SMALL, 9, 9 * 12)
        runs.append(example.generate(m, prompts, 2, 120, shared=True, budget=96))
        ref = torch.zeros_like(m.cache.ref)
        held = m.cache.table[m.cache.table >= 0].long()
        ref.index_add_(0, held, torch.ones_like(held, dtype=torch.int32))
        assert torch.equal(ref, m.cache.ref)
        assert m.cache.len.cpu().tolist()[:3] == [0, 0, 0] and int(m.cache.len.max()) <= 192
    assert runs[0] == runs[1] and all(len(r) == 120 for r in runs[0])


@pytest.mark.parametrize("budget", [192, 193, 4096, -1])
def test_budgets_that_cut_nothing(budget):
    """A budget that a full row is within would leave it full: each later token
    would be refused its place and written over the last one's."""
    spec = importlib.util.spec_from_file_location("paged_generate", os.path.join(ROOT, "examples", "paged_generate.py"))
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    with pytest.raises(ValueError, match="budget"):
        ex.generate(types.SimpleNamespace(cfg=ex.SMALL, cache=None), [np.arange(5)], 2, 8, budget=budget)
