"""The operators together, as examples/paged_generate.py uses them, against a
dense model in 64 bits from the dequantised weights.

Tolerance: the cache rounds keys and values to f16 (2^-11 of each value); per
layer that moves the attention's output by at most 2^-11 through the values and
about as much through the scores (their error is 2^-11 of scores of order 1),
and the residual stream passes it on: 2 layers, 2 effects, 2 for the norms'
gains: 8 x 2^-11 of the logits' norm.
"""
import importlib.util
import os

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example(gpu):
    spec = importlib.util.spec_from_file_location("paged_generate", os.path.join(ROOT, "examples", "paged_generate.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def matrix(blocks, rows, cols):
    b = blocks.reshape(-1, 34)
    d = b[:, :2].copy().view(np.float16).astype(np.float64)
    return (d * b[:, 2:].copy().view(np.int8)).reshape(rows, cols)


def dense_logits(model, tokens, positions=None):
    """Logits after `tokens` [n], all keys in 64 bits."""
    c = model.cfg
    h, d, H, kv = c["hidden"], c["d"], c["heads"], c["kv"]
    norm = lambda x: x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6)  # noqa: E731
    x = model.embed.double().cpu().numpy()[tokens]
    n = len(tokens)
    pos = np.arange(n) if positions is None else positions
    ang = pos[:, None] * c["base"] ** (-2.0 * np.arange(d // 2) / d)
    cos, sin = np.cos(ang)[:, None], np.sin(ang)[:, None]

    def turn(a):
        u, v = a[..., :d // 2], a[..., d // 2:]
        return np.concatenate([u * cos - v * sin, v * cos + u * sin], -1)

    for b in model.blocks:
        y = (norm(x) @ matrix(b["qkv"], (H + 2 * kv) * d, h).T).reshape(n, -1, d)
        q, k, v = turn(y[:, :H]), turn(y[:, H:H + kv]), y[:, H + kv:]
        out = np.empty((n, H, d))
        for i in range(H):
            s = q[:, i] @ k[:, i * kv // H].T / np.sqrt(d)
            s[np.triu_indices(n, 1)] = -np.inf
            e = np.exp(s - s.max(1, keepdims=True))
            out[:, i] = e / e.sum(1, keepdims=True) @ v[:, i * kv // H]
        x = x + out.reshape(n, -1) @ matrix(b["o"], h, H * d).T
        y = norm(x)
        g = y @ matrix(b["gate"], c["ffn"], h).T
        x = x + (g / (1 + np.exp(-g)) * (y @ matrix(b["up"], c["ffn"], h).T)) @ matrix(b["down"], h, c["ffn"]).T
    return norm(x[-1]) @ matrix(model.head_blocks, c["vocab"], h).T


def logits_of(model, hidden, torch):
    out = torch.empty((hidden.shape[0], model.cfg["vocab"]), device="cuda")
    model.lm_head.gemv(hidden.contiguous(), out, B=hidden.shape[0])
    return out.double().cpu().numpy()


def near(got, want):
    return np.linalg.norm(got - want) <= 8 * 2.0 ** -11 * np.linalg.norm(want)


@pytest.mark.gpu
def test_chunks_then_tokens(example, torch):
    """Prompts in one call, continued by a chunk, by single tokens and after a
    fork: the logits of a dense model over the same tokens."""
    rng = np.random.default_rng(3)
    m = example.PagedModel(example.SMALL, 6, 60)
    seqs = [rng.integers(0, 4096, k).tolist() for k in (60, 7, 1)]
    rows = example.words([2, 0, 4])
    start = example.words(np.concatenate([[0], np.cumsum([len(s) for s in seqs])]).tolist())
    m.cache.extend(example.words([len(s) for s in seqs]), rows=rows)
    out = m.forward(example.words(sum(seqs, [])), rows, start, 60)
    got = logits_of(m, out[(start[1:] - 1).long()], torch)
    for g, s in zip(got, seqs):
        assert near(g, dense_logits(m, np.array(s)))
    more = [rng.integers(0, 4096, k).tolist() for k in (1, 40, 3)]          # a token, a chunk, a few
    start = example.words(np.concatenate([[0], np.cumsum([len(s) for s in more])]).tolist())
    m.cache.extend(example.words([len(s) for s in more]), rows=rows)
    out = m.forward(example.words(sum(more, [])), rows, start, 40)
    got = logits_of(m, out[(start[1:] - 1).long()], torch)
    seqs = [s + x for s, x in zip(seqs, more)]
    for g, s in zip(got, seqs):
        assert near(g, dense_logits(m, np.array(s)))
    m.cache.fork(example.words([2, 0]), example.words([1, 3]))              # both go on by themselves
    rows = example.words([2, 0, 1, 3])
    seqs = [seqs[0], seqs[1], list(seqs[0]), list(seqs[1])]
    for _ in range(20):
        new = rng.integers(0, 4096, 4).tolist()
        m.cache.extend(1, rows=rows)
        out = m.forward(example.words(new), rows)
        for s, x in zip(seqs, new):
            s.append(x)
    for g, s in zip(logits_of(m, out, torch), seqs):
        assert near(g, dense_logits(m, np.array(s)))


@pytest.mark.gpu
def test_generate_past_the_context(example, torch):
    """Rows that fill up lose tokens and go on; the pages are accounted for,
    and the same call gives the same tokens."""
    rng = np.random.default_rng(4)
    prompts = [rng.integers(0, 4096, k) for k in (150, 190, 5)]
    runs = []
    for _ in range(2):
        m = example.PagedModel(example.SMALL, 9, 9 * 12)
        runs.append(example.generate(m, prompts, 2, 120))
        ref = torch.zeros_like(m.cache.ref)
        held = m.cache.table[m.cache.table >= 0].long()
        ref.index_add_(0, held, torch.ones_like(held, dtype=torch.int32))
        assert torch.equal(ref, m.cache.ref)
        assert m.cache.len.cpu().tolist()[:3] == [0, 0, 0] and int(m.cache.len.max()) <= 192
    assert runs[0] == runs[1] and all(len(r) == 120 for r in runs[0])


class Dense:
    """One conversation in 64 bits: keys before their rotation and values of
    each layer, and what happens to them."""

    def __init__(self, model):
        c, self.m = model.cfg, model
        h, d, H, kv = c["hidden"], c["d"], c["heads"], c["kv"]
        shapes = dict(qkv=((H + 2 * kv) * d, h), o=(h, H * d), gate=(c["ffn"], h), up=(c["ffn"], h), down=(h, c["ffn"]))
        self.w = [{n: matrix(b[n], *s) for n, s in shapes.items()} for b in model.blocks]
        self.head = matrix(model.head_blocks, c["vocab"], h)
        self.embed = model.embed.double().cpu().numpy()
        self.k = [np.empty((0, kv, d)) for _ in self.w]
        self.v = [np.empty((0, kv, d)) for _ in self.w]

    def turn(self, x, first):
        """x [n, heads, d] at positions first ..: as complex numbers."""
        d = self.m.cfg["d"]
        ang = (first + np.arange(len(x)))[:, None] * self.m.cfg["base"] ** (-2.0 * np.arange(d // 2) / d)
        z = (x[..., :d // 2] + 1j * x[..., d // 2:]) * np.exp(1j * ang)[:, None]
        return np.concatenate([z.real, z.imag], -1)

    def add(self, tokens):
        """The logits after the last of them."""
        c = self.m.cfg
        d, H, kv, n = c["d"], c["heads"], c["kv"], len(tokens)
        norm = lambda x: x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6)  # noqa: E731
        x = self.embed[np.array(tokens)]
        for i, w in enumerate(self.w):
            y = (norm(x) @ w["qkv"].T).reshape(n, -1, d)
            held = len(self.k[i])
            self.k[i], self.v[i] = np.concatenate([self.k[i], y[:, H:H + kv]]), np.concatenate([self.v[i], y[:, H + kv:]])
            q, k = self.turn(y[:, :H], held), self.turn(self.k[i], 0)
            a = np.empty((n, H, d))
            for t in range(n):
                for j in range(H):
                    s = k[:held + t + 1, j * kv // H] @ q[t, j] / np.sqrt(d)
                    e = np.exp(s - s.max())
                    a[t, j] = e / e.sum() @ self.v[i][:held + t + 1, j * kv // H]
            x = x + a.reshape(n, -1) @ w["o"].T
            y = norm(x)
            g = y @ w["gate"].T
            x = x + (g / (1 + np.exp(-g)) * (y @ w["up"].T)) @ w["down"].T
        return self.head @ norm(x[-1])

    def drop(self, start, end):
        self.k, self.v = ([np.delete(x, slice(start, end), 0) for x in y] for y in (self.k, self.v))


@pytest.mark.gpu
def test_tokens_after_a_drop(example, torch):
    """Rows that own their pages and rows that share them lose tokens, twice, and
    go on: the logits of a model that moves its own keys and values.  A drop
    rounds the moved keys once more: 3 effects per layer in place of 2, and 4
    after the second, of two layers: 16 x 2^-11 of the norm."""
    rng = np.random.default_rng(5)
    m = example.PagedModel(example.SMALL, 4, 48)
    seqs = [rng.integers(0, 4096, k).tolist() for k in (150, 61)]
    dense = [Dense(m) for _ in seqs]
    for x, s in zip(dense, seqs):
        x.add(s)
    rows = example.words([0, 1])
    m.cache.extend(example.words([150, 61]), rows=rows)
    m.forward(example.words(sum(seqs, [])), rows, example.words([0, 150, 211]), 150)
    m.cache.fork(example.words([0]), example.words([3]))        # row 0's full pages are shared now, row 1's are its own
    for cut, new in (([(8, 77), (5, 6)], 3), ([(0, 20), (30, 63)], 2)):
        m.cache.drop(example.words([a for a, _ in cut]), example.words([b for _, b in cut]), rows, rope=m.rope)
        for x, (a, b) in zip(dense, cut):
            x.drop(a, b)
        for _ in range(new):
            tokens = rng.integers(0, 4096, 2).tolist()
            m.cache.extend(1, rows=rows)
            got = logits_of(m, m.forward(example.words(tokens), rows), torch)
            for g, x, t in zip(got, dense, tokens):
                want = x.add([t])
                assert np.linalg.norm(g - want) <= 16 * 2.0 ** -11 * np.linalg.norm(want)
    # the fork still holds all of its tokens
    m.cache.extend(1, rows=example.words([3]))
    whole = seqs[0] + [7]
    got = logits_of(m, m.forward(example.words([7]), example.words([3])), torch)
    assert near(got[0], dense_logits(m, np.array(whole)))
    assert [len(x.k[0]) for x in dense] == m.cache.len.cpu().tolist()[:2]
