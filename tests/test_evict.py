"""Eviction from the paged cache (gs_kv_evict, include/gs_cache.h) against the
model of test_kv_cache.py with an eviction of its own.

Tables, lengths, counts, weights and every value that is only copied have to be
equal.  Turned keys: the bound of test_rope.py for the cache's type.
"""
import ctypes
import math

import numpy as np
import pytest

from test_kv_cache import NONE, Model, fake, make, run, words
from test_rope import bound, frequencies, turned


class Evicting(Model):
    def __init__(self, cache, mass):
        super().__init__(cache)
        self.mass = mass

    def stay(self, r, budget, first, recent):
        n = self.len[r]
        recent = min(recent, budget)
        first = min(first, budget - recent)
        weight = [math.inf if math.isnan(x) else x for x in self.mass[r].tolist()]
        nan = [math.isnan(x) for x in self.mass[r].tolist()]
        middle = sorted(range(first, n - recent), key=lambda t: (not nan[t], -weight[t], t))[:budget - first - recent]
        return list(range(first)) + sorted(middle) + list(range(n - recent, n))

    def evict(self, rows, budgets, first, recent, turn=None):
        """turn(keys [L, h, d], by) -> keys turned back; returns status and the places (page, slot) of turned keys."""
        free, used, status, seen, plans, places = [p for p, r in enumerate(self.ref) if r == 0], 0, [], set(), [], []
        for r, b in zip(rows, budgets):
            if r >= len(self.len) or r in seen:
                status.append(-1)
                continue
            seen.add(r)
            status.append(0)
            n = self.len[r]
            if n <= b:
                continue
            src = self.stay(r, b, first, recent)
            a = next((x for x, y in enumerate(src) if x != y), b)
            new = list(self.table[r])
            fresh = [j for j in range(a // self.P, self.pages(b)) if self.ref[self.table[r][j]] > 1]
            used += len(fresh)
            if fresh and used > len(free):
                status[-1] = -6
                continue
            for j, p in zip(fresh, free[used - len(fresh):used]):
                new[j] = p
            plans.append((r, a, src, new))
        kk, vv = self.k.copy(), self.v.copy()
        refs = list(self.ref)
        for r, a, src, new in plans:
            n, old, b = self.len[r], self.table[r], len(src)
            for t in range(a // self.P * self.P, b):
                y = src[t]
                p, q = old[y // self.P], new[t // self.P]
                k = kk[:, p, :, y % self.P]
                if t >= a and turn is not None:
                    k = turn(k, y - t)
                    places.append((q, t % self.P))
                self.k[:, q, :, t % self.P] = k
                self.v[:, q, :, t % self.P] = vv[:, p, :, y % self.P]
            for j in range(self.pages(n)):
                p = new[j] if j < self.pages(b) else NONE
                if p != old[j]:
                    refs[old[j]] -= 1
                    if p != NONE:
                        refs[p] = 1
                old[j] = p
            self.mass[r, :b], self.mass[r, b:n] = self.mass[r, src], 0.0
            self.len[r] = b
        self.ref = refs
        return status, places

    def check_all(self, cache, mass, places=(), tol=None):
        self.check(cache, places, tol)
        assert np.array_equal(mass.cpu().numpy(), self.mass, equal_nan=True)


def weights(torch, c, seed, steps=None):
    """Weights with many that are alike, in a tensor of the cache's and a copy."""
    m = c.mass()
    x = np.exp(2 * np.random.default_rng(seed).standard_normal(m.shape)).astype(np.float32)
    if steps:
        x = (np.round(x * steps) / steps).astype(np.float32)
    m.copy_(torch.from_numpy(x))
    return m, x.copy()


def build(gpu, torch, lens, held, shared, seed=0, steps=4, **kw):
    c, _ = make(gpu, torch, **kw)
    c.extend(words(torch, lens), rows=words(torch, held))
    if shared:                                                    # row 0 holds the first row's full pages too, row 7 the second's
        c.fork(words(torch, held[:2]), words(torch, [0, 7]))
    mass, x = weights(torch, c, seed, steps)
    return c, mass, Evicting(c, x)


CASES = [  # lengths, budgets, first, recent
    ([100, 33, 16], [50, 32, 16], 4, 8),                          # a half, one token, none
    ([100, 100, 1], [0, 1, 0], 0, 1),                             # all leave; the newest alone; the only one
    ([95, 64, 48], [96, 40, 5], 3, 40),                           # within its budget; no room but for the newest; fewer than those
    ([130, 129, 31], [129, 64, 30], 0, 0),                        # one token: reads and writes overlap
    ([150, 64, 64], [20, 20, 20], 30, 5),                         # the first ones take what the newest leave
    ([170, 17, 32], [48, 16, 16], 16, 16),                        # whole pages
]


@pytest.mark.gpu
@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("layout,rot,d,dtype", [(None, 0, 64, "float16"), ("half", 64, 64, "float16"),
                                                ("interleaved", 32, 80, "bfloat16"), ("half", 40, 80, "float16"),
                                                ("half", 256, 256, "bfloat16"), ("interleaved", 24, 24, "bfloat16"),
                                                ("interleaved", 20, 40, "float16")])
def test_evict(gpu, torch, shared, layout, rot, d, dtype):
    rope, turn, tol = None, None, None
    if layout:
        rope = gpu.Rope(d, rot=rot, layout=layout, base=1000.0, scaling="yarn", factor=4.0, context=64)
        f, _ = frequencies(rot, 1000.0, "yarn", 4.0, 64)

        def turn(k, by):
            y, _ = turned(k, np.full(k.shape[0], -by), f, 1.0, layout)
            return y

        # (largest |a| + |b| of a pair is below 12 for these values)
        tol = bound(np.float64(8.0), np.float64(12.0), dtype)
    for i, (lens, budgets, first, recent) in enumerate(CASES):
        rows = [4, 1, 6]
        c, mass, m = build(gpu, torch, lens, rows, shared, seed=i, pages=90, max_len=176, d=d, dtype=dtype)
        st = run(torch, c.evict, mass, words(torch, budgets), words(torch, rows), first=first, recent=recent, rope=rope, n=3)
        want, places = m.evict(rows, budgets, first, recent, turn)
        assert st == want
        m.check_all(c, mass, places, tol)
        c.extend(3)
        m.extend(range(8), [3] * 8)
        m.check_all(c, mass)
        # again, with one budget for all
        st = run(torch, c.evict, mass, 9, words(torch, rows), first=1, recent=3, rope=rope, n=3)
        want, places = m.evict(rows, [9] * 3, 1, 3, turn)
        assert st == want
        m.check_all(c, mass, places, tol)
        c.evict(mass, 0, words(torch, rows[:2]), first=2, recent=2)        # nothing is to stay
        m.evict(rows[:2], [0, 0], 2, 2)
        m.check_all(c, mass)
        c.evict(mass, 0, words(torch, []))                            # no rows


@pytest.mark.gpu
def test_turned_keys_bound(gpu, torch):
    """Turned keys value by value against the formula's own bound, each by its own way."""
    rope = gpu.Rope(128, base=1e6)
    c, mass, m = build(gpu, torch, [171], [2], False, layers=1, kv=3, d=128, pages=12, max_len=176)
    before = np.concatenate([m.k[0, p] for p in m.table[2][:11]], 1)[:, :171].transpose(1, 0, 2)
    src = np.array(m.stay(2, 70, 5, 9))
    c.evict(mass, 70, words(torch, [2]), first=5, recent=9, rope=rope)
    f, _ = frequencies(128, 1e6)
    want, mag = turned(before[src], np.arange(70) - src, f, 1.0, "half")
    after = torch.cat([c.k[0, p] for p in c.table[2][:5].tolist()], 1)[:, :70].double().cpu().numpy().transpose(1, 0, 2)
    assert (np.abs(after - want) <= bound(want, mag, "float16")).all()


@pytest.mark.gpu
@pytest.mark.parametrize("values", [[0.0], [0.0, -0.0], [1.0, 1.0 + 2 ** -23], [math.nan, math.inf, -math.inf, 0.0, -1.0],
                                    [1e-45, -1e-45, 0.0, 3e38, -3e38], [math.nan]])
def test_equal_and_odd_weights(gpu, torch, values):
    """Ties go to the lowest token; NaN counts more than any number, -0 as 0."""
    c, mass, m = build(gpu, torch, [150, 77], [4, 1], False, pages=30, max_len=160)
    rng = np.random.default_rng(len(values))
    m.mass = np.array(values, np.float32)[rng.integers(0, len(values), m.mass.shape)]
    mass.copy_(torch.from_numpy(m.mass))
    c.evict(mass, words(torch, [60, 20]), words(torch, [4, 1]), first=2, recent=7)
    m.evict([4, 1], [60, 20], 2, 7)
    m.check_all(c, mass)


@pytest.mark.gpu
@pytest.mark.parametrize("n,budget,first,recent", [(5000, 4999, 0, 0), (20011, 5003, 64, 1000), (8192, 1, 0, 0), (4097, 4096, 1, 1),
                                                   (12289, 8200, 0, 4100)])
def test_long_rows(gpu, torch, n, budget, first, recent):
    """More tokens than a step of any kernel, of rows that own their pages and rows that share them."""
    c, mass, m = build(gpu, torch, [n, 3 * n // 4], [4, 1], True, steps=64, layers=1, kv=1, d=8, pages=4 * n // 16 + 40,
                       max_len=n + 16)
    rows, budgets = [1, 4], [min(budget, n // 2), budget]
    st = run(torch, c.evict, mass, words(torch, budgets), words(torch, rows), first=first, recent=recent, n=2)
    want, _ = m.evict(rows, budgets, first, recent)
    assert st == want == [0, 0]
    m.check_all(c, mass)


@pytest.mark.gpu
def test_shortage_and_rows(gpu, torch):
    c, mass, m = build(gpu, torch, [64, 64], [0, 1], False, pages=11)
    c.fork(words(torch, [0, 1]), words(torch, [2, 3]))
    m.fork([0, 1], [2, 3])
    # 3 free pages: the first row takes 3, the next needs 3 more; then a row twice and none
    rows = [2, 3, 2, 12]
    got = run(torch, c.evict, mass, 40, words(torch, rows), first=0, recent=4, n=4)
    want, _ = m.evict(rows, [40] * 4, 0, 4)
    assert got == want == [0, -6, -1, -1]
    m.check_all(c, mass)


@pytest.mark.gpu
def test_many_rows(gpu, torch):
    """More rows than the threads of the bookkeeping, weights in rows of their own stride, rows in any order, some twice."""
    rng = np.random.default_rng(3)
    c, _ = make(gpu, torch, layers=1, pages=9000, kv=1, d=8, rows=1500, max_len=90, page=16)
    lens = rng.integers(0, 90, 1500)
    c.extend(words(torch, lens))
    wide = torch.rand((1500, 131), device="cuda")
    mass = wide[:, 5:5 + 96]
    m = Evicting(c, mass.cpu().numpy().copy())
    edge = wide.clone()
    rows = np.concatenate([rng.permutation(1500)[:1300], rng.integers(0, 1700, 100)])
    budgets = rng.integers(0, 90, 1400)
    got = run(torch, c.evict, mass, words(torch, budgets), words(torch, rows), first=2, recent=10, n=1400)
    want, _ = m.evict(rows.tolist(), budgets.tolist(), 2, 10)
    assert got == want
    m.check_all(c, mass)
    assert torch.equal(wide[:, :5], edge[:, :5]) and torch.equal(wide[:, 101:], edge[:, 101:])


@pytest.mark.gpu
def test_beside_other_calls(gpu, torch):
    rng = np.random.default_rng(12)
    c, mass, m = build(gpu, torch, [30, 40], [0, 1], False, layers=1, pages=60, kv=1, d=16, rows=12, max_len=300)
    for step in range(40):
        n = int(rng.integers(1, 8))
        rows = rng.permutation(12)[:n].tolist()
        if step % 3 == 0:
            adds = rng.integers(0, 70, n).tolist()
            assert run(torch, c.extend, words(torch, adds), n=n, rows=words(torch, rows)) == m.extend(rows, adds)
        elif step % 3 == 1:
            src = [int(x) if x < 12 else NONE for x in rng.integers(0, 13, n)]
            assert run(torch, c.fork, words(torch, src), words(torch, rows), n=n) == m.fork(src, rows)
        else:
            b, first, recent = rng.integers(0, 60, n), int(rng.integers(0, 20)), int(rng.integers(0, 30))
            got = run(torch, c.evict, mass, words(torch, b), words(torch, rows), first=first, recent=recent, n=n)
            assert got == m.evict(rows, b.tolist(), first, recent)[0]
        m.check_all(c, mass)


@pytest.mark.gpu
@pytest.mark.parametrize("shared", [False, True])
def test_weights_go_with_drops_and_frees(gpu, torch, shared):
    """Rows that a drop has shortened, or that a free has emptied for others, are
    cut by the weights that their tokens have."""
    rows, lens = [4, 1, 6], [170, 33, 96]
    c, mass, m = build(gpu, torch, lens, rows, shared, pages=90, max_len=176)
    for start, end in (([20, 0, 96], [90, 33, 200]), ([3, 5, 10], [4, 5, 40]), ([0, 0, 65], [100, 0, 66])):
        st = run(torch, c.drop, words(torch, start), words(torch, end), words(torch, rows), n=3, mass=mass)
        for r, a, b in zip(rows, start, end):
            n = m.len[r]
            a, b = min(a, n), min(max(a, b), n)
            m.mass[r, :n] = np.concatenate([m.mass[r, :a], m.mass[r, b:n], np.zeros(b - a, np.float32)])
        assert st == m.drop(rows, start, end)[0]
        m.check_all(c, mass)
        c.extend(9)
        m.extend(range(8), [9] * 8)
    run(torch, c.evict, mass, 25, words(torch, rows), first=2, recent=5, n=3)
    m.evict(rows, [25] * 3, 2, 5)
    m.check_all(c, mass)
    # one of a row twice, one that is not there, one that finds no page: weights are as before but for the first's
    gone = words(torch, [4, 4, 9])
    st = run(torch, c.drop, words(torch, [1, 2, 3]), words(torch, [9, 9, 9]), gone, n=3, mass=mass)
    n = m.len[4]
    m.mass[4, :n] = np.concatenate([m.mass[4, :1], m.mass[4, 9:n], np.zeros(8, np.float32)])
    assert st == m.drop([4, 4, 9], [1, 2, 3], [9, 9, 9])[0] == [0, -1, -1]
    m.check_all(c, mass)
    c.free(words(torch, [6, 11, 4]), mass=mass)
    m.fork([NONE] * 2, [6, 4])
    m.mass[[6, 4]] = 0.0
    m.check_all(c, mass)


@pytest.mark.gpu
@pytest.mark.parametrize("n,a,b", [(5000, 1, 2), (20011, 3, 7000), (8192, 0, 4096), (4100, 2049, 2050)])
def test_weights_of_long_drops(gpu, torch, n, a, b):
    c, mass, m = build(gpu, torch, [n], [1], False, layers=1, kv=1, d=8, pages=n // 16 + 9, max_len=n + 16)
    c.drop(words(torch, [a]), words(torch, [b]), words(torch, [1]), mass=mass)
    m.mass[1, :n] = np.concatenate([m.mass[1, :a], m.mass[1, b:n], np.zeros(b - a, np.float32)])
    m.drop([1], [a], [b])
    m.check_all(c, mass)


@pytest.mark.gpu
def test_graph_and_stream(gpu, torch):
    """extend and evict captured on a stream of their own, replayed with the
    program's own work between; a larger eager call after the capture, on the
    same stream, takes another workspace."""
    c, mass, m = build(gpu, torch, [60, 50, 9, 70], [0, 1, 2, 3], False, layers=1, pages=64, rows=8, max_len=160)
    rows = words(torch, [0, 1, 2, 3])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        with torch.cuda.graph(graph, stream=s):
            c.extend(5, rows=rows)
            c.evict(mass, 48, rows, first=2, recent=10)
    for step in range(6):
        new = np.random.default_rng(step).random(m.mass.shape).astype(np.float32)
        m.mass = new.copy()
        mass.copy_(torch.from_numpy(new))
        graph.replay()
        torch.cuda.synchronize()
        m.extend([0, 1, 2, 3], [5] * 4)
        m.evict([0, 1, 2, 3], [48] * 4, 2, 10)
        m.check_all(c, mass)
        if step == 2:
            b = words(torch, [40] * 8)
            with torch.cuda.stream(s):
                c.evict(mass, b, words(torch, list(range(8))))
            torch.cuda.synchronize()
            m.evict(range(8), [40] * 8, 0, 0)
            m.check_all(c, mass)


def test_refusals_without_gpu():
    import gs_sampler as gs
    lib = gs.load_library()
    P = ctypes.byref

    def call(c, **kw):
        x = dict(rows=4096, n=1, budget_all=8, mass=4096, ld_mass=64, ws=4096, ws_bytes=1 << 20)
        x.update(kw)
        return lib.gs_kv_evict(c, P(gs.GsKVEvictArgs(**x)), None)

    c = fake(gs)
    assert lib.gs_kv_evict(None, P(gs.GsKVEvictArgs()), None) == gs.GS_ERR_INVALID
    assert lib.gs_kv_evict(c, None, None) == gs.GS_ERR_INVALID
    for kw in (dict(rows=None), dict(mass=None), dict(mass=4098), dict(ld_mass=63), dict(ws=None), dict(ws=4100), dict(ws_bytes=31),
               dict(n=5)):
        assert call(c, **kw) == gs.GS_ERR_INVALID, kw
    assert call(c, ld_mass=(1 << 40) + 1) == gs.GS_ERR_UNSUPPORTED
    assert call(c, n=0) == gs.GS_OK
    assert call(fake(gs, page_size=24)) == gs.GS_ERR_UNSUPPORTED
    assert call(fake(gs, ws=None)) == gs.GS_ERR_INVALID
    assert call(fake(gs, n_layers=65535, n_kv=4096)) == gs.GS_ERR_UNSUPPORTED
    # the workspace: 4 bytes for each token that may stay
    assert lib.gs_kv_evict_workspace(c, 3, 8) == 3 * 8 * 4
    assert lib.gs_kv_evict_workspace(c, 3, 0) == lib.gs_kv_evict_workspace(c, 3, 1000) == 3 * 64 * 4
    assert lib.gs_kv_evict_workspace(c, 5, 8) == 0
    # a budget given as a tensor may be anything
    assert call(c, budget=4096, ws_bytes=255) == gs.GS_ERR_INVALID


def test_refusals_of_weights_without_gpu():
    """Weights of a drop and a free: none, or room for each token."""
    import gs_sampler as gs
    lib, c = gs.load_library(), fake(gs)
    for mass, ld, rc in ((None, 0, gs.GS_OK), (4096, 64, gs.GS_OK), (4098, 64, gs.GS_ERR_INVALID), (4096, 63, gs.GS_ERR_INVALID),
                         (4096, (1 << 40) + 1, gs.GS_ERR_UNSUPPORTED)):
        assert lib.gs_kv_free_mass(c, None, 0, mass, ld, None) == rc
        assert lib.gs_kv_drop_mass(c, None, 0, None, None, None, mass, ld, None, None) == rc
    assert lib.gs_kv_free_mass(c, None, 1, 4096, 64, None) == gs.GS_ERR_INVALID
    assert lib.gs_kv_drop_mass(c, 4096, 1, 4096, None, None, 4096, 64, None, None) == gs.GS_ERR_INVALID


@pytest.mark.gpu
def test_refusals(gpu, torch):
    c, mass, m = build(gpu, torch, [60], [1], False, pages=20, max_len=160)
    rows = words(torch, [1])
    for bad in (mass.double(), mass[0], mass.cpu(), mass.t()):
        with pytest.raises((TypeError, ValueError)):
            c.evict(bad, 8, rows)
    with pytest.raises(ValueError):
        c.evict(mass[:, :159], 8, rows)
    with pytest.raises(ValueError):
        c.evict(mass[:7], 8, rows)
    for kw in (dict(budget=-1), dict(budget=1 << 32), dict(budget=8, first=-1), dict(budget=8, recent=1 << 32)):
        with pytest.raises(ValueError):
            c.evict(mass, kw.pop("budget"), rows, **kw)
    with pytest.raises(ValueError):
        c.evict(mass, words(torch, [8, 8]), rows)
    with pytest.raises(gpu.SamplerError):
        c.evict(mass, 8, rows, rope=gpu.Rope(128))
    closed = gpu.Rope(64)
    closed.close()
    with pytest.raises(ValueError):
        c.evict(mass, 8, rows, rope=closed)
    with pytest.raises(gpu.SamplerError):
        c.evict(mass, 8, words(torch, list(range(9))))            # more rows than the cache has
    torch.cuda.synchronize()
    m.check_all(c, mass)
