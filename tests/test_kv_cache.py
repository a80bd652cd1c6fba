"""The paged cache (include/gs_cache.h) against a model of it in Python lists.

Whole numbers (tables, lengths, counts) have to be equal, and so has every
value that is only copied.  Turned keys: the bound of test_rope.py for the
cache's type.
"""
import ctypes

import numpy as np
import pytest

from test_rope import bound, frequencies, turned

NONE = 0xFFFFFFFF


class Model:
    """The cache's rules, a row and a token at a time.  data[x][page][slot] is
    the token's value in the layer 0, head 0 .. of all layers and heads as one
    array."""

    def __init__(self, cache):
        self.P, self.ld = cache.page, cache.table.shape[1]
        self.table = [[int(p) & NONE for p in r] for r in cache.table.cpu().numpy()]
        self.len = [int(x) for x in cache.len.cpu().numpy()]
        self.ref = [int(x) for x in cache.ref.cpu().numpy()]
        self.k = cache.k.double().cpu().numpy().copy()
        self.v = cache.v.double().cpu().numpy().copy()

    def pages(self, n):
        return -(-n // self.P)

    def lowest(self, m):
        free = [p for p, r in enumerate(self.ref) if r == 0]
        return free[:m]

    def extend(self, rows, adds):
        status, need = [], 0
        free = [p for p, r in enumerate(self.ref) if r == 0]
        for r, add in zip(rows, adds):
            if r >= len(self.len):
                status.append(-1)
                continue
            n, m = self.len[r], self.len[r] + add
            if m > self.ld * self.P:
                status.append(-7)
                continue
            want = self.pages(m) - self.pages(n)
            take = free[need:need + want]
            need += want
            if want and need > len(free):
                status.append(-6)
                continue
            for j, p in enumerate(take):
                self.table[r][self.pages(n) + j] = p
                self.ref[p] = 1
            self.len[r] = m
            status.append(0)
        return status

    def release(self, r):
        for j in range(self.pages(self.len[r])):
            self.ref[self.table[r][j]] -= 1
            self.table[r][j] = NONE
        self.len[r] = 0

    def fork(self, src, dst):
        free, used, status, new, seen = [p for p, r in enumerate(self.ref) if r == 0], 0, [], {}, set()
        for s, d in zip(src, dst):
            if d >= len(self.len) or (s >= len(self.len) and s != NONE) or d in seen:
                status.append(-1)
                if d < len(self.len):
                    seen.add(d)
                continue
            seen.add(d)
            status.append(0)
            if s == d:
                continue
            n = 0 if s == NONE else self.len[s]
            rest = n % self.P
            pages = [] if s == NONE else self.table[s][:n // self.P]
            if rest:
                used += 1
                if used > len(free):
                    status[-1] = -6
                    continue
                p, old = free[used - 1], self.table[s][n // self.P]
                pages = pages + [p]
                self.k[:, p, :, :rest] = self.k[:, old, :, :rest]
                self.v[:, p, :, :rest] = self.v[:, old, :, :rest]
            new[d] = (pages, n)
        for pages, _ in new.values():
            for p in pages:
                self.ref[p] += 1
        for d, (pages, n) in new.items():
            self.release(d)
            self.table[d][:len(pages)] = pages
            self.len[d] = n
        return status

    def drop(self, rows, start, end, turn=None):
        """turn(keys [L, n, h, d], by) -> keys turned back; returns the places
        (page, slot) of turned keys."""
        free, used, status, seen, plans, places = [p for p, r in enumerate(self.ref) if r == 0], 0, [], set(), [], []
        for r, a, b in zip(rows, start, end):
            if r >= len(self.len) or r in seen:
                status.append(-1)
                continue
            seen.add(r)
            status.append(0)
            n = self.len[r]
            a = min(a, n)
            gone = min(max(b, a), n) - a
            if not gone:
                continue
            new = list(self.table[r])
            written = range(a // self.P, self.pages(n - gone))
            shared = [j for j in written if self.ref[self.table[r][j]] > 1]
            used += len(shared)
            if shared and used > len(free):
                status[-1] = -6
                continue
            for j, p in zip(shared, free[used - len(shared):used]):
                new[j] = p
            plans.append((r, a, gone, new))
        kk, vv = self.k.copy(), self.v.copy()
        refs = list(self.ref)
        for r, a, gone, new in plans:
            n, old = self.len[r], self.table[r]
            for t in range(a // self.P * self.P, n - gone):
                y = t + gone if t >= a else t
                p, q = old[y // self.P], new[t // self.P]
                k = kk[:, p, :, y % self.P]
                if t >= a and turn is not None:
                    k = turn(k, gone)
                    places.append((q, t % self.P))
                self.k[:, q, :, t % self.P] = k
                self.v[:, q, :, t % self.P] = vv[:, p, :, y % self.P]
            for j in range(self.pages(n)):
                p = new[j] if j < self.pages(n - gone) else NONE
                if p != old[j]:
                    refs[old[j]] -= 1
                    if p != NONE:
                        refs[p] = 1
                old[j] = p
            self.len[r] = n - gone
        self.ref = refs
        return status, places

    def check(self, cache, places=(), tol=None):
        assert cache.len.cpu().numpy().view(np.uint32).tolist() == self.len
        assert cache.table.cpu().numpy().view(np.uint32).tolist() == self.table
        assert cache.ref.cpu().numpy().tolist() == self.ref
        k, v = cache.k.double().cpu().numpy(), cache.v.double().cpu().numpy()
        assert (v == self.v).all()
        off = k != self.k
        for p, s in places:
            assert (np.abs(k[:, p, :, s] - self.k[:, p, :, s]) <= tol).all()
            off[:, p, :, s] = False
        assert not off.any()
        self.k = k          # (turned keys as the cache rounded them)
        # the rules hold
        held = [0] * len(self.ref)
        for r, n in enumerate(self.len):
            for j in range(self.ld):
                assert (self.table[r][j] != NONE) == (j < self.pages(n))
                if j < self.pages(n):
                    held[self.table[r][j]] += 1
            if n % self.P:
                assert self.ref[self.table[r][n // self.P]] == 1
        assert held == self.ref


def words(torch, x):
    return torch.from_numpy(np.asarray(x, np.uint32).view(np.int32)).cuda()


def make(gpu, torch, layers=2, pages=40, kv=2, d=64, rows=8, max_len=160, page=16, dtype="float16"):
    c = gpu.KVCache.empty(layers, pages, kv, d, rows, max_len, page=page, dtype=getattr(torch, dtype))
    g = torch.Generator(device="cuda")
    g.manual_seed(pages + d)
    for x in (c.k, c.v):
        x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
    return c, Model(c)


def run(torch, fn, *a, n, **kw):
    st = torch.full((n,), 99, dtype=torch.int32, device="cuda")
    fn(*a, status=st, **kw)
    return st.cpu().tolist()


@pytest.mark.gpu
def test_extend(gpu, torch):
    c, m = make(gpu, torch, pages=20)
    for rows, adds in (([0, 3, 5], [1, 16, 17]), ([3], [0]), ([7, 0, 1], [160, 15, 1]), ([2, 9, 4], [161, 1, 33]),
                       ([6, 1, 0, 2], [100, 3, 1, 200])):         # the last: pages run out, and a row too long
        got = run(torch, c.extend, words(torch, adds), n=len(rows), rows=words(torch, rows))
        assert got == m.extend(rows, adds)
        m.check(c)
    c.extend(1)                                                   # every row, one token
    m.extend(range(8), [1] * 8)
    m.check(c)


@pytest.mark.gpu
def test_extend_many_rows(gpu, torch):
    """More rows than the bookkeeping's threads, more pages than one step of
    its search, and free pages that end in the middle."""
    c, m = make(gpu, torch, layers=1, pages=20000, kv=1, d=8, rows=2500, max_len=400, page=16)
    rng = np.random.default_rng(5)
    for _ in range(3):
        rows = rng.permutation(2500)[:2400]
        adds = rng.integers(0, 120, 2400)
        assert run(torch, c.extend, words(torch, adds), n=2400, rows=words(torch, rows)) == m.extend(rows.tolist(), adds.tolist())
        m.check(c)
        gone = rng.permutation(2500)[:700]
        c.free(words(torch, gone))
        for r in gone:
            m.release(int(r))
        m.check(c)


@pytest.mark.gpu
@pytest.mark.parametrize("page,dtype,d", [(16, "float16", 64), (32, "bfloat16", 80), (64, "float16", 8)])
def test_fork_and_free(gpu, torch, page, dtype, d):
    c, m = make(gpu, torch, page=page, dtype=dtype, d=d, pages=40, max_len=5 * page)
    rows, adds = [0, 1, 2], [2 * page + 5, 3 * page, 7]
    c.extend(words(torch, adds), rows=words(torch, rows))
    m.extend(rows, adds)
    for src, dst in (([0, 0, 1, 2], [3, 4, 5, 6]),
                     ([1, 0, 3], [0, 1, 3]),                      # two rows change places, one stays
                     ([NONE, 2, 2], [4, 4, 7]),                   # row 4 emptied; named again: refused
                     ([8, 0, NONE], [1, 9, 2]),                   # rows that are not there
                     ([7, 7, 7, 7, 7, 7, 7], [0, 1, 2, 3, 4, 5, 6])):
        assert run(torch, c.fork, words(torch, src), words(torch, dst), n=len(src)) == m.fork(src, dst)
        m.check(c)
    c.extend(page + 1)
    m.extend(range(8), [page + 1] * 8)
    m.check(c)
    c.free(words(torch, [3, 3, 0, 77]))                           # twice, and a row that is not there
    for r in (3, 0):
        m.release(r)
    m.check(c)
    c.reset()
    assert not c.len.any() and not c.ref.any() and bool((c.table == -1).all())


@pytest.mark.gpu
def test_fork_runs_out(gpu, torch):
    c, m = make(gpu, torch, pages=6)
    c.extend(words(torch, [40, 16]), rows=words(torch, [0, 1]))
    m.extend([0, 1], [40, 16])
    src, dst = [0, 1, 0, 0, 1], [2, 3, 4, 5, 6]                   # two free pages: the third partial page has none
    assert run(torch, c.fork, words(torch, src), words(torch, dst), n=5) == m.fork(src, dst) == [0, 0, 0, -6, 0]
    m.check(c)


DROPS = [  # lengths, from, to of the rows
    ([100, 33, 16], [10, 0, 16], [50, 16, 40]),
    ([100, 100, 1], [0, 99, 0], [100, 1000, 1]),                  # all, the last one, the only one
    ([95, 64, 48], [5, 64, 30], [5, 70, 20]),                     # nothing leaves
    ([130, 129, 31], [1, 17, 3], [2, 18, 31]),                    # one token: reads and writes overlap
    ([150, 64, 64], [16, 16, 0], [48, 32, 16]),                   # whole pages
]


@pytest.mark.gpu
@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("layout,rot,d,dtype", [(None, 0, 64, "float16"), ("half", 64, 64, "float16"),
                                                ("interleaved", 32, 80, "bfloat16"), ("half", 40, 80, "float16"),
                                                ("half", 256, 256, "bfloat16"), ("interleaved", 24, 24, "bfloat16")])
def test_drop(gpu, torch, shared, layout, rot, d, dtype):
    rope, turn, tol = None, None, None
    if layout:
        rope = gpu.Rope(d, rot=rot, layout=layout, base=1000.0, scaling="yarn", factor=4.0, context=64)
        f, _ = frequencies(rot, 1000.0, "yarn", 4.0, 64)

        def turn(k, by):
            y, _ = turned(k, np.full(k.shape[0], -by), f, 1.0, layout)
            return y

    for lens, start, end in DROPS:
        c, m = make(gpu, torch, pages=90, max_len=176, d=d, dtype=dtype)
        c.extend(words(torch, lens), rows=words(torch, [4, 1, 6]))
        m.extend([4, 1, 6], lens)
        if shared:                                                # row 0 holds row 4's full pages too
            c.fork(words(torch, [4, 1]), words(torch, [0, 7]))
            m.fork([4, 1], [0, 7])
        # (largest |a| + |b| of a pair is below 12 for these values)
        tol = bound(np.float64(8.0), np.float64(12.0), dtype) if layout else None
        rows = [4, 1, 6]
        st = run(torch, c.drop, words(torch, start), words(torch, end), words(torch, rows), rope=rope, n=3)
        want, places = m.drop(rows, start, end, turn)
        assert st == want
        m.check(c, places, tol)
        c.extend(3)
        m.extend(range(8), [3] * 8)
        m.check(c)


@pytest.mark.gpu
def test_drop_tight_bound(gpu, torch):
    """Turned keys value by value against the formula's own bound."""
    rope = gpu.Rope(128, base=1e6)
    c, m = make(gpu, torch, layers=1, kv=3, d=128, pages=12, max_len=176)
    c.extend(171, rows=words(torch, [2]))
    m.extend([2], [171])
    before = np.concatenate([m.k[0, p] for p in m.table[2][:11]], 1)[:, :171]
    c.drop(words(torch, [7]), words(torch, [30]), words(torch, [2]), rope=rope)
    f, gain = frequencies(128, 1e6)
    want, mag = turned(before[:, 30:].transpose(1, 0, 2), np.full(141, -23), f, 1.0, "half")
    after = torch.cat([c.k[0, p] for p in c.table[2][:10].tolist()], 1)[:, 7:148].double().cpu().numpy().transpose(1, 0, 2)
    assert (np.abs(after - want) <= bound(want, mag, "float16")).all()


@pytest.mark.gpu
def test_drop_refusals_and_shortage(gpu, torch):
    c, m = make(gpu, torch, pages=11)
    c.extend(words(torch, [64, 64]), rows=words(torch, [0, 1]))
    m.extend([0, 1], [64, 64])
    c.fork(words(torch, [0, 1]), words(torch, [2, 3]))
    m.fork([0, 1], [2, 3])
    # 3 free pages: the first row takes 3 (places 0 to 2), the next needs 3 more; then a row twice and none
    rows, a, b = [2, 3, 2, 12], [3, 3, 0, 0], [20, 20, 9, 9]
    got = run(torch, c.drop, words(torch, a), words(torch, b), words(torch, rows), n=4)
    want, places = m.drop(rows, a, b)
    assert got == want == [0, -6, -1, -1]
    m.check(c)


@pytest.mark.gpu
def test_random_calls(gpu, torch):
    rng = np.random.default_rng(11)
    c, m = make(gpu, torch, layers=1, pages=60, kv=1, d=16, rows=12, max_len=300, page=16)
    for step in range(60):
        n = int(rng.integers(1, 8))
        rows = rng.permutation(12)[:n].tolist()
        kind = rng.integers(0, 4)
        if kind == 0:
            adds = rng.integers(0, 70, n).tolist()
            assert run(torch, c.extend, words(torch, adds), n=n, rows=words(torch, rows)) == m.extend(rows, adds)
        elif kind == 1:
            src = [int(x) if x < 12 else NONE for x in rng.integers(0, 13, n)]
            assert run(torch, c.fork, words(torch, src), words(torch, rows), n=n) == m.fork(src, rows)
        elif kind == 2:
            a = rng.integers(0, 100, n)
            b = a + rng.integers(0, 60, n)
            got = run(torch, c.drop, words(torch, a), words(torch, b), words(torch, rows), n=n)
            assert got == m.drop(rows, a.tolist(), b.tolist())[0]
        else:
            c.free(words(torch, rows[:2]))
            for r in rows[:2]:
                m.release(r)
        m.check(c)


APPENDS = [  # lengths after the call, new tokens of each, heads, kv, d, rot, layout, type, cache, page
    ([1], [1], 4, 2, 64, 64, "half", "float32", "float16", 16),
    ([40, 17, 90], [1, 1, 1], 28, 4, 128, 128, "half", "float32", "float16", 16),
    ([40, 17, 90], [5, 17, 0], 8, 2, 128, 64, "interleaved", "bfloat16", "bfloat16", 32),
    ([70, 33], [70, 3], 3, 1, 80, 40, "half", "float16", "float16", 16),
    ([150, 20], [131, 20], 2, 2, 24, 24, "interleaved", "float32", "bfloat16", 64),
    ([30, 40], [35, 2], 2, 2, 64, 32, "half", "float16", "float16", 16),      # tokens before position 0
]


@pytest.mark.gpu
@pytest.mark.parametrize("lens,news,H,kv,d,rot,layout,dtype,cache,page", APPENDS)
def test_append(gpu, torch, lens, news, H, kv, d, rot, layout, dtype, cache, page):
    rng = np.random.default_rng(sum(lens) + d)
    c, m = make(gpu, torch, layers=3, pages=40, kv=kv, d=d, rows=6, max_len=192, page=page, dtype=cache)
    rows = rng.permutation(6)[:len(lens)].tolist()
    c.extend(words(torch, lens), rows=words(torch, rows))
    m.extend(rows, lens)
    T, td = sum(news), getattr(torch, dtype)
    # queries, keys and values as one product's output has them
    fused = torch.from_numpy(rng.standard_normal((T, (H + 2 * kv) * d), dtype=np.float32)).to(td).cuda()
    q, k, v = (x.unflatten(1, (-1, d)) for x in fused.split([H * d, kv * d, kv * d], 1))
    start = words(torch, np.concatenate([[0], np.cumsum(news)])) if set(news) != {1} else None
    rope = gpu.Rope(d, rot=rot, layout=layout, base=1e5, scaling="linear", factor=2.0)
    f, gain = frequencies(rot, 1e5, "linear", 2.0)
    pos = np.concatenate([np.arange(n - x, n) for n, x in zip(lens, news)])
    outs = {td, getattr(torch, cache)}
    for out_type in outs:
        q_out = torch.full((T, H, d), 9.0, dtype=out_type, device="cuda")
        c.append(1, k, v, q=q, q_out=q_out, rope=rope, rows=words(torch, rows), q_start=start)
        want, mag = turned(q.double().cpu().numpy(), pos, f, gain, layout)
        name = str(out_type).split(".")[1]
        assert (np.abs(q_out.double().cpu().numpy() - want) <= bound(want, mag, name)).all()
    want, mag = turned(k.double().cpu().numpy(), pos, f, gain, layout)
    tol = bound(want, mag, cache)
    vw = v.to(c.v.dtype).double().cpu().numpy()
    got = c.k.double().cpu().numpy()
    t = 0
    for r, n, x in zip(rows, lens, news):
        for i in range(x):
            p = n - x + i
            if p >= 0:
                page_id, slot = m.table[r][p // page], p % page
                assert (np.abs(got[1, page_id, :, slot] - want[t]) <= tol[t]).all()
                m.k[1, page_id, :, slot] = got[1, page_id, :, slot]
                m.v[1, page_id, :, slot] = vw[t]
            t += 1
    m.check(c)                                                    # and nothing else was written
    c.append(2, k, v, rows=words(torch, rows), q_start=start)     # no rotation, no queries
    t = 0
    kw = k.to(c.k.dtype).double().cpu().numpy()
    for r, n, x in zip(rows, lens, news):
        for i in range(x):
            p = n - x + i
            if p >= 0:
                m.k[2, m.table[r][p // page], :, p % page] = kw[t]
                m.v[2, m.table[r][p // page], :, p % page] = vw[t]
            t += 1
    m.check(c)


@pytest.mark.gpu
def test_append_rows_out_of_range(gpu, torch):
    c, m = make(gpu, torch, rows=4)
    c.extend(5, rows=words(torch, [1]))
    m.extend([1], [5])
    k = torch.randn((3, 2, 64), device="cuda")
    q = torch.randn((3, 2, 64), device="cuda")
    q_out = torch.empty_like(q)
    c.append(0, k, k, q=q, q_out=q_out, rope=gpu.Rope(64), rows=words(torch, [4, 3, NONE]))   # not there, empty, not there
    assert bool(torch.isfinite(q_out).all())
    m.check(c)


@pytest.mark.gpu
def test_on_another_stream_and_in_a_graph(gpu, torch):
    """The calls of a decoding step, captured, with the program's own work and
    synchronisations between the replays."""
    c, m = make(gpu, torch, layers=1, pages=64, rows=4, max_len=160)
    rows = words(torch, [0, 1, 2, 3])
    c.extend(words(torch, [3, 15, 16, 30]), rows=rows)
    m.extend([0, 1, 2, 3], [3, 15, 16, 30])
    k = torch.randn((4, 2, 64), device="cuda")
    rope = gpu.Rope(64)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        with torch.cuda.graph(graph, stream=s):
            c.extend(1, rows=rows)
            c.append(0, k, k, rope=rope, rows=rows)
    f, gain = frequencies(64, 10000.0)
    for step in range(20):
        k.copy_(torch.randn((4, 2, 64), device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        m.extend([0, 1, 2, 3], [1] * 4)
        pos = np.array(m.len) - 1
        want, mag = turned(k.double().cpu().numpy(), pos, f, gain, "half")
        tol = bound(want, mag, "float16")
        vw = k.half().double().cpu().numpy()
        got = c.k.double().cpu().numpy()
        for r in range(4):
            p = m.table[r][pos[r] // 16]
            assert (np.abs(got[0, p, :, pos[r] % 16] - want[r]) <= tol[r]).all()
            m.k[0, p, :, pos[r] % 16] = got[0, p, :, pos[r] % 16]
            m.v[0, p, :, pos[r] % 16] = vw[r]
        m.check(c)


def fake(gs, **kw):
    """A cache whose sizes are checked and whose memory is never touched."""
    x = dict(k=4096, v=4096, type=1, n_layers=1, n_pages=8, n_kv=2, page_size=16, d=64, rows=4, ld_table=4, table=4096,
             len=4096, ref=4096, ws=4096)
    x.update(kw)
    return ctypes.byref(gs.GsKVCache(**x))


def test_refusals_without_gpu():
    import gs_sampler as gs
    lib = gs.load_library()
    INV, UNS = gs.GS_ERR_INVALID, gs.GS_ERR_UNSUPPORTED
    for kw, rc in ((dict(k=None), INV), (dict(v=4104), INV), (dict(table=None), INV), (dict(len=None), INV), (dict(ref=None), INV),
                   (dict(ws=None), INV), (dict(n_layers=0), INV), (dict(n_pages=0), INV), (dict(n_kv=0), INV), (dict(rows=0), INV),
                   (dict(ld_table=0), INV), (dict(d=0), INV), (dict(type=0), UNS), (dict(type=2), UNS), (dict(page_size=8), UNS),
                   (dict(page_size=48), UNS), (dict(page_size=2048), UNS), (dict(d=12), UNS), (dict(d=264), UNS),
                   (dict(ld_table=1 << 28), UNS)):
        c = fake(gs, **kw)
        assert lib.gs_kv_extend(c, None, 1, None, 1, None, None) == rc, kw
        assert lib.gs_kv_reset(c, None) == rc, kw
        if "ws" not in kw:
            assert lib.gs_kv_workspace(c) == 0, kw
    c = fake(gs)
    assert lib.gs_kv_workspace(c) > 0
    assert lib.gs_kv_workspace(None) == 0
    assert lib.gs_kv_extend(c, None, 5, None, 1, None, None) == INV       # more rows than there are
    assert lib.gs_kv_fork(c, None, 4096, 1, None, None) == INV
    assert lib.gs_kv_fork(c, 4096, None, 1, None, None) == INV
    assert lib.gs_kv_free(c, None, 1, None) == INV
    assert lib.gs_kv_drop(c, None, 1, 4096, 4096, None, None, None) == INV
    assert lib.gs_kv_drop(c, 4096, 1, None, 4096, None, None, None) == INV
    for f in (lambda: lib.gs_kv_extend(c, None, 0, None, 1, None, None), lambda: lib.gs_kv_fork(c, None, None, 0, None, None),
              lambda: lib.gs_kv_free(c, None, 0, None), lambda: lib.gs_kv_drop(c, None, 0, None, None, None, None, None)):
        assert f() == gs.GS_OK                                            # no rows: nothing to do

    def append(layer=0, b=(1, 1, None, None), **kw):
        x = dict(type=0, k=4096, v=4096, ld_k=128, ld_v=128, q=4096, ld_q=256, q_out=8192, ld_q_out=256, q_out_type=0, n_heads=4)
        x.update(kw)
        return lib.gs_kv_append(c, layer, ctypes.byref(gs.GsKVBatch(*b)), None, ctypes.byref(gs.GsKVNew(**x)), None)

    assert lib.gs_kv_append(c, 0, None, None, None, None) == INV
    assert append(layer=1) == INV
    assert append(b=(2, 1, None, None)) == INV                            # one token each: as many as sequences
    assert append(b=(5, 5, None, None)) == INV                            # more rows than there are
    assert append(b=(0, 3, None, 4096)) == INV
    assert append(b=(65537, 65537, 4096, None)) == UNS
    for kw in (dict(k=None), dict(v=None), dict(ld_k=127), dict(ld_v=64), dict(q_out=None), dict(ld_q=255), dict(ld_q_out=0),
               dict(n_heads=0), dict(k=4097), dict(q_out=8194), dict(q_out=4096, ld_q_out=264)):
        assert append(**kw) == INV, kw
    assert append(type=30) == UNS                                         # not the cache's type
    assert append(type=1, q_out_type=0) == UNS
    assert append(b=(0, 0, None, 4096)) == gs.GS_OK


@pytest.mark.gpu
def test_extend_more_rows_than_a_grid_is_high(gpu, torch):
    c = gpu.KVCache.empty(1, 70010, 1, 8, 70000, 32, page=16, dtype=torch.float16)
    c.extend(3)
    c.extend(2)
    assert (c.len == 5).all() and (c.table[:, 1] == -1).all()
    assert torch.equal(c.table[:, 0], torch.arange(70000, device="cuda", dtype=torch.int32))
    assert c.ref.sum() == 70000 and (c.ref[70000:] == 0).all()
    many = torch.zeros(65536, dtype=torch.int32, device="cuda")
    with pytest.raises(gpu.SamplerError):
        c.free(many)


@pytest.mark.gpu
def test_append_more_heads_than_counted(gpu, torch):
    """Items of a token are counted in 16 bits: more of them are refused."""
    for kv, fits in ((2047, True), (2048, False), (4095, False)):
        c = gpu.KVCache.empty(1, 1, kv, 256, 1, 16, page=16, dtype=torch.float16)
        c.extend(1)
        k = torch.randn((1, kv, 256), device="cuda").half()
        if fits:
            c.append(0, k, k, rope=gpu.Rope(256, layout="half"))
            assert torch.equal(c.v[0, 0, :, 0], k[0]) and torch.equal(c.k[0, 0, :, 0], k[0])
        else:
            with pytest.raises(gpu.SamplerError):
                c.append(0, k, k, rope=gpu.Rope(256, layout="half"))


def test_drop_of_more_streams_than_a_grid_is_wide():
    """Refused before anything is launched: the row's table would be written
    without its tokens having moved."""
    import gs_sampler as gs
    lib = gs.load_library()
    for layers, kv in ((2048, 4096), (65535, 4096), (2049, 4095)):
        c = fake(gs, n_layers=layers, n_kv=kv)
        assert lib.gs_kv_drop(c, 4096, 1, 4096, 4096, None, None, None) == gs.GS_ERR_UNSUPPORTED
        assert lib.gs_kv_drop(c, None, 0, None, None, None, None, None) == gs.GS_OK


def test_a_closed_rotation_is_refused_without_gpu():
    """It has no handle, and no handle means no rotation to the library."""
    import gs_sampler as gs

    class Rows:
        def numel(self):
            return 1

    rope, cache = gs.Rope.__new__(gs.Rope), gs.KVCache.__new__(gs.KVCache)
    rope._h, cache._lib = None, None                              # (nothing can be called)
    for call in (lambda: cache.append(0, None, None, rope=rope), lambda: cache.drop(None, None, Rows(), rope=rope)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.gpu
def test_a_closed_rotation_writes_nothing(gpu, torch):
    c, m = make(gpu, torch)
    rows = words(torch, [1])
    c.extend(40, rows=rows)
    m.extend([1], [40])
    rope = gpu.Rope(64)
    rope.close()
    k = torch.randn((1, 2, 64), device="cuda")
    pos = words(torch, [3])
    for call in (lambda: c.append(0, k, k, rope=rope, rows=rows), lambda: c.drop(pos, words(torch, [9]), rows, rope=rope),
                 lambda: rope.apply(k, pos)):
        with pytest.raises(ValueError):
            call()
    m.check(c)


@pytest.mark.gpu
def test_tensors_of_other_devices_are_refused(gpu, torch):
    c = gpu.KVCache.empty(1, 4, 2, 64, 2, 32, page=16)
    for i in range(5):
        x = [c.k, c.v, c.table, c.len, c.ref]
        x[i] = x[i].cpu()
        with pytest.raises(TypeError):
            gpu.KVCache(*x)
    c.extend(1)
    k, q, pos = torch.randn((2, 2, 64), device="cuda"), torch.randn((2, 4, 64), device="cuda"), words(torch, [0, 1])
    for call in (lambda: c.append(0, k, k.cpu()), lambda: c.append(0, k, k, q=q, q_out=q.cpu()), lambda: c.attend(0, q, q.cpu()),
                 lambda: c.append(0, k, k, rows=pos.cpu()), lambda: c.drop(pos, pos.cpu(), pos),
                 lambda: gpu.Rope(64).apply(k, pos, out=k.cpu()), lambda: gpu.Rope(64).apply(k.cpu(), pos)):
        with pytest.raises(TypeError):
            call()


@pytest.mark.gpu
def test_calls_make_the_tensors_device_current(gpu, torch, monkeypatch):
    """With another device current, which is only said here."""
    c, m = make(gpu, torch)
    rope, k, q, rows = gpu.Rope(64), torch.randn((1, 2, 64), device="cuda"), torch.randn((1, 4, 64), device="cuda"), words(torch, [1])
    out, status, to = torch.empty_like(q), words(torch, [7]), words(torch, [2])
    c.attend(0, q, out, rows=rows)
    on = []

    class Device:
        def __init__(self, device):
            on.append(device)

        def __enter__(self):
            pass

        def __exit__(self, *a):
            pass

    dt = gpu._dtypes()
    monkeypatch.setattr(gpu, "_DT", dt[:3] + (lambda: 1,))
    monkeypatch.setattr(torch.cuda, "device", Device)
    for call in (lambda: c.extend(20, rows=rows), lambda: c.append(0, k, k, q=q, q_out=out, rope=rope, rows=rows),
                 lambda: c.attend(0, q, out, rows=rows), lambda: c.fork(rows, to, status=status), lambda: rope.apply(q, rows, out=out),
                 lambda: c.drop(rows, to, rows, rope=rope), lambda: c.free(to), lambda: c.reset()):
        call()
        assert on == [0]
        on.clear()
    assert status.cpu().tolist() == [0]


@pytest.mark.gpu
def test_a_rotation_of_another_device_is_refused(gpu, torch):
    """A copy of a plan (struct gs_rope of csrc/gs_cache.hpp) that says device 1."""
    class Plan(ctypes.Structure):
        _fields_ = [("d", ctypes.c_uint32), ("rot", ctypes.c_uint32), ("layout", ctypes.c_uint32), ("gain", ctypes.c_float),
                    ("device", ctypes.c_int), ("turns", ctypes.c_void_p)]

    c, m = make(gpu, torch)
    rows = words(torch, [1])
    c.extend(40, rows=rows)
    m.extend([1], [40])
    rope = gpu.Rope(64)
    k, pos = torch.randn((1, 2, 64), device="cuda"), words(torch, [3])
    keep, plan = rope._h, Plan.from_buffer_copy(Plan.from_address(rope._h.value))
    assert (plan.d, plan.rot, plan.layout, plan.device) == (64, 64, 1, torch.cuda.current_device())
    plan.device += 1
    rope._h = ctypes.c_void_p(ctypes.addressof(plan))
    try:
        for call in (lambda: c.append(0, k, k, rope=rope, rows=rows), lambda: c.drop(pos, words(torch, [9]), rows, rope=rope),
                     lambda: rope.apply(k, pos)):
            with pytest.raises(gpu.SamplerError):
                call()
    finally:
        rope._h = keep
    m.check(c)


def test_extend_by_no_number_of_tokens_without_gpu():
    """A C uint32 would take them modulo 2^32."""
    import gs_sampler as gs
    cache = gs.KVCache.__new__(gs.KVCache)
    cache.rows, cache.dev, cache._lib = 1, 0, None                # (nothing can be called)
    for add in (-1, 1 << 32, (1 << 32) + 5):
        with pytest.raises(ValueError):
            cache.extend(add)
