"""The weight that cached tokens get from the newest ones (gs_attn_weigh,
include/gs_attn.h) against the formula in 64 bits, with the logarithms of the
sums that the call is given.

Tolerance of a token's sum of weights w:
  sum w (s + 2^-22 (|score| + |lse| + 1)) + (terms / 16 + 32) 2^-24 sum w + 2^-23 |keep mass|
s: a score's error, d 2^-24 scale sum |q k| (f32 sums of d products); the scale,
the difference to lse, the factor log2(e) and the exponential round at 2^-24
of what they are; 16 lanes add their terms and are joined, with the heads.
"""
import ctypes
import math

import numpy as np
import pytest

from test_attn import CHUNKS, ONE, build, starts
from test_kv_cache import NONE, fake, words


def want(c, layer, q, lse, mass, rows, news, keep, scale=None, window=0):
    """(mass, tolerance) in 64 bits: NaN tolerance where a token is not the call's."""
    k = c.k[layer].double().cpu().numpy()
    table, lens = c.table.cpu().numpy(), c.len.cpu().numpy()
    q, lse, out = q.double().cpu().numpy(), lse.double().cpu().numpy(), mass.double().cpu().numpy()
    tol, seen, t = np.full(out.shape, np.nan), set(), 0
    T, H, d = q.shape
    G = H // c.kv
    scale = 1 / math.sqrt(d) if scale is None else scale
    for r, new in zip(rows, news):
        n = int(lens[r]) if 0 <= r < len(lens) else 0
        if r in seen or n == 0:
            t += new
            continue
        seen.add(r)
        add, off = np.zeros(n), np.zeros(n)
        for i in range(new):
            p = n - new + i
            if p >= 0:
                idx = np.arange(max(0, p + 1 - window) if window else 0, p + 1)
                pg, sl = table[r][idx // c.page], idx % c.page
                for h in range(c.kv):
                    kk, qq, ll = k[pg, h, sl], q[t, h * G:(h + 1) * G], lse[t, h * G:(h + 1) * G, None]
                    s = scale * qq @ kk.T
                    w = np.exp(s - ll)
                    ds = d * 2.0 ** -24 * abs(scale) * np.abs(qq) @ np.abs(kk).T
                    add[idx] += w.sum(0)
                    off[idx] += (w * (ds + 2.0 ** -22 * (np.abs(s) + np.abs(ll) + 1))).sum(0)
            t += 1
        old = 0.0 if keep == 0 else keep * out[r, :n]
        out[r, :n] = old + add
        tol[r, :n] = off + (new * H / 16 + 32) * 2.0 ** -24 * add + 2.0 ** -23 * np.abs(old)
    return out, tol


def check(got, ref):
    got = got.double().cpu().numpy()
    out, tol = ref
    mine = ~np.isnan(tol)
    assert np.array_equal(got[~mine], out[~mine], equal_nan=True)
    bad = ~(np.abs(got - out)[mine] <= tol[mine])
    assert not bad.any(), (np.argwhere(bad)[:5], np.abs(got - out)[mine][bad][:5], tol[mine][bad][:5])


def fresh(torch, c, seed=0):
    m = c.mass()
    m.copy_(torch.from_numpy(np.random.default_rng(seed).random(m.shape, dtype=np.float32)))
    return m


@pytest.mark.gpu
@pytest.mark.parametrize("lens,H,kv,d,page,dtype,cache,window", ONE)
def test_single_tokens(gpu, torch, lens, H, kv, d, page, dtype, cache, window):
    rng = np.random.default_rng(d + H + len(lens))
    c = build(gpu, torch, lens, kv, d, page, cache, layers=2)
    rows = rng.permutation(len(lens)).tolist()
    q = (torch.from_numpy(rng.standard_normal((len(rows), H, d), dtype=np.float32)) * 2).to(getattr(torch, dtype)).cuda()
    lse = torch.empty((len(rows), H), device="cuda")
    c.attend(1, q, rows=words(torch, rows), window=window, lse=lse)
    for keep in (1.0, 0.0, 0.5):
        mass = fresh(torch, c)
        ref = want(c, 1, q, lse, mass, rows, [1] * len(rows), keep, window=window)
        again = mass.clone()
        c.weigh(1, q, lse, mass, rows=words(torch, rows), window=window, keep=keep)
        check(mass, ref)
        c.weigh(1, q, lse, again, rows=words(torch, rows), window=window, keep=keep)
        assert torch.equal(mass, again)
    # weights of a softmax: all heads' together
    mass.fill_(math.nan)                                          # (does not count where keep is 0)
    c.weigh(1, q, lse, mass, rows=words(torch, rows), window=window, keep=0.0)
    for r, n in enumerate(lens):
        assert not n or abs(float(mass[r, :n].double().sum()) - H) < 1e-4 * H
        assert bool(mass[r, n:].isnan().all())


@pytest.mark.gpu
@pytest.mark.parametrize("lens,news,H,kv,d,page,dtype,cache,window", CHUNKS)
def test_chunks(gpu, torch, lens, news, H, kv, d, page, dtype, cache, window):
    rng = np.random.default_rng(d + H + sum(news))
    c = build(gpu, torch, lens, kv, d, page, cache)
    rows = rng.permutation(len(lens)).tolist()
    news = [news[r] for r in rows]
    wide = (torch.from_numpy(rng.standard_normal((sum(news), (H + 2) * d), dtype=np.float32)) * 2).to(getattr(torch, dtype)).cuda()
    q = wide[:, d:(H + 1) * d].unflatten(1, (H, d))               # queries inside a wider row
    start, lse = starts(torch, news), torch.empty((sum(news), H), device="cuda")
    c.attend(0, q, rows=words(torch, rows), q_start=start, window=window, lse=lse)
    for keep, max_q in ((1.0, 0), (0.0, max(news)), (-0.25, 1)):  # (the hint only changes the way)
        mass = fresh(torch, c)
        ref = want(c, 0, q, lse, mass, rows, news, keep, window=window)
        c.weigh(0, q, lse, mass, rows=words(torch, rows), q_start=start, window=window, keep=keep, max_q=max_q)
        check(mass, ref)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float16", "float32"])
def test_rows_twice_or_not_there(gpu, torch, dtype):
    """The first sequence of a row counts; rows that are not there, empty ones, sequences without tokens."""
    lens = [100, 33, 0, 260, 70]
    c = build(gpu, torch, lens, 2, 64, 16, "float16")
    rows, news = [3, 0, 3, 5, 2, 1, 0, 4], [2, 1, 1, 1, 2, 40, 3, 0]
    q = torch.randn((sum(news), 4, 64), generator=torch.Generator("cuda").manual_seed(1), device="cuda").to(getattr(torch, dtype))
    lse, start = torch.empty((sum(news), 4), device="cuda"), starts(torch, news)
    c.attend(0, q, rows=words(torch, rows), q_start=start, lse=lse)
    for keep in (1.0, 0.5):
        mass = fresh(torch, c)
        ref = want(c, 0, q, lse, mass, rows, news, keep)
        c.weigh(0, q, lse, mass, rows=words(torch, rows), q_start=start, keep=keep)
        check(mass, ref)
    many = words(torch, [3] * 300)                                # the same row, far from one another
    q = torch.randn((300, 4, 64), device="cuda").to(getattr(torch, dtype))
    lse = torch.empty((300, 4), device="cuda")
    c.attend(0, q, rows=many, lse=lse)
    mass = fresh(torch, c)
    ref = want(c, 0, q, lse, mass, [3] * 300, [1] * 300, 1.0)
    c.weigh(0, q, lse, mass, rows=many)
    check(mass, ref)
    mass = fresh(torch, c)
    c.weigh(0, q[:0], lse[:0], mass, rows=words(torch, [0]), q_start=words(torch, [0, 0]), keep=0.5)       # no tokens
    old = fresh(torch, c)
    assert torch.equal(mass[0, :100], old[0, :100] * 0.5) and torch.equal(mass[0, 100:], old[0, 100:]) and torch.equal(mass[1:], old[1:])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,cache", [("bfloat16", "bfloat16"), ("float32", "float16")])
@pytest.mark.parametrize("news", [[1, 1, 1], [90, 33, 90]])
def test_scales(gpu, torch, dtype, cache, news):
    """Scales given by the caller, also below 0, with scores far apart; a chunk's row named twice."""
    c = build(gpu, torch, [300, 170], 2, 64, 16, cache, seed=4)
    for r, t, f in ((0, 3, 9.0), (0, 120, 12.0), (0, 299, 5.0), (1, 50, 10.0)):
        c.k[0, int(c.table[r, t // 16]), :, t % 16] *= f
    rows = [0, 1, 0]
    q = torch.randn((sum(news), 4, 64), generator=torch.Generator("cuda").manual_seed(8), device="cuda").to(getattr(torch, dtype))
    lse, start = torch.empty((sum(news), 4), device="cuda"), starts(torch, news)
    for scale, window in ((0.3, 0), (-0.05, 0), (1e-6, 0), (-0.2, 40)):
        c.attend(0, q, rows=words(torch, rows), q_start=start, scale=scale, window=window, lse=lse)
        mass = fresh(torch, c)
        ref = want(c, 0, q, lse, mass, rows, news, 1.0, scale=float(np.float32(scale)), window=window)
        c.weigh(0, q, lse, mass, rows=words(torch, rows), q_start=start, scale=scale, window=window, max_q=max(news))
        check(mass, ref)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float16", "float32"])
@pytest.mark.parametrize("news", [3, 120])
def test_queries_that_are_no_numbers(gpu, torch, dtype, news):
    """A token whose query has a NaN makes the weights of what it sees none, and leaves the rest."""
    c = build(gpu, torch, [260, 300], 2, 64, 16, "float16", seed=4)
    q = torch.randn((2 * news, 4, 64), generator=torch.Generator("cuda").manual_seed(8), device="cuda").to(getattr(torch, dtype))
    lse, start = torch.empty((2 * news, 4), device="cuda"), starts(torch, [news, news])
    q[1, 2, 9] = math.nan
    c.attend(0, q, q_start=start, lse=lse)
    assert bool(lse[1, 2].isnan()) and int(lse.isnan().sum()) == 1
    mass = c.mass()
    c.weigh(0, q, lse, mass, q_start=start, max_q=news)
    p = 260 - news + 1
    assert bool(mass[0, :p + 1].isnan().all()) and bool(torch.isfinite(mass[0, p + 1:]).all()) and bool(torch.isfinite(mass[1]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,cache", [("float16", "float16"), ("float32", "float16"), ("float32", "bfloat16")])
@pytest.mark.parametrize("news", [[1, 1], [3, 5], [70, 150]])
def test_keys_that_are_no_numbers(gpu, torch, dtype, cache, news):
    """Keys of infinities and NaN in masked places leave the others' weights;
    one that scores -inf has no weight."""
    lens, H, kv, d = [200, 333], 8, 2, 128
    c = build(gpu, torch, lens, kv, d, 16, cache)
    q = torch.randn((sum(news), H, d), generator=torch.Generator("cuda").manual_seed(3), device="cuda")
    q[:, :, 5] = q[:, :, 5].abs() + 0.1
    q = q.to(getattr(torch, dtype))
    start, lse = starts(torch, news), torch.empty((sum(news), H), device="cuda")
    put = lambda r, t, at, x: c.k[0, int(c.table[r, t // 16]), :, t % 16].__setitem__((slice(None), at), x)  # noqa: E731
    put(0, 20, 5, -math.inf)
    c.attend(0, q, q_start=start, lse=lse, window=180)
    assert bool(torch.isfinite(lse).all())
    mass = fresh(torch, c)
    c.weigh(0, q, lse, mass, q_start=start, window=180, keep=0.0)
    assert bool((mass[0, 20] == 0.0).all()) and bool(torch.isfinite(mass).all())
    # past the window of every token, and the last token's key, which the others do not see
    clean = mass.clone()
    put(1, 2, 7, math.nan)
    put(1, 333 - 1, 9, math.inf)
    got = fresh(torch, c)
    c.weigh(0, q, lse, got, q_start=start, window=180, keep=0.0)
    assert torch.equal(got[0], clean[0])
    assert bool(torch.isfinite(got[1, :332]).all())


@pytest.mark.gpu
def test_layers_and_heads_add_up(gpu, torch):
    c = build(gpu, torch, [300, 41], 2, 64, 16, "bfloat16", layers=3)
    q = torch.randn((3, 2, 8, 64), device="cuda").bfloat16()
    mass = c.mass()
    for layer in range(3):
        lse = torch.empty((2, 8), device="cuda")
        c.attend(layer, q[layer], lse=lse)
        assert c.weigh(layer, q[layer], lse, mass) is mass
    assert torch.allclose(mass.sum(1), torch.full((2,), 24.0, device="cuda"), atol=1e-3)


@pytest.mark.gpu
def test_many_sequences(gpu, torch):
    rng = np.random.default_rng(12)
    lens = rng.integers(0, 90, 700).tolist()
    c = build(gpu, torch, lens, 1, 64, 16, "float16")
    q, lse = torch.randn((700, 2, 64), device="cuda").half(), torch.empty((700, 2), device="cuda")
    c.attend(0, q, lse=lse)
    mass = fresh(torch, c)
    ref = want(c, 0, q, lse, mass, range(700), [1] * 700, 1.0)
    c.weigh(0, q, lse, mass)
    check(mass, ref)


@pytest.mark.gpu
def test_a_far_page_and_wide_weights(gpu, torch):
    """Pages past 2^32 values, and weights in rows whose offset passes 2^32 bytes."""
    pages, kv, page, d = 33000, 8, 64, 256
    c = gpu.KVCache.empty(1, pages, kv, d, 3, 256, page=page, dtype=torch.float16)
    small = build(gpu, torch, [200], kv, d, page, "float16", seed=6)
    far = [pages - 1, 17, pages - 2, 32800]
    for j, p in enumerate(far):
        c.k[0, p] = small.k[0, int(small.table[0, j])]
    c.table[2, :4] = torch.tensor(far, dtype=torch.int32)
    c.len[2] = 200
    q, lse = torch.randn((1, 16, d), device="cuda").half(), torch.empty((1, 16), device="cuda")
    small.attend(0, q, lse=lse)
    mass = torch.empty((3, (1 << 29) + 10), device="cuda")[:, :256]
    mass.zero_()
    got = small.mass()
    small.weigh(0, q, lse, got)
    c.weigh(0, q, lse, mass, rows=words(torch, [2]))
    assert torch.equal(mass[2, :200], got[0, :200]) and not mass[:2].any() and not mass[2, 200:].any()


@pytest.mark.gpu
def test_graph_and_stream(gpu, torch):
    a, b = (build(gpu, torch, [100, 31, 256], 2, 128, 16, "float16", spare=30) for _ in range(2))
    for c in (a, b):
        c.ref[c.table[c.table >= 0].long()] = 1
    q, k = torch.randn((3, 8, 128), device="cuda"), torch.randn((3, 2, 128), device="cuda")
    out, lse = torch.empty_like(q), torch.empty((3, 8), device="cuda")
    ma, mb = fresh(torch, a), fresh(torch, b)
    rows = words(torch, [0, 1, 2])

    def step(c, mass, out, lse):
        c.extend(1)
        c.append(0, k, k)
        c.attend(0, q, out, lse=lse)
        c.weigh(0, q, lse, mass, rows=rows, keep=0.9)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        a.attend(0, q, out)
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            step(a, ma, out, lse)
    eager, elog = torch.empty_like(out), torch.empty_like(lse)
    for i in range(6):
        q.copy_(torch.randn_like(q))
        k.copy_(torch.randn_like(k))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        step(b, mb, eager, elog)
        torch.cuda.synchronize()
        assert torch.equal(lse, elog) and torch.equal(ma, mb)


def test_refusals_without_gpu():
    import gs_sampler as gs
    lib = gs.load_library()
    INV, UNS = gs.GS_ERR_INVALID, gs.GS_ERR_UNSUPPORTED
    c = fake(gs)
    ws = lib.gs_attn_weigh_workspace(c)
    assert ws > 0 and lib.gs_attn_weigh_workspace(fake(gs, d=12)) == 0

    def call(layer=0, b=(1, 1, None, None), cache=c, **kw):
        x = dict(type=1, n_heads=4, q=4096, ld_q=256, lse=4096, mass=4096, ld_mass=64, keep=1.0, scale=0.0, window=0, max_q=0,
                 ws=4096, ws_bytes=ws)
        x.update(kw)
        return lib.gs_attn_weigh(cache, layer, ctypes.byref(gs.GsKVBatch(*b)), ctypes.byref(gs.GsWeighArgs(**x)), None)

    for kw in (dict(layer=1), dict(n_heads=3), dict(n_heads=0), dict(q=None), dict(ld_q=255), dict(ld_q=260), dict(q=4104),
               dict(lse=None), dict(lse=4098), dict(mass=None), dict(mass=4097), dict(ld_mass=63), dict(scale=math.nan),
               dict(ws=None), dict(ws=4104), dict(ws_bytes=ws - 1), dict(keep=math.inf), dict(keep=math.nan), dict(b=(2, 1, None, None)), dict(b=(5, 5, None, None)),
               dict(cache=fake(gs, k=None))):
        assert call(**kw) == INV, kw
    assert call(type=30) == UNS and call(type=2) == UNS and call(ld_mass=(1 << 40) + 1) == UNS
    assert call(b=(65537, 65537, 4096, None)) == UNS
    assert call(b=(0, 0, None, 4096)) == gs.GS_OK
    assert lib.gs_attn_weigh(c, 0, None, None, None) == INV


@pytest.mark.gpu
def test_refusals(gpu, torch):
    c = build(gpu, torch, [40, 3], 2, 64, 16, "float16")
    q, lse, mass = torch.randn((2, 4, 64), device="cuda").half(), torch.empty((2, 4), device="cuda"), c.mass()
    for bad in (None, lse.half(), lse.cpu(), torch.empty((4, 2), device="cuda").t()):
        with pytest.raises(TypeError):
            c.weigh(0, q, bad, mass)
    with pytest.raises(ValueError):
        c.weigh(0, q, lse[:1], mass)
    for bad in (mass.double(), mass.cpu(), mass.t(), mass[0]):
        with pytest.raises((TypeError, ValueError)):
            c.weigh(0, q, lse, bad)
    with pytest.raises(ValueError):
        c.weigh(0, q, lse, mass[:, :40])
    for kw in (dict(window=-1), dict(window=1 << 32)):
        with pytest.raises(ValueError):
            c.weigh(0, q, lse, mass, **kw)
    with pytest.raises(gpu.SamplerError):
        c.weigh(0, q, lse, mass, keep=math.nan)
    with pytest.raises(TypeError):
        c.weigh(0, q.int(), lse, mass)
