"""Attention over the paged cache (include/gs_attn.h) against the formula in 64
bits, on the values that the cache and the queries hold.

Tolerance of a value: with w_j the weights and v_j the values,
  sum |w_j v_j| (u_p + 2 s + (keys / 32 + 64) 2^-23) + u_o |out|
u_p: the weights' rounding (2^-11 f16, 2^-8 bf16; three parts: 2^-23), s: the
scores' error, d 2^-24 scale sum |q k| at its largest over the keys (f32 sums
of d products); the running sums of keys / 32 blocks and the joins round at
2^-24; u_o: the output's rounding (2^-11, 2^-8, 2^-24), and f16's 2^-25 near 0.
"""
import ctypes
import math

import numpy as np
import pytest

from test_kv_cache import NONE, fake, words

U = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def build(gpu, torch, lens, kv, d, page, dtype, layers=1, seed=0, spare=3):
    """A cache whose rows' pages lie in no order, NaN wherever no token is."""
    rng = np.random.default_rng(seed)
    need = [-(-n // page) for n in lens]
    c = gpu.KVCache.empty(layers, sum(need) + spare, kv, d, len(lens), max(max(lens), 1) + page, page=page,
                          dtype=getattr(torch, dtype))
    order = rng.permutation(sum(need) + spare).astype(np.int32)
    table, at = c.table.cpu().numpy().copy(), 0
    k = np.full((layers, sum(need) + spare, kv, page, d), np.nan, np.float32)
    v = k.copy()
    for r, n in enumerate(need):
        table[r, :n] = order[at:at + n]
        for j in range(n):
            x = min(page, lens[r] - j * page)
            k[:, order[at + j], :, :x] = rng.standard_normal((layers, kv, x, d))
            v[:, order[at + j], :, :x] = rng.standard_normal((layers, kv, x, d)) + 0.5
        at += n
    c.k.copy_(torch.from_numpy(k))
    c.v.copy_(torch.from_numpy(v))
    c.table.copy_(torch.from_numpy(table))
    c.len.copy_(torch.tensor(lens, dtype=torch.int32))
    return c


def want(c, layer, q, rows, news, scale=None, window=0):
    """(out, tolerance) in 64 bits."""
    k, v = c.k[layer].double().cpu().numpy(), c.v[layer].double().cpu().numpy()
    table, lens = c.table.cpu().numpy(), c.len.cpu().numpy()
    name, cache = str(q.dtype).split(".")[1], str(c.k.dtype).split(".")[1]
    u_p = 2.0 ** -23 if name == "float32" else U[cache]
    q = q.double().cpu().numpy()
    T, H, d = q.shape
    G = H // c.kv
    scale = 1 / math.sqrt(d) if scale is None else scale
    out, tol, t = np.zeros_like(q), np.zeros_like(q), 0
    for r, new in zip(rows, news):
        n = int(lens[r]) if 0 <= r < len(lens) else 0
        for i in range(new):
            p = n - new + i
            lo = max(0, p + 1 - window) if window else 0
            if p >= 0:
                idx = np.arange(lo, p + 1)
                pg, sl = table[r][idx // c.page], idx % c.page
                for h in range(c.kv):
                    kk, vv = k[pg, h, sl], v[pg, h, sl]
                    qq = q[t, h * G:(h + 1) * G]
                    s = scale * qq @ kk.T
                    e = np.exp(s - s.max(1, keepdims=True))
                    w = e / e.sum(1, keepdims=True)
                    o = w @ vv
                    ds = d * 2.0 ** -24 * abs(scale) * (np.abs(qq) @ np.abs(kk).T).max(1, keepdims=True)
                    out[t, h * G:(h + 1) * G] = o
                    tol[t, h * G:(h + 1) * G] = (w @ np.abs(vv)) * (u_p + 2 * ds + (len(idx) / 32 + 64) * 2.0 ** -23) \
                        + U[name] * np.abs(o) + (2.0 ** -25 if name == "float16" else 0)
            t += 1
    return out, tol


def check(got, ref):
    got = got.double().cpu().numpy()
    out, tol = ref
    assert np.isfinite(got).all()
    bad = np.abs(got - out) > tol
    assert not bad.any(), (np.argwhere(bad)[:5], float(np.max(np.abs(got - out) / np.maximum(tol, 1e-30))))


def starts(torch, news):
    return words(torch, np.concatenate([[0], np.cumsum(news)]))


ONE = [  # lengths, heads, kv, d, page, type, cache, window
    ([1], 1, 1, 64, 16, "float16", "float16", 0),
    ([4001], 28, 4, 128, 16, "float32", "float16", 0),
    ([1, 2, 15, 16, 17, 31, 32, 33, 127, 128, 129, 0, 1000], 8, 2, 128, 16, "float16", "float16", 0),
    ([1, 31, 64, 65, 300, 0, 777], 32, 8, 128, 64, "bfloat16", "bfloat16", 0),
    ([500, 90, 3], 16, 1, 64, 32, "float16", "float16", 0),
    ([500, 90, 3], 40, 1, 64, 32, "bfloat16", "bfloat16", 0),          # 40 heads on the same keys
    ([777, 1030], 64, 1, 128, 128, "float16", "float16", 0),
    ([500, 90], 7, 7, 80, 16, "float32", "bfloat16", 0),
    ([500, 257], 10, 2, 96, 16, "bfloat16", "bfloat16", 0),
    ([700, 40], 16, 8, 256, 32, "bfloat16", "bfloat16", 0),
    ([700, 40], 24, 1, 256, 32, "float32", "float16", 0),
    ([300, 129], 6, 2, 192, 64, "float16", "float16", 0),
    ([60, 9], 3, 1, 8, 16, "float32", "float16", 0),
    ([20000, 1, 5000], 4, 2, 128, 1024, "bfloat16", "bfloat16", 0),
    ([1000, 130, 128, 5, 0], 8, 2, 128, 16, "float16", "float16", 100),
    ([1000, 130, 128, 5], 8, 2, 64, 16, "float32", "float16", 1),
]


@pytest.mark.gpu
@pytest.mark.parametrize("lens,H,kv,d,page,dtype,cache,window", ONE)
def test_single_tokens(gpu, torch, lens, H, kv, d, page, dtype, cache, window):
    rng = np.random.default_rng(d + H + len(lens))
    c = build(gpu, torch, lens, kv, d, page, cache, layers=2)
    rows = rng.permutation(len(lens)).tolist()
    q = (torch.from_numpy(rng.standard_normal((len(rows), H, d), dtype=np.float32)) * 2).to(getattr(torch, dtype)).cuda()
    out = torch.full_like(q, 99.0)
    c.attend(1, q, out, rows=words(torch, rows), window=window)
    check(out, want(c, 1, q, rows, [1] * len(rows), window=window))
    again = c.attend(1, q, rows=words(torch, rows), window=window)
    assert torch.equal(out, again)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("d,H,kv,news", [(64, 8, 2, 1), (64, 8, 2, 8), (128, 16, 1, 1), (128, 8, 8, 1), (128, 28, 4, 4), (256, 8, 2, 3)])
def test_weights_of_few_rows(gpu, torch, dtype, d, H, kv, news):
    """16-bit queries.  With up to 16 rows per head of keys a bf16 weight reaches
    the values in two parts, off by 2^-16 of itself at most, which twice the
    32-bit form's (keys / 32 + 64) 2^-23 covers; besides, the result's own
    rounding.  Other weights are rounded once."""
    lens = [700, 33, 260]
    c = build(gpu, torch, lens, kv, d, 16, dtype, seed=15)
    q = torch.randn((3 * news, H, d), generator=torch.Generator("cuda").manual_seed(10), device="cuda").to(getattr(torch, dtype))
    got = c.attend(0, q, q_start=starts(torch, [news] * 3), max_q=news)
    out, tol = want(c, 0, q.float(), [0, 1, 2], [news] * 3)
    two = dtype == "bfloat16" and H // kv * news <= 16
    check(got, (out, 3 * tol + U[dtype] * np.abs(out)) if two else want(c, 0, q, [0, 1, 2], [news] * 3))


CHUNKS = [  # lengths, new tokens, heads, kv, d, page, type, cache, window
    ([5], [5], 4, 2, 64, 16, "float16", "float16", 0),
    ([300], [300], 8, 2, 128, 16, "float16", "float16", 0),
    ([1000, 333, 64], [129, 333, 1], 8, 2, 128, 64, "bfloat16", "bfloat16", 0),
    ([700, 50, 20, 0, 9], [3, 0, 25, 4, 9], 6, 3, 128, 16, "float16", "float16", 0),   # tokens before position 0
    ([640, 641], [128, 257], 7, 1, 128, 32, "bfloat16", "bfloat16", 0),
    ([400, 130], [200, 66], 4, 4, 80, 16, "float16", "float16", 0),
    ([400, 130], [200, 66], 5, 1, 256, 32, "bfloat16", "bfloat16", 0),
    ([260, 700, 31], [2, 3, 4], 12, 2, 128, 16, "float32", "float16", 0),
    ([260, 170], [130, 65], 4, 1, 256, 16, "float32", "bfloat16", 0),
    ([600, 170], [130, 65], 6, 2, 96, 64, "float32", "float16", 0),
    ([900, 500, 40], [300, 1, 40], 8, 2, 128, 16, "float16", "float16", 130),
    ([900, 500], [100, 130], 4, 2, 192, 32, "bfloat16", "bfloat16", 64),
    ([2000, 1], [1500, 1], 2, 1, 64, 16, "bfloat16", "bfloat16", 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("lens,news,H,kv,d,page,dtype,cache,window", CHUNKS)
def test_chunks(gpu, torch, lens, news, H, kv, d, page, dtype, cache, window):
    rng = np.random.default_rng(d + H + sum(news))
    c = build(gpu, torch, lens, kv, d, page, cache)
    rows = rng.permutation(len(lens)).tolist()
    lens_of = [lens[r] for r in rows]
    news = [min(n, 10 ** 9) for n in news]
    # the chunks go with the rows
    news = [news[r] for r in rows]
    assert lens_of
    # queries inside a wider row, as a fused product has them
    wide = (torch.from_numpy(rng.standard_normal((sum(news), (H + 2) * d), dtype=np.float32)) * 2).to(getattr(torch, dtype)).cuda()
    q = wide[:, d:(H + 1) * d].unflatten(1, (H, d))
    out = torch.full((sum(news), H, d), 99.0, dtype=q.dtype, device="cuda")
    ref = want(c, 0, q, rows, news, window=window)
    for max_q in (0, max(news), 1):                     # (the hint only changes the way)
        out.fill_(99.0)
        c.attend(0, q, out, rows=words(torch, rows), q_start=starts(torch, news), window=window, max_q=max_q)
        check(out, ref)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,cache", [("float16", "float16"), ("bfloat16", "bfloat16"), ("float32", "float16")])
@pytest.mark.parametrize("news", [[3, 5], [70, 150]])
def test_masked_values_do_not_count(gpu, torch, dtype, cache, news):
    """Infinities and NaN in keys and values that some rows of a chunk see and
    others do not: the others get what they get without them."""
    lens, H, kv, d = [200, 333], 8, 2, 128
    c = build(gpu, torch, lens, kv, d, 16, cache)
    q = (torch.randn((sum(news), H, d), generator=torch.Generator("cuda").manual_seed(3), device="cuda")).to(getattr(torch, dtype))
    start = starts(torch, news)
    clean = c.attend(0, q, q_start=start)
    plant = [(0, lens[0] - 2, "v", math.nan, 3), (0, lens[0] - 1, "k", math.inf, 9), (1, lens[1] - 4, "v", math.inf, 77),
             (1, lens[1] - 2, "v", -math.inf, 127), (1, lens[1] - 2, "k", math.nan, 0)]
    first = {0: lens[0] - 2, 1: lens[1] - 4}
    for r, t, x, value, at in plant:
        getattr(c, x)[0, int(c.table[r, t // 16]), :, t % 16, at] = value
    got = c.attend(0, q, q_start=start)
    t = 0
    for r, new in enumerate(news):
        for i in range(new):
            p = lens[r] - new + i
            if p < first[r]:
                assert torch.equal(got[t], clean[t]), (r, p)
            else:
                assert not bool(torch.isfinite(got[t]).all()), (r, p)
            if r == 1 and first[r] <= p < lens[1] - 2:          # one value of the heads only
                keep = torch.ones(d, dtype=torch.bool, device="cuda")
                keep[77] = False
                assert bool(torch.isfinite(got[t][:, keep]).all()) and not bool(torch.isfinite(got[t][:, 77]).any())
            t += 1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("news", [3, 190])
def test_values_beside_an_infinity(gpu, torch, dtype, d, news):
    """A key whose value has an infinity, in tiles that only some rows see whole,
    and after it in the same tile a key whose score is 2^12 of weight and more
    above all before it: the other values of the rows that see both are the
    formula's."""
    lens, H, kv, page = [333, 262], 4, 2, 16
    c = build(gpu, torch, lens, kv, d, page, dtype, seed=11)
    for r, n in enumerate(lens):
        for key, big in ((n - 70, 0), (n - 40, 1), (n - 12, 0), (n - 3, 1)):
            at = (0, int(c.table[r, key // page]), slice(None), key % page)
            if big:
                c.k[at][:, 0] = 24.0 if key == n - 3 else 12.0
            else:
                c.v[at][:, 7] = math.inf if key == n - 12 else -math.inf
    q = torch.randn((2 * news, H, d), generator=torch.Generator("cuda").manual_seed(6), device="cuda")
    q[:, :, 0] = math.sqrt(d)                           # the large keys score 12 and 24
    q = q.to(getattr(torch, dtype))
    got = c.attend(0, q, q_start=starts(torch, [news, news]), max_q=news).double().cpu().numpy()
    with np.errstate(invalid="ignore"):
        out, tol = want(c, 0, q, [0, 1], [news, news])
        seen = ~np.isfinite(out)
        assert seen.any() and not seen[..., :7].any() and not seen[..., 8:].any()
        assert not np.isfinite(got[seen]).any()
        bad = ~seen & ~(np.abs(got - out) <= tol)
    assert not bad.any(), np.argwhere(bad)[:5]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,cache", [("float32", "float16"), ("float32", "bfloat16"), ("float16", "float16"),
                                         ("bfloat16", "bfloat16")])
@pytest.mark.parametrize("d,H,kv", [(64, 4, 2), (80, 20, 1), (128, 6, 2), (256, 2, 1)])
@pytest.mark.parametrize("news", [1, 5, 90])
def test_infinities_that_all_rows_see(gpu, torch, dtype, cache, d, H, kv, news):
    """A key that scores -inf has the weight 0 and the rest is the formula's; a
    value with an infinity gives infinities of its sign in its place, not NaN.
    Row 1 has a key that scores +inf: no number."""
    lens, page = [420, 300], 16
    c = build(gpu, torch, lens, kv, d, page, cache, seed=13)
    put = lambda x, r, key, at, value: x[0, int(c.table[r, key // page]), :, key % page].__setitem__((slice(None), at), value)  # noqa: E731
    put(c.k, 0, 20, 5, -math.inf)
    put(c.k, 0, 163, 5, -math.inf)
    put(c.v, 0, 40, 9, math.inf)
    put(c.v, 0, 150, 11, -math.inf)
    put(c.k, 1, 10, 5, math.inf)
    q = torch.randn((2 * news, H, d), generator=torch.Generator("cuda").manual_seed(7), device="cuda")
    q[:, :, 5] = q[:, :, 5].abs() + 0.1
    q = q.to(getattr(torch, dtype))
    got = c.attend(0, q, q_start=starts(torch, [news, news])).double().cpu().numpy()
    assert np.isnan(got[news:]).all()
    assert (got[:news, :, 9] == np.inf).all() and (got[:news, :, 11] == -np.inf).all()
    rest = np.delete(np.arange(d), [9, 11])
    # the same without the two keys' part in the scores' error
    small = build(gpu, torch, lens, kv, d, page, cache, seed=13)
    keep = [t for t in range(lens[0]) if t not in (20, 163)]
    k, v = small.k[0].clone(), small.v[0].clone()
    for t, f in enumerate(keep):
        for x, y in ((small.k, k), (small.v, v)):
            x[0, int(small.table[0, t // page]), :, t % page] = y[int(small.table[0, f // page]), :, f % page]
    small.len[0] = len(keep)
    out, tol = want(small, 0, q[:news], [0], [news])
    bad = ~(np.abs(got[:news] - out) <= tol)[..., rest]
    assert not bad.any(), np.argwhere(bad)[:5]


@pytest.mark.gpu
@pytest.mark.parametrize("d,H,kv", [(64, 4, 2), (80, 2, 1), (256, 6, 2)])
@pytest.mark.parametrize("news,dtype", [([200, 40], "bfloat16"), ([3, 30], "float32")])
def test_masked_values_of_other_heads(gpu, torch, d, H, kv, news, dtype):
    """The same for the other sizes of heads, and with a window: values before
    it and after a token leave its row as it is."""
    lens, window = [500, 90], 60
    c = build(gpu, torch, lens, kv, d, 16, "bfloat16", seed=7)
    q = (torch.randn((sum(news), H, d), generator=torch.Generator("cuda").manual_seed(4), device="cuda")).to(getattr(torch, dtype))
    start = starts(torch, news)
    clean = c.attend(0, q, q_start=start, window=window)
    at = {0: 440, 1: 70}
    for r, t in at.items():
        c.v[0, int(c.table[r, t // 16]), :, t % 16, d - 1] = math.nan
        c.v[0, int(c.table[r, t // 16]), :, t % 16, 0] = math.inf
    got = c.attend(0, q, q_start=start, window=window)
    t = 0
    for r, new in enumerate(news):
        for i in range(new):
            p = lens[r] - new + i
            if p < at[r] or p - window >= at[r]:
                assert torch.equal(got[t], clean[t]), (r, p)
            else:
                assert not bool(torch.isfinite(got[t][:, [0, d - 1]]).any()), (r, p)
                assert bool(torch.isfinite(got[t][:, 1:d - 1]).all()), (r, p)
            t += 1


@pytest.mark.gpu
def test_bits_do_not_depend_on_the_call(gpu, torch):
    """A row's result over one run of its keys is the same bits whatever else is
    in the call, as long as both fit one run."""
    c = build(gpu, torch, [90, 60, 128], 2, 128, 16, "float16", seed=9)
    q = torch.randn((3, 8, 128), generator=torch.Generator("cuda").manual_seed(5), device="cuda").half()
    both = c.attend(0, q)
    for r in range(3):
        assert torch.equal(c.attend(0, q[r:r + 1], rows=words(torch, [r]))[0], both[r])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float16", "float32"])
def test_scores_far_apart(gpu, torch, dtype):
    """Weights over the whole range: one key far above the others, and rows
    whose largest score comes first, last and in between."""
    lens = [1500, 700]
    c = build(gpu, torch, lens, 1, 64, 16, "float16", seed=4)
    for r, t, f in ((0, 3, 30.0), (0, 1499, 29.0), (1, 350, 40.0)):
        c.k[0, int(c.table[r, t // 16]), 0, t % 16] *= f
    q = (torch.randn((2, 4, 64), generator=torch.Generator("cuda").manual_seed(8), device="cuda") * 3).to(getattr(torch, dtype))
    check(c.attend(0, q), want(c, 0, q, [0, 1], [1, 1]))
    check(c.attend(0, q, scale=0.5), want(c, 0, q, [0, 1], [1, 1], scale=0.5))
    check(c.attend(0, q, scale=-0.05), want(c, 0, q, [0, 1], [1, 1], scale=-0.05))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("d", [64, 80, 128, 256])
def test_scores_far_apart_in_chunks(gpu, torch, dtype, d):
    """The same for chunks: the largest scores first, in the middle of a tile,
    late after many tiles and last; scales given by the caller, also below 0."""
    lens, news = [1500, 700, 333], [150, 300, 333]
    c = build(gpu, torch, lens, 1, d, 16, dtype, seed=4)
    for r, t, f in ((0, 3, 5.0), (0, 37, 9.0), (0, 1400, 12.0), (0, 1499, 14.0), (1, 450, 10.0), (1, 699, 9.0), (2, 0, 12.0), (2, 300, 6.0)):
        c.k[0, int(c.table[r, t // 16]), 0, t % 16] *= f
    q = (torch.randn((sum(news), 2, d), generator=torch.Generator("cuda").manual_seed(8), device="cuda") * 2).to(getattr(torch, dtype))
    start = starts(torch, news)
    for scale in (0.0, 0.3, -0.05, -1.0 / math.sqrt(d)):
        check(c.attend(0, q, q_start=start, max_q=333, scale=scale),
              want(c, 0, q, [0, 1, 2], news, scale=float(np.float32(scale)) or None))
    check(c.attend(0, q, q_start=start, max_q=333, scale=-0.2, window=70),
          want(c, 0, q, [0, 1, 2], news, scale=float(np.float32(-0.2)), window=70))


@pytest.mark.gpu
def test_queries_of_any_size(gpu, torch):
    """f32 queries beyond f16's range, and small ones."""
    c = build(gpu, torch, [300], 1, 64, 16, "float16", seed=5)
    for size in (1e-30, 1e-6, 1.0, 1e6, 1e30):
        q = torch.randn((1, 3, 64), generator=torch.Generator("cuda").manual_seed(9), device="cuda") * size
        scale = 0.125 / size
        check(c.attend(0, q, scale=scale), want(c, 0, q, [0], [1], scale=float(np.float32(scale))))


@pytest.mark.gpu
def test_rows_without_keys(gpu, torch):
    c = build(gpu, torch, [0, 40], 2, 128, 16, "bfloat16")
    q = torch.randn((4, 4, 128), device="cuda").bfloat16()
    out = c.attend(0, q, rows=words(torch, [0, 1, 2, NONE]))            # empty, a row, and two that are not there
    assert not out[0].any() and out[1].any() and not out[2].any() and not out[3].any()
    c.attend(0, q[:0], q_start=starts(torch, [0, 0]))                   # no tokens


@pytest.mark.gpu
def test_a_far_page(gpu, torch):
    """Pages whose offset passes 2^32 bytes and 2^32 values."""
    pages, kv, page, d = 33000, 8, 64, 256
    c = gpu.KVCache.empty(1, pages, kv, d, 2, 256, page=page, dtype=torch.float16)
    small = build(gpu, torch, [200], kv, d, page, "float16", seed=6)
    far = [pages - 1, 17, pages - 2, 32800]
    for j, p in enumerate(far):
        c.k[0, p] = small.k[0, int(small.table[0, j])]
        c.v[0, p] = small.v[0, int(small.table[0, j])]
    c.table[1, :4] = torch.tensor(far, dtype=torch.int32)
    c.len[1] = 200
    q = torch.randn((1, 16, d), device="cuda").half()
    assert torch.equal(c.attend(0, q, rows=words(torch, [1])), small.attend(0, q))
    q = torch.randn((150, 16, d), device="cuda").half()
    assert torch.equal(c.attend(0, q, rows=words(torch, [1]), q_start=starts(torch, [150])),
                       small.attend(0, q, q_start=starts(torch, [150])))
    c.ref[far[0]] = 1
    k = torch.randn((1, kv, d), device="cuda").half()
    c.len[1] = 64                                                       # the write goes to the far page too
    c.append(0, k, k, rows=words(torch, [1]))
    assert torch.equal(c.k[0, far[0], :, 63], k[0]) and torch.equal(c.v[0, far[0], :, 63], k[0])


@pytest.mark.gpu
def test_more_tiles_than_32_bits_count(gpu, torch):
    """66000 tokens over 2^23: 4.3e9 tiles of 16 rows and 128 keys in one
    sequence.  Keys of zeros weigh all alike, so every row is the values' mean."""
    n, news, page, d = 1 << 23, 66000, 1024, 8
    c = gpu.KVCache.empty(1, n // page, 1, d, 1, n, page=page, dtype=torch.bfloat16)
    c.k.zero_()
    c.v.fill_(1.0)
    c.table[0] = torch.arange(n // page, dtype=torch.int32, device="cuda")
    c.len.fill_(n)
    q = torch.randn((news, 16, d), device="cuda").bfloat16()
    out = torch.full_like(q, 99.0)
    c.attend(0, q, out, q_start=starts(torch, [news]), max_q=1)
    assert bool((out == 1.0).all())


@pytest.mark.gpu
def test_many_sequences(gpu, torch):
    rng = np.random.default_rng(12)
    lens = rng.integers(0, 90, 700).tolist()
    c = build(gpu, torch, lens, 1, 64, 16, "float16")
    q = torch.randn((700, 2, 64), device="cuda").half()
    check(c.attend(0, q), want(c, 0, q, range(700), [1] * 700))


@pytest.mark.gpu
def test_streams_and_graph(gpu, torch):
    """A captured step (room, write, attention) replayed with other work and
    synchronisations between, each against the eager call on a second cache."""
    lens, H, kv, d = [100, 31, 256], 8, 2, 128
    a, b = (build(gpu, torch, lens, kv, d, 16, "float16", spare=30) for _ in range(2))
    for c in (a, b):
        held = c.table[c.table >= 0].long()
        c.ref[held] = 1
    q, k = torch.randn((3, H, d), device="cuda"), torch.randn((3, kv, d), device="cuda")
    out, q_out = torch.empty_like(q), torch.empty_like(q)
    rope = gpu.Rope(d)
    s = torch.cuda.Stream()

    def step(c, out, q_out):
        c.extend(1)
        c.append(0, k, k, q=q, q_out=q_out, rope=rope)
        c.attend(0, q_out, out)

    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        a.attend(0, q, out)                             # (the workspace of this stream)
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            step(a, out, q_out)
    eager, eq = torch.empty_like(out), torch.empty_like(out)
    for i in range(12):
        q.copy_(torch.randn_like(q))
        k.copy_(torch.randn_like(k))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        step(b, eager, eq)
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.equal(a.len, b.len) and torch.equal(a.table, b.table)


def test_refusals_without_gpu():
    import gs_sampler as gs
    lib = gs.load_library()
    INV, UNS = gs.GS_ERR_INVALID, gs.GS_ERR_UNSUPPORTED
    c = fake(gs)
    ws = lib.gs_attn_workspace(c, 4)
    assert ws > 0 and lib.gs_attn_workspace(c, 5) == 0 and lib.gs_attn_workspace(c, 0) == 0
    assert lib.gs_attn_workspace(fake(gs, d=12), 4) == 0

    def call(layer=0, b=(1, 1, None, None), cache=c, **kw):
        x = dict(type=1, n_heads=4, q=4096, ld_q=256, out=8192, ld_out=256, scale=0.0, window=0, max_q=0, ws=4096, ws_bytes=ws)
        x.update(kw)
        return lib.gs_attn(cache, layer, ctypes.byref(gs.GsKVBatch(*b)), ctypes.byref(gs.GsAttnArgs(**x)), None)

    for kw in (dict(layer=1), dict(n_heads=3), dict(n_heads=0), dict(q=None), dict(out=None), dict(out=4096), dict(ld_q=255),
               dict(ld_q=260), dict(ld_out=200), dict(ld_out=257), dict(q=4104), dict(out=8200), dict(ws=None), dict(ws=4104),
               dict(ws_bytes=ws - 1), dict(scale=math.nan), dict(scale=math.inf), dict(b=(2, 1, None, None)),
               dict(b=(5, 5, None, None)), dict(b=(0, 2, None, 4096)), dict(cache=fake(gs, k=None))):
        assert call(**kw) == INV, kw
    assert call(type=30) == UNS and call(type=2) == UNS
    assert call(b=(65537, 65537, 4096, None)) == UNS
    assert call(b=(0, 0, None, 4096)) == gs.GS_OK
    assert lib.gs_attn(c, 0, None, None, None) == INV


@pytest.mark.gpu
def test_memory_of_another_stream(gpu, torch):
    """What a call on a stream of its own allocates does not come from memory
    that the stream of the moment has freed, where work may still use it."""
    c = build(gpu, torch, [100, 31], 2, 64, 16, "float16", seed=9)
    q = torch.randn((2, 4, 64), device="cuda")
    here = c.attend(0, q)
    n = next(iter(c._attn_ws.values())).numel()
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    freed = [torch.empty(n, dtype=torch.uint8, device="cuda"), torch.empty_like(q)]
    places = [x.data_ptr() for x in freed]
    del freed
    got = c.attend(0, q, stream=other)
    torch.cuda.synchronize()
    assert c._attn_ws[other.cuda_stream, 4].data_ptr() != places[0] and got.data_ptr() != places[1]
    assert torch.equal(got, here)


@pytest.mark.gpu
def test_one_workspace_of_a_stream(gpu, torch):
    """Calls of other numbers of heads share it; another stream has its own."""
    c = build(gpu, torch, [100, 31], 2, 64, 16, "float16", seed=9)
    q = torch.randn((2, 8, 64), device="cuda")
    for heads in (2, 8, 4):
        check(c.attend(0, q[:, :heads]), want(c, 0, q[:, :heads], [0, 1], [1, 1]))
    assert len({w.data_ptr() for w in c._attn_ws.values()}) == 1
    here = c.attend(0, q)
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    got = c.attend(0, q, stream=other)
    torch.cuda.synchronize()
    assert torch.equal(got, here) and len({w.data_ptr() for w in c._attn_ws.values()}) == 2


def test_a_window_that_is_no_number_of_positions_without_gpu():
    """A C uint32 would take it modulo 2^32: 2^32 + 5 as 5, -1 as none."""
    import gs_sampler as gs
    cache = gs.KVCache.__new__(gs.KVCache)
    cache.dev = cache.d = 0                                             # (nothing can be called)
    for window in (-1, (1 << 32) + 5):
        with pytest.raises(ValueError):
            cache.attend(0, None, window=window)
