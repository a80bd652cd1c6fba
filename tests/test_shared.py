"""Attention of families of rows that begin with the same pages (gs_attn_shared,
include/gs_attn.h), and the logarithms of the softmax's sums, against the
formula in 64 bits; the bounds of test_attn.py for the values.

Tolerance of a logarithm of a sum: 2 s + (keys / 32 + 64) 2^-23 + 2^-22 (|lse| +
largest |score|): s the scores' error as in test_attn.py, each off by at most
that; the sum's relative error is the logarithm's own; the factor from powers
of two to e, on the scores and back, and the logarithm itself round four times
at 2^-24 of what they are.
"""
import ctypes
import math

import numpy as np
import pytest

from test_attn import U, build, check, starts, want
from test_kv_cache import NONE, fake, words


def want_lse(c, layer, q, rows, news, scale=None, window=0):
    k = c.k[layer].double().cpu().numpy()
    table, lens = c.table.cpu().numpy(), c.len.cpu().numpy()
    q = q.double().cpu().numpy()
    T, H, d = q.shape
    G = H // c.kv
    scale = 1 / math.sqrt(d) if scale is None else scale
    out, tol, t = np.full((T, H), -np.inf), np.zeros((T, H)), 0
    for r, new in zip(rows, news):
        n = int(lens[r]) if 0 <= r < len(lens) else 0
        for i in range(new):
            p = n - new + i
            if p >= 0:
                idx = np.arange(max(0, p + 1 - window) if window else 0, p + 1)
                pg, sl = table[r][idx // c.page], idx % c.page
                for h in range(c.kv):
                    qq = q[t, h * G:(h + 1) * G]
                    s = scale * qq @ k[pg, h, sl].T
                    m = s.max(1)
                    x = m + np.log(np.exp(s - m[:, None]).sum(1))
                    ds = d * 2.0 ** -24 * abs(scale) * (np.abs(qq) @ np.abs(k[pg, h, sl]).T).max(1)
                    out[t, h * G:(h + 1) * G] = x
                    tol[t, h * G:(h + 1) * G] = 2 * ds + (len(idx) / 32 + 64) * 2.0 ** -23 + 2.0 ** -22 * (np.abs(x) + np.abs(s).max(1))
            t += 1
    return out, tol


def check_lse(got, ref):
    got = got.double().cpu().numpy()
    out, tol = ref
    none = np.isneginf(out)
    assert (np.isneginf(got) == none).all()
    assert (np.abs(got[~none] - out[~none]) <= tol[~none]).all()


def family(gpu, torch, prompts, each, adds, kv, d, page, dtype, layers=1, seed=0):
    """A cache whose rows len(prompts) .. hold copies of the prompts (each[i] of
    prompt i) and adds[..] tokens of their own; NaN wherever no token is."""
    kids = sum(each)
    spare = kids * (2 + (max(adds) + page) // page) + 2
    c = build(gpu, torch, prompts + [0] * kids, kv, d, page, dtype, layers=layers, seed=seed, spare=spare)
    wide = torch.full((c.rows, (max(prompts) + max(adds)) // page + 3), -1, dtype=torch.int32, device="cuda")
    wide[:, :c.table.shape[1]] = c.table[:, :wide.shape[1]]
    c.ref.zero_()
    c.ref[c.table[c.table >= 0].long()] = 1
    c = gpu.KVCache(c.k, c.v, wide, c.len, c.ref)
    m = len(prompts)
    c.fork(words(torch, np.repeat(np.arange(m), each)), words(torch, np.arange(m, m + kids)))
    c.free(words(torch, np.arange(m)))
    rows = words(torch, np.arange(m, m + kids))
    c.extend(words(torch, adds), rows=rows)
    if sum(adds):
        g = torch.Generator("cuda").manual_seed(seed)
        for layer in range(layers):
            k, v = (torch.randn((sum(adds), kv, d), generator=g, device="cuda") for _ in range(2))
            c.append(layer, k, v + 0.5, rows=rows, q_start=starts(torch, adds))
    return c


CASES = [  # prompts, rows of each, own tokens, new tokens, heads, kv, d, page, type, cache, window
    ([37], [3], [1, 2, 17], [1, 1, 1], 4, 2, 64, 16, "float16", "float16", 0),
    ([601], [4], [1, 40, 7, 20], [1] * 4, 28, 4, 128, 16, "float32", "float16", 0),
    ([300, 17, 640], [2, 3, 1], [5, 1, 90, 3, 16, 33], [1] * 6, 8, 2, 128, 64, "bfloat16", "bfloat16", 0),
    ([1000], [40], list(range(1, 41)), [1] * 40, 8, 1, 64, 32, "float16", "float16", 0),
    ([1500, 800], [9, 20], [3 + i for i in range(29)], [1] * 29, 16, 2, 128, 16, "bfloat16", "bfloat16", 0),
    ([500], [6], [8, 9, 30, 100, 5, 61], [8, 1, 0, 33, 5, 2], 10, 2, 96, 16, "float16", "float16", 0),
    ([700], [5], [70, 1, 9, 130, 64], [70, 1, 3, 129, 8], 6, 3, 128, 16, "float16", "float16", 0),
    ([700], [3], [20, 1, 9], [3, 1, 2], 20, 1, 256, 32, "bfloat16", "bfloat16", 0),
    ([333], [5], [4, 1, 9, 2, 2], [2, 1, 1, 2, 1], 10, 2, 192, 16, "float32", "bfloat16", 0),
    ([700], [4], [200, 1, 9, 64], [150, 1, 3, 2], 4, 2, 80, 16, "float32", "float16", 0),
    ([900], [6], [30, 200, 1, 99, 100, 101], [1] * 6, 8, 2, 128, 16, "float16", "float16", 100),   # windows that end in, at and past the prompt
    ([900], [30], [1 + 9 * i for i in range(30)], [1] * 30, 8, 2, 64, 16, "bfloat16", "bfloat16", 128),
    ([900], [6], [30, 200, 8, 99, 100, 101], [5, 8, 8, 1, 1, 40], 8, 2, 256, 64, "float16", "float16", 500),
    ([260], [4], [10, 300, 3, 4], [1] * 4, 3, 1, 8, 16, "float32", "float16", 64),
    ([5], [4], [10, 3, 3, 4], [1] * 4, 4, 2, 128, 16, "bfloat16", "bfloat16", 0),                   # nothing in common: less than a page
    ([64], [40], [1] * 40, [1] * 40, 4, 2, 128, 16, "float16", "float16", 1),                       # a token sees itself alone
]


@pytest.mark.gpu
@pytest.mark.parametrize("prompts,each,adds,news,H,kv,d,page,dtype,cache,window", CASES)
def test_families(gpu, torch, prompts, each, adds, news, H, kv, d, page, dtype, cache, window):
    rng = np.random.default_rng(d + H)
    c = family(gpu, torch, prompts, each, adds, kv, d, page, cache, layers=2)
    ends = np.cumsum([0] + each)
    # rows in any order within their families
    rows = np.concatenate([len(prompts) + a + rng.permutation(b - a) for a, b in zip(ends, ends[1:])]).tolist()
    news = [news[r - len(prompts)] for r in rows]
    wide = (torch.from_numpy(rng.standard_normal((sum(news), (H + 2) * d), dtype=np.float32)) * 2).to(getattr(torch, dtype)).cuda()
    q = wide[:, d:(H + 1) * d].unflatten(1, (H, d))               # queries inside a wider row
    start = None if set(news) == {1} else starts(torch, news)
    ref, ref_lse = (f(c, 1, q, rows, news, window=window) for f in (want, want_lse))
    whole = words(torch, [0, len(rows)])                          # (rows of several prompts as one family have less in common)
    for families in (words(torch, ends), whole, words(torch, np.arange(len(rows) + 1))):
        out = torch.full((sum(news), H, d), 99.0, dtype=q.dtype, device="cuda")
        lse = torch.full((sum(news), H), 99.0, device="cuda")
        c.attend_shared(1, q, families, out, rows=words(torch, rows), q_start=start, window=window, max_q=max(news), lse=lse)
        check(out, ref)
        check_lse(lse, ref_lse)
        again = c.attend_shared(1, q, families, rows=words(torch, rows), q_start=start, window=window)
        assert torch.equal(out, again)
    lse.fill_(99.0)
    c.attend(1, q, out, rows=words(torch, rows), q_start=start, window=window, lse=lse)
    check(out, ref)
    check_lse(lse, ref_lse)


WEIGHTS = [  # prompts, rows of each, own tokens, new tokens, heads, kv, d, window: of the rows kernel alone, of the second alone, of both
    ([300], [2], [5, 40], [1, 1], 8, 2, 128, 0),
    ([300], [2], [5, 40], [2, 3], 8, 1, 64, 0),
    ([300], [2], [5, 40], [1, 1], 8, 2, 256, 0),
    ([600, 40], [9, 6], [1 + 3 * i for i in range(15)], [1] * 15, 16, 2, 128, 0),
    ([600], [8], [1 + 3 * i for i in range(8)], [1, 1, 1, 2, 3, 4, 5, 6], 16, 2, 64, 200),
    ([600], [8], [9 + 3 * i for i in range(8)], [1, 1, 1, 2, 3, 4, 5, 9], 12, 2, 256, 0),
    ([300, 77], [20, 13], [1 + i % 9 for i in range(33)], [1] * 33, 16, 8, 128, 0),
    ([300, 77], [20, 13], [1 + i % 9 for i in range(33)], [1] * 33, 16, 8, 256, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("prompts,each,adds,news,H,kv,d,window", WEIGHTS)
def test_weights_reach_the_values_in_parts(gpu, torch, dtype, prompts, each, adds, news, H, kv, d, window):
    """16-bit queries and keys of small whole numbers, whose products have no
    rounding.  With W the sum of the weights times the values' magnitudes, the
    result is off by no more than
      W 2^-22                         a weight's parts, two of f16, three of bf16,
      W 2^-21 (1 + largest |score|)   the exponent, the reference it is taken
                                      from and the exponential, of up to three
                                      joined sums: four roundings of 2^-24 of
                                      log2(e) |score| and two of 2^-23,
      W (keys / 32 + 64) 2^-23        sums in 32 bits, as elsewhere,
    and its own rounding.  A single rounding of a weight is up to 2^-11 (bf16:
    2^-8) of it."""
    c = family(gpu, torch, prompts, each, adds, kv, d, 16, dtype, seed=6)
    g = torch.Generator("cuda").manual_seed(12)
    t = getattr(torch, dtype)
    c.k.copy_(torch.where(c.k.isnan(), c.k, torch.randint(-1, 2, c.k.shape, generator=g, device="cuda").to(t)))
    c.v.copy_(torch.where(c.v.isnan(), c.v, torch.randn(c.v.shape, generator=g, device="cuda").to(t)))    # (sums near 0, which round little)
    rows = list(range(len(prompts), len(prompts) + sum(each)))
    q = torch.randint(-1, 2, (sum(news), H, d), generator=g, device="cuda").to(t)
    families = words(torch, np.cumsum([0] + each))
    scale = 1 / 16
    got = c.attend_shared(0, q, families, rows=words(torch, rows), q_start=starts(torch, news), max_q=max(news), window=window, scale=scale)
    out = want(c, 0, q.float(), rows, news, scale=scale, window=window)[0]
    c.v.abs_()
    W = want(c, 0, q.float(), rows, news, scale=scale, window=window)[0]
    top, keys = scale * d, int(c.len.max())                       # (a score is d products of -1, 0 and 1)
    tol = W * (2.0 ** -22 + 2.0 ** -21 * (1 + top) + (keys / 32 + 64) * 2.0 ** -23)
    check(got, (out, tol + U[dtype] * (np.abs(out) + tol) + (2.0 ** -25 if dtype == "float16" else 0)))


def many(n, each):
    """n rows' own and new tokens, each as many new ones as `each` says in turn."""
    news = [each[i % len(each)] for i in range(n)]
    return [x + i % 21 for i, x in enumerate(news)], news


BOTH = [  # prompts, rows of each, new tokens in turn, heads, kv, d, page, type, window: more heads of keys of sequences than the second kernel has runs
    ([300, 77], [25, 11], [1], 16, 8, 128, 16, "float16", 0),
    ([300, 77], [25, 11], [1], 16, 8, 128, 16, "bfloat16", 0),
    ([300], [33], [1], 24, 8, 128, 32, "bfloat16", 150),           # windows that end inside the common pages,
    ([300], [33], [1], 24, 8, 96, 16, "float16", 31),              # and past them for some rows
    ([200], [34], [1], 8, 8, 192, 16, "bfloat16", 190),
    ([200, 120], [20, 14], [1], 16, 8, 256, 16, "bfloat16", 0),
    ([200, 120], [20, 14], [1], 16, 8, 256, 16, "float16", 180),
    ([200], [36], [1], 40, 8, 80, 16, "float16", 0),
    ([200], [34], [5], 32, 8, 128, 16, "bfloat16", 0),             # own rows of two tiles
    ([200], [34], [5], 32, 8, 64, 16, "float16", 120),
    ([200], [34], [7, 2, 0, 8], 32, 8, 128, 16, "float16", 0),
    ([150], [34], [1, 1, 1, 40, 3], 16, 8, 128, 16, "bfloat16", 0),    # own keys of both kernels
    ([150], [34], [1, 1, 1, 40, 3], 16, 8, 64, 16, "bfloat16", 100),
    ([150], [34], [1, 20, 1, 9, 3], 16, 8, 256, 16, "float16", 0),
    ([150], [34], [1, 20, 1, 17, 3], 16, 8, 192, 32, "bfloat16", 50),
]


@pytest.mark.gpu
@pytest.mark.parametrize("prompts,each,turn,H,kv,d,page,dtype,window", BOTH)
def test_both_kernels(gpu, torch, prompts, each, turn, H, kv, d, page, dtype, window):
    """Calls whose jobs of few rows go to one kernel and whose others go to a
    second, of other parts, lifts and rows in a unit."""
    n = sum(each)
    assert n * kv > 256 and n * H // kv > 16
    adds, news = many(n, turn)
    c = family(gpu, torch, prompts, each, adds, kv, d, page, dtype, layers=2, seed=2)
    rows = list(range(len(prompts), len(prompts) + n))
    q = torch.randn((sum(news), H, d), generator=torch.Generator("cuda").manual_seed(3), device="cuda").to(getattr(torch, dtype)) * 2
    start = None if set(news) == {1} else starts(torch, news)
    ref, ref_lse = (f(c, 1, q, rows, news, window=window) for f in (want, want_lse))
    ends = np.cumsum([0] + each).tolist()
    outs = []
    for families, most in ((ends, max(news)), (ends, 0), ([0, n], max(news)), ([3, n - 2], max(news)), (ends, 1)):   # (1: less than the most)
        out = torch.full((sum(news), H, d), 99.0, dtype=q.dtype, device="cuda")
        lse = torch.full((sum(news), H), 99.0, device="cuda")
        c.attend_shared(1, q, words(torch, families), out, rows=words(torch, rows), q_start=start, window=window, max_q=most, lse=lse)
        check(out, ref)
        check_lse(lse, ref_lse)
        outs.append(out)
    again = c.attend_shared(1, q, words(torch, ends), rows=words(torch, rows), q_start=start, window=window, max_q=max(news))
    assert torch.equal(outs[0], again)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,cache", [("float16", "float16"), ("float32", "bfloat16")])
def test_rows_that_have_nothing_to_share(gpu, torch, dtype, cache):
    """Families of rows of other prompts, of empty rows, rows that are not there,
    sequences without tokens and with more than their rows hold, and sequences
    of no family."""
    c = family(gpu, torch, [300, 200], [3, 3], [5, 9, 1, 30, 2, 8], 2, 64, 16, cache)
    rows = [2, 5, 3, 0, 8, 4, 6, 2, 7]
    news = [1, 2, 3, 2, 1, 0, 8, 6, 1]
    H = 4
    q = torch.randn((sum(news), H, 64), generator=torch.Generator("cuda").manual_seed(1), device="cuda").to(getattr(torch, dtype))
    ref = want(c, 0, q, rows, news)
    ref_lse = want_lse(c, 0, q, rows, news)
    c.len[5] = 1                                                  # two new tokens: one lies before position 0
    ref = want(c, 0, q, rows, news)
    ref_lse = want_lse(c, 0, q, rows, news)
    for families in ([0, 9], [2, 5, 8], [0, 3, 3, 9], [9, 9], [0, 0], [0, 2, 200]):
        out = torch.full_like(q, 99.0)
        lse = torch.full((sum(news), H), 99.0, device="cuda")
        c.attend_shared(0, q, words(torch, families), out, rows=words(torch, rows), q_start=starts(torch, news), lse=lse)
        check(out, ref)
        check_lse(lse, ref_lse)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,cache,each", [("float16", "float16", 3), ("bfloat16", "bfloat16", 30), ("float32", "float16", 9)])
def test_scales(gpu, torch, dtype, cache, each):
    """Scales given by the caller, also below 0, with scores far apart."""
    c = family(gpu, torch, [300], [each], [1 + 3 * i for i in range(each)], 2, 64, 16, cache, seed=4)
    rows = list(range(1, each + 1))
    for t, f in ((3, 9.0), (120, 12.0)):
        c.k[0, int(c.table[1, t // 16]), :, t % 16] *= f
    q = torch.randn((each, 4, 64), generator=torch.Generator("cuda").manual_seed(8), device="cuda").to(getattr(torch, dtype))
    for scale, window in ((0.3, 0), (-0.05, 0), (-0.2, 200)):
        lse = torch.empty((each, 4), device="cuda")
        out = c.attend_shared(0, q, words(torch, [0, each]), rows=words(torch, rows), scale=scale, window=window, lse=lse)
        check(out, want(c, 0, q, rows, [1] * each, scale=float(np.float32(scale)), window=window))
        check_lse(lse, want_lse(c, 0, q, rows, [1] * each, scale=float(np.float32(scale)), window=window))


@pytest.mark.gpu
def test_tokens_of_no_sequence_stay(gpu, torch):
    c = family(gpu, torch, [100], [2], [5, 9], 2, 64, 16, "float16")
    q = torch.randn((7, 4, 64), device="cuda").half()
    out, lse = torch.full_like(q, 99.0), torch.full((7, 4), 99.0, device="cuda")
    c.attend_shared(0, q, words(torch, [0, 2]), out, rows=words(torch, [1, 2]), q_start=words(torch, [0, 2, 5]), lse=lse)
    check(out[:5], want(c, 0, q[:5], [1, 2], [2, 3]))
    assert bool((out[5:] == 99.0).all()) and bool((lse[5:] == 99.0).all())
    c.attend_shared(0, q[:0], words(torch, [0, 2]), rows=words(torch, [1, 2]), q_start=words(torch, [0, 0, 0]))    # no tokens


@pytest.mark.gpu
def test_more_rows_than_a_step(gpu, torch):
    """Families of more rows than the plan's threads, and many of few."""
    n = 1100
    c = family(gpu, torch, [70], [n], [1 + i % 3 for i in range(n)], 1, 16, 16, "float16")
    rows = list(range(1, n + 1))
    q = torch.randn((n, 2, 16), generator=torch.Generator("cuda").manual_seed(1), device="cuda").half()
    c.table[700, 2] = c.table[700, 0]                             # one row parts from the others at its third page
    ref, ref_lse = want(c, 0, q, rows, [1] * n), want_lse(c, 0, q, rows, [1] * n)
    for families in ([0, n], list(range(0, n + 1, 10)), [30, 1090]):
        lse = torch.empty((n, 2), device="cuda")
        check(c.attend_shared(0, q, words(torch, families), rows=words(torch, rows), lse=lse), ref)
        check_lse(lse, ref_lse)


@pytest.mark.gpu
def test_the_table_says_what_is_common(gpu, torch):
    """Rows whose pages part in the middle, by an eviction of one of them: the
    pages behind are each row's own."""
    c = family(gpu, torch, [400], [4], [5, 9, 1, 30], 2, 64, 16, "float16")
    q = torch.randn((4, 4, 64), generator=torch.Generator("cuda").manual_seed(2), device="cuda").half()
    rows = [1, 2, 3, 4]
    mass = c.mass()
    mass.uniform_(generator=torch.Generator("cuda").manual_seed(3))
    c.evict(mass, 350, words(torch, [3]), first=130, recent=20)
    for families in ([0, 4], [0, 2, 4]):
        check(c.attend_shared(0, q, words(torch, families), rows=words(torch, rows)), want(c, 0, q, rows, [1] * 4))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,cache,each", [("float16", "float16", 3), ("bfloat16", "bfloat16", 24), ("float32", "float16", 5)])
def test_values_that_are_no_numbers(gpu, torch, dtype, cache, each):
    """An infinite value in the common pages reaches all rows in its place; what
    lies in a row's own keys reaches that row; what windows leave out, none."""
    H, kv, d = 8, 2, 128
    c = family(gpu, torch, [300], [each], [20 + i for i in range(each)], kv, d, 16, cache)
    rows = list(range(1, each + 1))
    q = torch.randn((each, H, d), generator=torch.Generator("cuda").manual_seed(4), device="cuda").to(getattr(torch, dtype))
    families = words(torch, [0, each])
    near = c.attend_shared(0, q, families, rows=words(torch, rows), window=64)
    ref, ref_near = want(c, 0, q, rows, [1] * each), want(c, 0, q, rows, [1] * each, window=64)
    c.v[0, int(c.table[1, 3]), :, 5, 9] = math.inf
    c.v[0, int(c.table[1, 18]), :, 15, 40] = math.nan              # token 303: the first row's own
    got = c.attend_shared(0, q, families, rows=words(torch, rows)).double()
    assert bool((got[:, :, 9] == math.inf).all())
    assert bool(got[0, :, 40].isnan().all()) and bool(torch.isfinite(got[1:, :, 40]).all())
    rest = [i for i in range(d) if i not in (9, 40)]
    check(got[:, :, rest], [x[:, :, rest] for x in ref])
    far = c.attend_shared(0, q, families, rows=words(torch, rows), window=64)      # the infinity is before every window
    assert torch.equal(far[1:], near[1:])
    check(far[:1, :, rest], [x[:1, :, rest] for x in ref_near])    # (a row with a NaN may be computed another way)


@pytest.mark.gpu
def test_streams_and_graph(gpu, torch):
    """Captured, and replayed while rows grow, with eager work between; calls of
    two streams have workspaces of their own."""
    each = 12
    a, b = (family(gpu, torch, [200], [each], [3 + i for i in range(each)], 2, 64, 16, "float16") for _ in range(2))
    rows, families = words(torch, list(range(1, each + 1))), words(torch, [0, each])
    a, b = (gpu.KVCache(x.k, x.v, torch.cat([x.table, torch.full_like(x.table, -1)], 1), x.len, x.ref) for x in (a, b))
    q, k = torch.randn((each, 8, 64), device="cuda").half(), torch.randn((each, 2, 64), device="cuda").half()
    out, lse = torch.empty_like(q), torch.empty((each, 8), device="cuda")

    def step(c, out, lse):
        c.extend(1, rows=rows)
        c.append(0, k, k, rows=rows)
        c.attend_shared(0, q, families, out, rows=rows, lse=lse)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        a.attend_shared(0, q, families, out, rows=rows)
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            step(a, out, lse)
    eager, elog = torch.empty_like(out), torch.empty_like(lse)
    for i in range(6):
        q.copy_(torch.randn_like(q))
        k.copy_(torch.randn_like(k))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        step(b, eager, elog)
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.equal(lse, elog)
        if i == 2:                                                # more tokens than the graph's workspace is for
            with torch.cuda.stream(s):
                big = torch.randn((900, 8, 64), device="cuda").half()
                b.attend_shared(0, big, families, rows=rows, q_start=words(torch, [75 * j for j in range(each + 1)]))
            torch.cuda.synchronize()
    assert len({w.data_ptr() for x in (a, b) for held in x._more_ws.values() for w in held}) >= 3


@pytest.mark.gpu
def test_workspaces_of_growing_calls(gpu, torch):
    """A call that is a little larger than the last takes the same workspace or
    one in its place; one that a capture has had stays."""
    c = family(gpu, torch, [40], [2], [5, 9], 2, 64, 16, "float16")
    rows, families = words(torch, [1, 2]), words(torch, [0, 2])

    def need(n):
        return c._lib.gs_attn_shared_workspace(c._c, 64, 2, 1, n)

    def call(n):
        q = torch.randn((n, 64, 64), device="cuda").half()
        return c.attend_shared(0, q, families, rows=rows, q_start=words(torch, [0, 1, n]))

    def held():
        return [w.numel() for k, x in c._more_ws.items() if k[0] == "attend_shared" for w in x]

    for n in (500, 501, 502, 4000, 4001):
        call(n)
        assert len(held()) == 1 and need(n) <= held()[0] <= need(n) * 9 // 8 + 1, n
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    q = torch.randn((600, 64, 64), device="cuda").half()
    out, start = torch.empty_like(q), words(torch, [0, 1, 600])
    c._more_ws.clear()
    c._graph_ws.clear()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        with torch.cuda.graph(graph, stream=s):
            c.attend_shared(0, q, families, out, rows=rows, q_start=start)
        first = held()
        for n in (2000, 4000, 8000):                              # (the ones between go, the graph's does not)
            call(n)
            assert held()[0] == first[0] and len(held()) == 2 and held()[1] >= max(need(n), 2 * first[0])
    torch.cuda.synchronize()
    want_out = c.attend_shared(0, q, families, rows=rows, q_start=start)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want_out)


def test_refusals_without_gpu():
    import gs_sampler as gs
    lib = gs.load_library()
    INV, UNS = gs.GS_ERR_INVALID, gs.GS_ERR_UNSUPPORTED
    c = fake(gs)
    ws = lib.gs_attn_shared_workspace(c, 4, 2, 1, 2)
    assert ws > lib.gs_attn_workspace(c, 4) // 2
    for bad in ((5, 2, 1, 2), (0, 2, 1, 2), (4, 65537, 1, 2), (4, 2, 65537, 2), (4, 2, 1, 0x7fffffff)):
        assert lib.gs_attn_shared_workspace(c, *bad) == 0

    def call(layer=0, b=(2, 2, None, None), cache=c, families=4096, n=1, lse=None, **kw):
        x = dict(type=1, n_heads=4, q=4096, ld_q=256, out=8192, ld_out=256, scale=0.0, window=0, max_q=0, ws=4096, ws_bytes=ws)
        x.update(kw)
        return lib.gs_attn_shared(cache, layer, ctypes.byref(gs.GsKVBatch(*b)), families, n, ctypes.byref(gs.GsAttnArgs(**x)), lse, None)

    for kw in (dict(layer=1), dict(n_heads=3), dict(q=None), dict(out=4096), dict(ld_q=255), dict(ld_out=257), dict(q=4104),
               dict(ws=None), dict(ws=4104), dict(ws_bytes=ws - 1), dict(scale=math.nan), dict(families=None), dict(n=0), dict(lse=4098),
               dict(b=(5, 5, None, None)), dict(cache=fake(gs, k=None))):
        assert call(**kw) == INV, kw
    assert call(type=30) == UNS and call(n=65537) == UNS
    assert call(b=(0, 0, None, 4096)) == gs.GS_OK
    # gs_attn_lse refuses what gs_attn does
    x = gs.GsAttnArgs(type=1, n_heads=4, q=4096, ld_q=256, out=8192, ld_out=256, ws=4096, ws_bytes=lib.gs_attn_workspace(c, 4))
    assert lib.gs_attn_lse(c, 0, ctypes.byref(gs.GsKVBatch(1, 1, None, None)), ctypes.byref(x), 4098, None) == INV


@pytest.mark.gpu
def test_refusals(gpu, torch):
    c = family(gpu, torch, [40], [2], [5, 9], 2, 64, 16, "float16")
    q = torch.randn((2, 4, 64), device="cuda").half()
    rows, families = words(torch, [1, 2]), words(torch, [0, 2])
    for kw in (dict(lse=torch.empty((2, 4), device="cuda").half()), dict(lse=torch.empty((4, 2), device="cuda").t()),
               dict(lse=torch.empty((2, 4)))):
        for f in (lambda **k: c.attend_shared(0, q, families, rows=rows, **k), lambda **k: c.attend(0, q, rows=rows, **k)):
            with pytest.raises(TypeError):
                f(**kw)
    with pytest.raises(ValueError):
        c.attend_shared(0, q, families, rows=rows, lse=torch.empty((2, 3), device="cuda"))
    for bad in (families.float(), families.cpu(), words(torch, [0, 1, 2, 2])[::2]):
        with pytest.raises(TypeError):
            c.attend_shared(0, q, bad, rows=rows)
    with pytest.raises(ValueError):
        c.attend_shared(0, q, families[:1], rows=rows)
    for window in (-1, (1 << 32) + 5):
        with pytest.raises(ValueError):
            c.attend_shared(0, q, families, rows=rows, window=window)
    with pytest.raises(ValueError):
        c.attend_shared(0, q, families, out=torch.empty((2, 4, 64), device="cuda"), rows=rows)
