"""Timed work of the operators between a model's projections: rotary positions,
the paged cache of keys and values, and the attention that reads it.

Each case is one pass through public entry points of gs_sampler.py:

  rotate  Rope.apply: rotary positions of T tokens' heads
  append  KVCache.append: new tokens' queries and keys turned to their
          positions, keys and values written to the rows' pages
  fork    KVCache.free, fork, extend: rows dropped, made again as copies of
          others that share their pages, and lengthened
  drop    KVCache.free, fork, drop: a range of tokens taken out of rows that
          share their pages, the later keys turned back to their new positions
  attend  KVCache.attend: causal attention of each row's newest tokens over
          its pages

`own` False: the same results from elementary torch operations.
listed() holds the sizes of real use; draw() spreads over the same ranges.

Layouts: tokens' heads are [T, heads, d]; a cache's k and v are [layers, pages,
kv heads, page, d]; table [rows, ld] holds a row's page numbers in order (-1
past its last), len [rows] its tokens, ref [pages] how many rows hold a page.
New pages are the lowest-numbered free ones, in the order of the rows of the
call; a row's last page is shared only when it is full.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # The queries of one chat token: the latency of the call.
        dict(name="rotate_1x32x128_f32", kind="rotate", T=1, H=32, d=128, rot=128, layout="half", base=1e6,
             scaling="none", factor=1.0, span=32768, type="f32"),
        # A long prompt's heads, a third of each head not turned, positions past the trained context.
        dict(name="rotate_12001x32x96_bf16", kind="rotate", T=12001, H=32, d=96, rot=64, layout="interleaved",
             base=500000.0, scaling="yarn", factor=8.0, span=131072, type="bf16"),
        # One chat token of one layer, as the 32-bit projections give it.
        dict(name="append_1_f32", kind="append", n=1, lo=2999, hi=2999, q=1, H=28, kv=4, d=128, rot=128, layout="half",
             base=1e6, scaling="none", factor=1.0, type="f32", cache="f16", page=16),
        # Chunks of four prompts.
        dict(name="append_4x2048_f16", kind="append", n=4, lo=2100, hi=8192, q=2048, H=32, kv=8, d=128, rot=128,
             layout="half", base=500000.0, scaling="yarn", factor=4.0, type="f16", cache="f16", page=64),
        # Eight answers to one prompt: the children share its pages.
        dict(name="fork_1to8_1021", kind="fork", n=1, each=8, lo=1021, hi=1021, add=1, layers=28, kv=4, d=128, page=16,
             cache="f16"),
        # A serving batch of many answers to each prompt.
        dict(name="fork_16to256", kind="fork", n=16, each=16, lo=1500, hi=2500, add=33, layers=28, kv=4, d=128, page=64,
             cache="bf16"),
        # One conversation at the end of its context: the oldest quarter after the system prompt goes.
        dict(name="drop_1x8192", kind="drop", n=1, lo=8192, hi=8192, keep=211, gone=2048, layers=28, kv=4, d=128, rot=128,
             layout="half", base=1e6, page=16, cache="f16"),
        # The same for a batch of rows of odd lengths.
        dict(name="drop_16x6000", kind="drop", n=16, lo=2500, hi=6000, keep=64, gone=777, layers=8, kv=8, d=128, rot=128,
             layout="interleaved", base=10000.0, page=64, cache="bf16"),
        # One chat token over a conversation, with the 32-bit activations of the projections.
        dict(name="attend_1x4001_f32", kind="attend", n=1, lo=4001, hi=4001, q=1, H=28, kv=4, d=128, type="f32",
             cache="f16", page=16, window=0, mixed=False),
        # A serving batch, one token each, from short to long conversations.
        dict(name="attend_64x32768_bf16", kind="attend", n=64, lo=1000, hi=32768, q=1, H=28, kv=4, d=128, type="bf16",
             cache="bf16", page=64, window=0, mixed=False),
        # Chunks of four prompts over what is in the cache already.
        dict(name="attend_4x2048_f16", kind="attend", n=4, lo=2100, hi=8192, q=2048, H=32, kv=8, d=128, type="f16",
             cache="f16", page=64, window=0, mixed=False),
        # Single tokens and chunks in one call, wide heads, a sliding window, rows in any order.
        dict(name="attend_mixed_24_bf16", kind="attend", n=24, lo=700, hi=8192, q=601, H=16, kv=8, d=256, type="bf16",
             cache="bf16", page=32, window=4096, mixed=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("rotate", "append", "append", "fork", "drop", "attend", "attend", "attend", "attend"))
    kv = rng.choice((1, 2, 4, 8))
    H = kv * rng.choice((1, 2, 4, 5, 7, 8))
    d = rng.choice((64, 80, 96, 128, 128, 128, 192, 256))
    rot = rng.choice((d, d, d // 2))
    cache = rng.choice(("f16", "bf16"))
    page = rng.choice((16, 32, 64, 128))
    turn = dict(rot=rot, layout=rng.choice(("half", "interleaved")), base=rng.choice((10000.0, 500000.0, 1e6)))
    long = dict(scaling=rng.choice(("none", "linear", "yarn")), factor=rng.choice((2.0, 4.0, 8.0)))
    if kind == "rotate":
        return dict(kind=kind, T=min(_log(rng, 1, 16000), 36000000 // (H * d)), H=H, d=d, **turn, **long,
                    span=_log(rng, 1000, 131072), type=rng.choice(("f32", "f16", "bf16")))
    if kind == "append":
        n = _log(rng, 1, 64)
        q = 1 if rng.random() < 0.5 else max(1, min(_log(rng, 2, 2048), 30000000 // (n * (H + 2 * kv) * d)))
        lo = _log(rng, 100, 2000)
        return dict(kind=kind, n=n, lo=max(lo, q), hi=max(lo, q) + _log(rng, 1, 2000), q=q, H=H, kv=kv, d=d, **turn, **long,
                    type=rng.choice(("f32", cache)), cache=cache, page=page)
    if kind == "fork":
        n, each = _log(rng, 1, 16), _log(rng, 1, 16)
        lo = _log(rng, 20, 2000)
        return dict(kind=kind, n=n, each=each, lo=lo, hi=lo + _log(rng, 1, 500), add=_log(rng, 1, 100),
                    layers=rng.choice((1, 8, 28)) if kv * d <= 512 else 8, kv=kv, d=d, page=rng.choice((16, 32, 64)),
                    cache=cache)
    if kind == "drop":
        n, lo = _log(rng, 1, 12), _log(rng, 500, 4000)
        keep = rng.choice((0, rng.randint(1, 300)))
        return dict(kind=kind, n=n, lo=lo, hi=lo + _log(rng, 1, 2000), keep=keep, gone=_log(rng, 1, lo), layers=4, kv=kv,
                    d=d, **turn, page=page, cache=cache)
    case = dict(kind=kind, n=_log(rng, 1, 64), H=H, kv=kv, d=d, cache=cache, page=page,
                window=rng.choice((0, 0, 0, 1000)), mixed=False)
    case["type"] = rng.choice(("f32", cache))
    case["q"] = 1 if rng.random() < 0.5 else _log(rng, 2, 2048 if case["type"] == cache else 64)
    case["mixed"] = case["q"] > 1 and rng.random() < 0.4
    if case["q"] > 1:
        case["n"] = min(case["n"], 12 if case["mixed"] else 4)
    case["lo"] = max(case["q"], _log(rng, 1, 2000))
    case["hi"] = min(case["lo"] + _log(rng, 1, 60000000 // (case["n"] * kv * d) if case["q"] == 1 else 6000), 32768)
    while work(case)["flops"] > 4e11 * (1.0 if case["type"] == cache else 0.1):
        case["q"] = max(1, case["q"] // 2)
    return case


def _gen(seed, what):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 16 + what)
    return g


def _lens(case):
    """The rows' lengths: spread over lo .. hi, by their logarithm."""
    lo, hi = case["lo"], case["hi"]
    return [int(round(lo * (hi / lo) ** ((0.35 + 0.618034 * i) % 1.0))) for i in range(case["n"])] if hi > lo else [lo] * case["n"]


def _news(case):
    """New tokens of each row: q, or in a mixed call one token for most."""
    return [max(1, case["q"] - 37 * (i // 6)) if not case.get("mixed") or i % 6 == 3 else 1 for i in range(case["n"])]


def _rows(case):
    """The cache's row of each sequence of the call: any order in a mixed one."""
    return np.random.default_rng(case["n"]).permutation(case["n"]).tolist() if case["mixed"] else list(range(case["n"]))


def _frequencies(case):
    """Turns per position of each pair (64 bits), and the factor on cos and
    sin.  Linear: all divided by the factor.  YaRN: pairs that turn less than
    once in the trained context (32 times: not at all) are divided by it, a
    ramp over the pairs' numbers between; values times 0.1 ln(factor) + 1."""
    rot, base, s = case["rot"], case["base"], case.get("factor", 1.0)
    i = np.arange(rot // 2, dtype=np.float64)
    f = base ** (-2.0 * i / rot) / (2.0 * math.pi)
    if case.get("scaling", "none") == "linear":
        return f / s, 1.0
    if case.get("scaling", "none") == "yarn":
        at = [rot * math.log(_context(case) / (2.0 * math.pi * r)) / (2.0 * math.log(base)) for r in (32.0, 1.0)]
        low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rot - 1)
        ramp = np.clip((i - low) / max(high - low, 0.001), 0.0, 1.0)
        return f / s * ramp + f * (1.0 - ramp), 0.1 * math.log(s) + 1.0
    return f, 1.0


def _context(case):
    return 8192


def _pages(case):
    """Pages of the pool: the parents', the children's and some spare."""
    P = case["page"]
    held = sum(-(-x // P) for x in _lens(case))
    if case["kind"] == "fork":
        return held + case["n"] * case["each"] * (case["add"] // P + 3) + 5
    return held * (2 if case["kind"] == "drop" else 1) + case["n"] + 5


def _cache(case, seed):
    """A pool whose pages the rows hold in no order; children start empty."""
    P, n, dt = case["page"], case["n"], TYPES[case["cache"]]
    rows = n * (1 + case["each"]) if case["kind"] == "fork" else 2 * n if case["kind"] == "drop" else n
    lens, total = _lens(case), _pages(case)
    ld = max(-(-x // P) for x in lens) + case.get("add", 0) // P + 2
    g = _gen(seed, 1)
    shape = (case.get("layers", 1), total, case["kv"], P, case["d"])
    st = {x: torch.randn(shape, generator=g, device="cuda", dtype=dt) for x in ("k", "v")}
    # values have a mean of their own in each channel
    st["v"] += torch.randn((case["kv"], 1, case["d"]), generator=g, device="cuda", dtype=dt)
    order = np.random.default_rng(seed).permutation(total).astype(np.int32)
    table, ref = np.full((rows, ld), -1, np.int32), np.zeros(total, np.int32)
    held = np.arange(ld) < -(-np.array(lens)[:, None] // P)
    table[:n][held] = order[:held.sum()]
    ref[order[:held.sum()]] = 1
    st["table"], st["ref"] = torch.from_numpy(table).cuda(), torch.from_numpy(ref).cuda()
    st["len"] = torch.tensor(lens + [0] * (rows - n), dtype=torch.int32, device="cuda")
    return st


def _int(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    kind, st = case["kind"], dict(case=case)
    if kind != "rotate":
        st.update(_cache(case, seed))
        st["rows"] = torch.arange(case["n"], dtype=torch.int32, device="cuda")
    if kind != "attend" and kind != "fork":
        f, st["gain"] = _frequencies(case)
        st["turns"] = torch.from_numpy(np.round(f * 2.0 ** 43).astype(np.int64)).cuda()   # positions < 2^19
    g = _gen(seed, 2)
    if kind == "rotate":
        st["x"] = torch.randn((case["T"], case["H"], case["d"]), generator=g, device="cuda").to(TYPES[case["type"]])
        st["pos"] = torch.randint(0, case["span"], (case["T"],), generator=g, device="cuda", dtype=torch.int32)
        st["out"] = torch.empty_like(st["x"])
    if kind in ("append", "attend"):
        new = _news(case)
        st["start"] = _int(np.concatenate([[0], np.cumsum(new)]).tolist())
        st["q"] = torch.randn((sum(new), case["H"], case["d"]), generator=g, device="cuda")
        # scores of about 2.5: some keys count much more than others
        st["q"] = (st["q"] * 2.5 if kind == "attend" else st["q"]).to(TYPES[case["type"]])
        st["out"] = torch.empty_like(st["q"])
        # where the padded form of the rows finds each token
        st["at"] = torch.from_numpy(np.concatenate([np.arange(m) + i * max(new) for i, m in enumerate(new)])).cuda()
    if kind == "append":
        st["kn"], st["vn"] = (torch.randn((sum(new), case["kv"], case["d"]), generator=g, device="cuda")
                              .to(TYPES[case["type"]]) for _ in range(2))
    if kind == "attend":
        st["rows"] = _int(_rows(case))
    if kind == "fork":
        st["src"] = torch.arange(case["n"], dtype=torch.int32, device="cuda").repeat_interleave(case["each"])
    if kind == "drop":
        st["src"] = torch.arange(case["n"], dtype=torch.int32, device="cuda")
        st["from"] = torch.full((case["n"],), case["keep"], dtype=torch.int32, device="cuda")
        st["to"] = st["from"] + case["gone"]
    if kind in ("fork", "drop"):
        st["dst"] = torch.arange(case["n"], st["len"].numel(), dtype=torch.int32, device="cuda")
    if own:
        _handles(st)
    return st


def _handles(st):
    """What a program keeps beside the tensors: the plan of the rotation and
    the cache's description."""
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gguf-rs-cli_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import gs_sampler as gs
    case = st["case"]
    if "turns" in st:
        st["rope"] = gs.Rope(case["d"], rot=case["rot"], layout=case["layout"], base=case["base"],
                             scaling=case.get("scaling", "none"), factor=case.get("factor", 1.0), context=_context(case))
    if "k" in st:
        st["cache"] = gs.KVCache(st["k"], st["v"], st["table"], st["len"], st["ref"])


# ---- the plain forms ---------------------------------------------------------

def _rotated(st, x, pos, gain):
    """x [.., heads, d] at positions pos [..]: pairs (a, b) of the first `rot`
    values become (a cos - b sin, b cos + a sin).  The turns are whole numbers
    of 2^-43, so that only the part of a turn is left to round."""
    case = st["case"]
    part = (pos.long()[..., None] * st["turns"]) & ((1 << 43) - 1)
    angle = part.float() * (2.0 * math.pi / (1 << 43))
    c, s = (torch.cos(angle) * gain)[..., None, :], (torch.sin(angle) * gain)[..., None, :]
    rot, x = case["rot"], x.float()
    if case["layout"] == "half":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat([a * c - b * s, b * c + a * s], -1)
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    return torch.cat([y, x[..., rot:]], -1)


def _plain_append(st):
    case, P = st["case"], st["case"]["page"]
    start = st["start"].long()
    T = st["q"].shape[0]
    row = torch.bucketize(torch.arange(T, device="cuda"), start[1:], right=True)
    pos = st["len"].long()[row] - start[row + 1] + torch.arange(T, device="cuda")
    page, slot = st["table"].long()[row, pos // P], pos % P
    st["k"][0, page, :, slot] = _rotated(st, st["kn"], pos, st["gain"]).to(st["k"].dtype)
    st["v"][0, page, :, slot] = st["vn"].to(st["v"].dtype)
    st["out"].copy_(_rotated(st, st["q"], pos, st["gain"]))
    return dict(q=st["out"], k=st["k"], v=st["v"])


def _held(st, rows):
    """The rows' page numbers and which of the table's places hold one."""
    P, table = st["case"]["page"], st["table"].long()[rows]
    n = (st["len"].long()[rows] + P - 1) // P
    return table, torch.arange(table.shape[1], device="cuda") < n[:, None]


def _count(st, pages, by):
    st["ref"].index_add_(0, pages, torch.full_like(pages, by).int())


def _free_pages(st):
    return torch.argsort((st["ref"] != 0).to(torch.int32), stable=True)


def _plain_free(st, rows):
    table, held = _held(st, rows)
    _count(st, table[held], -1)
    st["table"][rows] = -1
    st["len"][rows] = 0


def _plain_fork(st, src, dst):
    P = st["case"]["page"]
    L, table = st["len"].long()[src], st["table"].long()[src]
    full, rest = L // P, L % P
    place = torch.arange(table.shape[1], device="cuda")
    shared, last = place < full[:, None], (place == full[:, None]) & (rest > 0)[:, None]
    new = _free_pages(st)[(rest > 0).long().cumsum(0) - 1]
    st["table"][dst] = torch.where(shared, table, torch.where(last, new[:, None], -1)).int()
    st["len"][dst] = L.int()
    _count(st, table[shared], 1)
    take = rest > 0
    old, new, rest = table[last], new[take], rest[take]
    _count(st, new, 1)
    here = (torch.arange(P, device="cuda") < rest[:, None])[:, None, :, None]
    st["k"][:, new] = torch.where(here, st["k"][:, old], st["k"][:, new])
    st["v"][:, new] = torch.where(here, st["v"][:, old], st["v"][:, new])


def _plain_extend(st, rows, add):
    P, table, L = st["case"]["page"], st["table"].long()[rows], st["len"].long()[rows]
    was, now = (L + P - 1) // P, (L + add + P - 1) // P
    place = torch.arange(table.shape[1], device="cuda")
    given = (place >= was[:, None]) & (place < now[:, None])
    new = _free_pages(st)[:table.numel()][(given.reshape(-1).long().cumsum(0) - 1).clamp(0, st["ref"].numel() - 1)]
    new = new.reshape(given.shape)
    st["table"][rows] = torch.where(given, new, table).int()
    _count(st, new[given], 1)
    st["len"][rows] = (L + add).int()


def _plain_drop(st, rows, start, end):
    P, table, L = st["case"]["page"], st["table"].long()[rows], st["len"].long()[rows]
    a = torch.minimum(start.long(), L)
    n = torch.minimum(torch.maximum(end.long(), a), L) - a
    left = L - n
    place = torch.arange(table.shape[1], device="cuda")
    was, now = (L + P - 1) // P, (left + P - 1) // P
    held = place < was[:, None]
    written = (place >= (a // P)[:, None]) & (place < now[:, None]) & (n > 0)[:, None]
    fresh = written & (st["ref"].long()[table.clamp(min=0)] > 1)
    new = _free_pages(st)[:table.numel()][(fresh.reshape(-1).long().cumsum(0) - 1).clamp(0, st["ref"].numel() - 1)]
    new = torch.where(fresh, new.reshape(fresh.shape), torch.where(place < now[:, None], table, -1))
    # every token from the first written page on: where it was, where it goes
    t = torch.arange(table.shape[1] * P, device="cuda").expand(len(rows), -1)
    moves = (t >= (a // P * P)[:, None]) & (t < left[:, None]) & (n > 0)[:, None]
    r, t = moves.nonzero(as_tuple=True)
    later = t >= a[r]
    s = torch.where(later, t + n[r], t)
    page, slot, to, at = table[r, s // P], s % P, new[r, t // P], t % P
    k, v = st["k"][:, page, :, slot], st["v"][:, page, :, slot]
    turned = _rotated(st, k, torch.where(later, -n[r], 0)[:, None], 1.0).to(k.dtype)
    st["k"][:, to, :, at] = torch.where(later[:, None, None, None], turned, k)
    st["v"][:, to, :, at] = v
    _count(st, table[fresh | (held & (place >= now[:, None]))], -1)
    _count(st, new[fresh], 1)
    st["table"][rows] = new.int()
    st["len"][rows] = left.int()


def _plain_attend(st):
    case = st["case"]
    P, H, kv, d, n = case["page"], case["H"], case["kv"], case["d"], case["n"]
    rows, start = st["rows"].long(), st["start"].long()
    L, new = st["len"].long()[rows], start[1:] - start[:-1]
    Q = max(_news(case))
    q = torch.zeros((n * Q, H, d), device="cuda")
    q[st["at"]] = st["q"].float()
    table, held = _held(st, rows)
    S = table.shape[1] * P
    pages = torch.where(held, table, 0)
    k = st["k"][0][pages].float().permute(0, 2, 1, 3, 4).reshape(n, kv, S, d)
    v = st["v"][0][pages].float().permute(0, 2, 1, 3, 4).reshape(n, kv, S, d)
    q = q.reshape(n, Q, kv, H // kv, d).permute(0, 2, 3, 1, 4).reshape(n, kv, H // kv * Q, d)
    s = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(1.0 / math.sqrt(d)).reshape(n, kv, H // kv, Q, S)
    pos = (L - new)[:, None, None] + torch.arange(Q, device="cuda")[:, None]
    key = torch.arange(S, device="cuda")
    seen = (key <= pos) & (key < L[:, None, None])
    if case["window"]:
        seen &= key > pos - case["window"]
    seen = seen[:, None, None]
    s.masked_fill_(~seen, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(m == -math.inf, 0.0, m)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.reshape(n, kv, H // kv * Q, S), v).reshape(n, kv, H // kv, Q, d) / torch.where(total == 0, 1.0, total)
    o = o.permute(0, 3, 1, 2, 4).reshape(n * Q, H, d)
    st["out"].copy_(o[st["at"]])
    return st["out"]


def _plain(st):
    kind = st["case"]["kind"]
    if kind == "rotate":
        st["out"].copy_(_rotated(st, st["x"], st["pos"], st["gain"]))
        return st["out"]
    if kind == "append":
        return _plain_append(st)
    if kind == "attend":
        return _plain_attend(st)
    dst = st["dst"].long()
    _plain_free(st, dst)
    _plain_fork(st, st["src"].long(), dst)
    if kind == "fork":
        _plain_extend(st, dst, st["case"]["add"])
    else:
        _plain_drop(st, dst, st["from"], st["to"])
    return dict(k=st["k"], v=st["v"], table=st["table"], len=st["len"], ref=st["ref"])


def run(state):
    if not own:
        return _plain(state)
    st, case = state, state["case"]
    kind = case["kind"]
    if kind == "rotate":
        st["rope"].apply(st["x"], st["pos"], out=st["out"])
        return st["out"]
    cache = st["cache"]
    one = None if case.get("q", 1) == 1 else st["start"]
    if kind == "append":
        cache.append(0, st["kn"], st["vn"], q=st["q"], q_out=st["out"], rope=st["rope"], rows=st["rows"], q_start=one)
        return dict(q=st["out"], k=st["k"], v=st["v"])
    if kind == "attend":
        cache.attend(0, st["q"], st["out"], rows=st["rows"], q_start=one, max_q=case["q"], window=case["window"])
        return st["out"]
    cache.free(st["dst"])
    cache.fork(st["src"], st["dst"])
    if kind == "fork":
        cache.extend(case["add"], rows=st["dst"])
    else:
        cache.drop(st["from"], st["to"], rows=st["dst"], rope=st["rope"])
    return dict(k=st["k"], v=st["v"], table=st["table"], len=st["len"], ref=st["ref"])


# ---- the work ----------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "rotate":
        size = case["T"] * case["H"] * case["d"]
        return dict(bytes=2 * size * TYPES[case["type"]].itemsize + 4 * case["T"], flops=3 * size * case["rot"] // case["d"])
    item = TYPES[case["cache"]].itemsize
    token = 2 * case["kv"] * case["d"] * item                     # of one layer
    if kind == "append":
        T, w = sum(_news(case)), TYPES[case["type"]].itemsize
        size = T * case["d"] * (2 * case["H"] + 2 * case["kv"])
        return dict(bytes=size * w + T * token, flops=3 * T * (case["H"] + case["kv"]) * case["rot"])
    P, lens = case["page"], _lens(case)
    if kind == "fork":
        kids = case["each"] * sum(x % P for x in lens)
        pages = case["each"] * sum(-(-(x + case["add"]) // P) for x in lens)
        return dict(bytes=2 * kids * token * case["layers"] + 4 * 6 * pages, flops=0)
    if kind == "drop":
        moved = last = 0
        for x in lens:
            a = min(case["keep"], x)
            n = min(case["gone"], x - a)
            moved += x - n - a // P * P
            last += x % P
        return dict(bytes=2 * (moved + last) * token * case["layers"] + 4 * 4 * _pages(case),
                    flops=3 * moved * case["layers"] * case["kv"] * case["rot"])
    keys = pairs = 0
    for i, m in zip(_rows(case), _news(case)):
        x, w = lens[i], case["window"] or 1 << 30
        first = max(0, x - m + 1 - w)
        keys += x - first
        pairs += sum(max(0, min(x - m + j + 1, w)) for j in range(m))
    q = sum(_news(case)) * case["H"] * case["d"] * TYPES[case["type"]].itemsize
    return dict(bytes=keys * token + 2 * q, flops=4 * pairs * case["H"] * case["d"])


# ---- the values in 64 bits, from the definitions -------------------------------

def _turned(case, x, pos, gain=None):
    """Row by row as complex numbers: (a + ib) e^(i angle)."""
    f, g = _frequencies(case)
    g = g if gain is None else gain
    angle = pos.double()[..., None] * torch.from_numpy(f * 2.0 * math.pi).cuda()
    z = torch.polar(torch.full_like(angle, g), angle).unsqueeze(-2)
    rot, y = case["rot"], x.double().clone()
    one = (slice(0, rot // 2), slice(rot // 2, rot)) if case["layout"] == "half" else (slice(0, rot, 2), slice(1, rot, 2))
    w = torch.complex(y[..., one[0]].contiguous(), y[..., one[1]].contiguous()) * z
    y[..., one[0]], y[..., one[1]] = w.real, w.imag
    return y


def exact(case, seed):
    st, kind = prepare(case, seed), case["kind"]
    if kind == "rotate":
        return _turned(case, st["x"], st["pos"])
    P = case["page"]
    table, lens = st["table"].cpu().numpy(), st["len"].cpu().numpy()
    if kind == "append":
        k, v, q, at = st["k"].double(), st["v"].double(), st["q"].double(), 0
        for i, m in enumerate(_news(case)):
            pos = torch.arange(int(lens[i]) - m, int(lens[i]), device="cuda")
            here = torch.from_numpy(table[i].astype(np.int64)).cuda()[pos // P]
            k[0, here, :, pos % P] = _turned(case, st["kn"][at:at + m], pos)
            v[0, here, :, pos % P] = st["vn"][at:at + m].double()
            q[at:at + m] = _turned(case, st["q"][at:at + m], pos)
            at += m
        return dict(q=q, k=k, v=v)
    if kind == "attend":
        out, at, rows = st["q"].double(), 0, st["rows"].cpu().tolist()
        group = case["H"] // case["kv"]
        for i, m in enumerate(_news(case)):
            x = int(lens[rows[i]])
            here = torch.from_numpy(table[rows[i], :-(-x // P)].astype(np.int64)).cuda()
            for h in range(case["kv"]):
                k, v = (st[c][0, here, h].reshape(-1, case["d"])[:x].double() for c in ("k", "v"))
                for c in range(0, m, 256):                        # queries c .. of the chunk
                    pos = torch.arange(x - m + c, x - m + min(c + 256, m), device="cuda")
                    q = st["q"][at + c:at + min(c + 256, m), h * group:(h + 1) * group].double()
                    s = torch.tensordot(q, k, dims=([2], [1])) / math.sqrt(case["d"])
                    key = torch.arange(x, device="cuda")
                    off = key[None, :] > pos[:, None]
                    if case["window"]:
                        off |= key[None, :] <= pos[:, None] - case["window"]
                    p = torch.softmax(s.masked_fill(off[:, None, :], -math.inf), -1).nan_to_num(0.0)
                    out[at + c:at + min(c + 256, m), h * group:(h + 1) * group] = torch.tensordot(p, v, dims=([2], [0]))
            at += m
        return out
    # The pages: the bookkeeping a row after the other, the keys and values of
    # each written page in 64 bits.
    ref = st["ref"].cpu().numpy().copy()
    k, v = st["k"].double(), st["v"].double()
    src, dst = st["src"].cpu().tolist(), st["dst"].cpu().tolist()

    def lowest():
        page = int(np.flatnonzero(ref == 0)[0])
        ref[page] = 1
        return page

    for s, c in zip(src, dst):                                    # the children start empty
        x = int(lens[s])
        lens[c] = x
        table[c, :x // P] = table[s, :x // P]
        ref[table[s, :x // P]] += 1
        if x % P:
            old, new = int(table[s, x // P]), lowest()
            table[c, x // P] = new
            k[:, new, :, :x % P], v[:, new, :, :x % P] = k[:, old, :, :x % P], v[:, old, :, :x % P]
    if case["kind"] == "fork":
        for c in dst:
            for j in range(-(-int(lens[c]) // P), -(-(int(lens[c]) + case["add"]) // P)):
                table[c, j] = lowest()
            lens[c] += case["add"]
        return dict(k=k, v=v, table=None, len=None, ref=None)
    gone = []
    for c in dst:
        x = int(lens[c])
        a = min(case["keep"], x)
        n = min(case["gone"], x - a)
        if not n:
            continue
        old = table[c].copy()
        kk = torch.cat([k[:, int(p)] for p in old[:-(-x // P)]], 2)[:, :, :x].clone()
        vv = torch.cat([v[:, int(p)] for p in old[:-(-x // P)]], 2)[:, :, :x].clone()
        back = torch.full((x - n - a,), -n, dtype=torch.int64, device="cuda")
        kk = torch.cat([kk[:, :, :a], _turned(case, kk[:, :, a + n:].transpose(1, 2), back[None, :], 1.0).transpose(1, 2)], 2)
        vv = torch.cat([vv[:, :, :a], vv[:, :, a + n:]], 2)
        for j in range(-(-x // P)):
            if j * P >= x - n:
                gone.append(int(old[j]))
                table[c, j] = -1
            elif j >= a // P:
                if ref[old[j]] > 1:
                    gone.append(int(old[j]))
                    table[c, j] = lowest()
                m = min(P, x - n - j * P)
                k[:, int(table[c, j]), :, :m] = kk[:, :, j * P:j * P + m]
                v[:, int(table[c, j]), :, :m] = vv[:, :, j * P:j * P + m]
        lens[c] = x - n
    return dict(k=k, v=v, table=None, len=None, ref=None)
