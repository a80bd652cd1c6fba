#!/usr/bin/env python3
"""Generation for many conversations over one paged cache.

A small decoder-only model with random weights runs through the library's own
operators: quantised projections (QMatrix), rotary positions and the write of
keys and values to their pages (KVCache.append), attention over them
(KVCache.attend), sampling and the decode loop's state (Decoder).  Prompts of
different lengths go through in one call per layer, each conversation is forked
into several answers that share the prompt's pages, the answers are generated
token by token without a word to the host, and a conversation whose context is
full loses its oldest tokens instead of running its prompt again
(gguf-rs-cli's smart context, src/main.rs:205-256).  With --shared a prompt's
pages are read once for all of its answers (KVCache.attend_shared); with
--budget a full conversation is cut to that many tokens by the weight that they
have had from the later ones (KVCache.weigh, evict).

    python examples/paged_generate.py [--answers 4] [--new 48] [--shared] [--budget 96]
"""
import argparse
import os
import sys
import time

import numpy as np
import torch

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gguf-rs-cli_amd")
if _PKG not in sys.path:
    sys.path.insert(0, _PKG)
import gs_sampler as gs  # noqa: E402

SMALL = dict(vocab=4096, hidden=256, heads=8, kv=2, d=32, ffn=512, layers=2, base=10000.0, context=192, page=16)


def q8_blocks(rows, cols, rng):
    """Random Q8_0 blocks of a rows x cols matrix whose products keep a vector's size."""
    blk = np.empty((rows * cols // 32, 34), np.uint8)
    d = np.full(rows * cols // 32, 1.0 / (73.0 * cols ** 0.5), np.float16)      # 73: rms of the int8 values
    blk[:, :2] = d.view(np.uint8).reshape(-1, 2)
    blk[:, 2:] = rng.integers(-127, 128, (rows * cols // 32, 32)).astype(np.int8).view(np.uint8)
    return blk.reshape(-1)


class PagedModel:
    """The layers of a llama-like model over a KVCache: forward() takes the new
    tokens of any rows, from single tokens to whole prompts."""

    def __init__(self, cfg, rows, pages, seed=0):
        rng = np.random.default_rng(seed)
        self.cfg = cfg
        h, d, ffn = cfg["hidden"], cfg["d"], cfg["ffn"]
        shapes = dict(qkv=((cfg["heads"] + 2 * cfg["kv"]) * d, h), o=(h, cfg["heads"] * d), gate=(ffn, h), up=(ffn, h), down=(h, ffn))
        self.blocks = [{n: q8_blocks(*s, rng) for n, s in shapes.items()} for _ in range(cfg["layers"])]
        self.w = [{n: gs.QMatrix(gs.QTYPE_Q8_0, b[n], *shapes[n]) for n in shapes} for b in self.blocks]
        self.head_blocks = q8_blocks(cfg["vocab"], h, rng)
        self.lm_head = gs.QMatrix(gs.QTYPE_Q8_0, self.head_blocks, cfg["vocab"], h)
        self.embed = torch.from_numpy(rng.standard_normal((cfg["vocab"], h), dtype=np.float32)).cuda()
        self.rope = gs.Rope(d, base=cfg["base"])
        self.cache = gs.KVCache.empty(cfg["layers"], pages, cfg["kv"], d, rows, cfg["context"], page=cfg["page"])

    def _project(self, m, x):
        out = torch.empty((x.shape[0], m.rows), device="cuda")
        m.gemv(x, out, B=x.shape[0], stream=torch.cuda.current_stream())
        return out

    @staticmethod
    def _norm(x):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)

    def forward(self, tokens, rows, q_start=None, max_q=1, families=None, mass=None):
        """tokens [T] of `rows` (one each, or those from q_start[i] to
        q_start[i + 1]), for which extend() has made room; returns the hidden
        states [T, hidden] before the output projection.  families: which of
        the rows begin with the same pages; mass: gets the weights that the
        rows' tokens have from these."""
        cfg, n = self.cfg, tokens.shape[0]
        lse = None if mass is None else torch.empty((n, cfg["heads"]), device="cuda")
        x = self.embed[tokens.long()]
        for i, w in enumerate(self.w):
            heads = self._project(w["qkv"], self._norm(x)).view(n, -1, cfg["d"])
            q, k, v = heads.split([cfg["heads"], cfg["kv"], cfg["kv"]], 1)      # parts of one row: strides, no copies
            turned = torch.empty((n, cfg["heads"], cfg["d"]), device="cuda")
            self.cache.append(i, k, v, q=q, q_out=turned, rope=self.rope, rows=rows, q_start=q_start)
            if families is None:
                a = self.cache.attend(i, turned, rows=rows, q_start=q_start, max_q=max_q, lse=lse)
            else:
                a = self.cache.attend_shared(i, turned, families, rows=rows, q_start=q_start, max_q=max_q, lse=lse)
            if mass is not None:
                self.cache.weigh(i, turned, lse, mass, rows=rows, q_start=q_start, max_q=max_q)
            x = x + self._project(w["o"], a.view(n, -1))
            y = self._norm(x)
            y = torch.nn.functional.silu(self._project(w["gate"], y)) * self._project(w["up"], y)
            x = x + self._project(w["down"], y)
        return self._norm(x)


def words(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def generate(model, prompts, answers, new, seed=42, keep=8, shared=False, budget=0):
    """`answers` continuations of each prompt, `new` tokens each; the oldest
    half of what follows the first `keep` tokens leaves a row that is full, or
    with a budget all but the first `keep`, the newest quarter of the budget and
    those of greatest weight between.  shared: an answer's attention reads the
    pages of its prompt together with the prompt's other answers.
    Returns the generated ids [prompts * answers][<= new]."""
    cfg, cache, n = model.cfg, model.cache, len(prompts)
    if not 0 <= budget < cfg["context"]:
        raise ValueError("budget must be less than the context's %d tokens (0: none)" % cfg["context"])
    B = n * answers
    kids = words(list(range(n, n + B)))
    # the prompts, all at once
    lens = [len(p) for p in prompts]
    start = words(np.concatenate([[0], np.cumsum(lens)]).tolist())
    parents = words(list(range(n)))
    cache.extend(words(lens), rows=parents)
    mass = cache.mass() if budget else None
    families = words(list(range(0, B + 1, answers))) if shared else None
    hidden = model.forward(words(np.concatenate(prompts).astype(np.int64).tolist()), parents, start, max(lens), mass=mass)
    # each answer is a row that shares its prompt's pages; the prompt's own row goes
    of = torch.arange(n, device="cuda", dtype=torch.int32).repeat_interleave(answers)
    cache.fork(of, kids)
    if budget:
        mass[kids.long()] = mass[of.long()]                     # the answers' tokens weigh what their prompts' do
    cache.free(parents, mass=mass)
    x = hidden[(start[1:] - 1).long()][of.long()].contiguous()
    sampler = gs.Sampler(0.8, 40, 0.95, 1.1, seed=seed)
    sampler.reserve(B, cfg["vocab"])
    dec = gs.Decoder(B, W=64, max_new=new)
    dec.init(sampler, [seed + b for b in range(B)])
    logits = torch.empty((B, cfg["vocab"]), device="cuda")
    held = [lens[b // answers] for b in range(B)]               # (the host counts along; the device need not be asked)
    for step in range(new):
        dec.step(sampler, logits=logits, lm_head=model.lm_head, x=x)
        if step + 1 == new:
            break
        full = [b for b in range(B) if held[b] == cfg["context"]]
        if full and budget:
            cache.evict(mass, budget, words([n + b for b in full]), first=keep, recent=budget // 4, rope=model.rope)
            for b in full:
                held[b] = min(held[b], budget)
        elif full:
            gone = (cfg["context"] - keep) // 2
            cache.drop(words([keep] * len(full)), words([keep + gone] * len(full)), words([n + b for b in full]), rope=model.rope)
            for b in full:
                held[b] -= gone
        cache.extend(1, rows=kids)
        held = [x + 1 for x in held]
        x = model.forward(dec.next, kids, families=families, mass=mass)
    return [g.tolist() for g in dec.generated_ids()]


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--answers", type=int, default=4)
    ap.add_argument("--new", type=int, default=48)
    ap.add_argument("--shared", action="store_true")
    ap.add_argument("--budget", type=int, default=0)
    a = ap.parse_args()
    rng = np.random.default_rng(1)
    prompts = [rng.integers(0, SMALL["vocab"], k) for k in (150, 37, 5)]
    rows = len(prompts) * (1 + a.answers)
    model = PagedModel(SMALL, rows, pages=rows * SMALL["context"] // SMALL["page"])
    t = time.perf_counter()
    ids = generate(model, prompts, a.answers, a.new, shared=a.shared, budget=a.budget)
    t = time.perf_counter() - t
    for i, p in enumerate(prompts):
        print("prompt of %d tokens:" % len(p))
        for k in range(a.answers):
            print("   ", ids[i * a.answers + k][:16], "...")
    print("%d tokens in %.2f s; %d of %d pages held" % (sum(map(len, ids)), t, int((model.cache.ref > 0).sum()), model.cache.pages))


if __name__ == "__main__":
    main()
