"""Rotary positions (include/gs_rope.h) against the formula in 64 bits.

Tolerances: an angle is off by at most 2 pi 2^-25 (the part of a turn in f32)
and sin and cos by 2 ulp, 5e-7 in all; the two products and the sum add 3
roundings of 2^-24.  Together below 8e-7 (|a| + |b|) gain, then the rounding to
the type: 2^-11 (f16) or 2^-8 (bf16) of the value, and f16's 2^-25 near zero.
"""
import ctypes
import math

import numpy as np
import pytest

U = {"float32": 0.0, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def frequencies(rot, base, scaling="none", factor=1.0, context=0, beta_fast=32.0, beta_slow=1.0, divisors=None):
    """Radians per position of each pair, and the gain."""
    i = np.arange(rot // 2, dtype=np.longdouble)
    f = np.longdouble(base) ** (-2 * i / rot)
    if divisors is not None:
        f = f / np.asarray(divisors, np.float32).astype(np.longdouble)      # (a rope_freqs tensor is f32)
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "yarn":
        c = [rot * math.log(context / (2 * math.pi * r)) / (2 * math.log(base)) for r in (beta_fast, beta_slow)]
        low, high = max(math.floor(c[0]), 0), min(math.ceil(c[1]), rot - 1)
        y = np.clip((i - low) / max(high - low, 0.001), 0, 1)
        return f * (1 - y) + f / factor * y, 0.1 * math.log(factor) + 1
    return f, 1.0


def turned(x, pos, f, gain, layout):
    """x [T, H, d] in 64 bits, and the bound's |a| + |b| for each value."""
    rot = 2 * len(f)
    turns = pos.astype(np.longdouble)[:, None] * f[None, :] / (2 * np.longdouble(math.pi) + np.longdouble(1.2246467991473532e-16) * 2)
    ang = ((turns - np.floor(turns)) * 2 * np.longdouble(math.pi)).astype(np.float64)
    c, s = np.cos(ang)[:, None, :] * gain, np.sin(ang)[:, None, :] * gain
    ia, ib = (np.arange(rot // 2), np.arange(rot // 2) + rot // 2) if layout == "half" else (
        np.arange(0, rot, 2), np.arange(1, rot, 2))
    y, mag = x.copy(), np.zeros_like(x)
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    mag[..., ia] = mag[..., ib] = (np.abs(a) + np.abs(b)) * gain
    return y, mag


def bound(y, mag, dtype):
    return 8e-7 * mag + U[dtype] * (np.abs(y) + 8e-7 * mag) + (2.0 ** -25 if dtype == "float16" else 0)


CASES = [  # T, heads, d, rot, layout, type, what the plan scales
    (1, 1, 2, 2, "half", "float32", {}),
    (1, 32, 128, 128, "half", "float32", {}),
    (3, 28, 128, 128, "interleaved", "float16", {}),
    (5, 8, 96, 64, "half", "bfloat16", {}),
    (7, 5, 80, 32, "interleaved", "bfloat16", dict(scaling="linear", factor=8.0)),
    (65, 3, 80, 40, "half", "float16", {}),          # 20 pairs: not whole vectors
    (6, 2, 80, 40, "interleaved", "float32", {}),
    (9, 3, 36, 12, "half", "float32", {}),
    (2, 2, 512, 512, "half", "float16", {}),
    (4099, 2, 64, 64, "half", "bfloat16", dict(scaling="yarn", factor=4.0, context=8192)),
    (4097, 3, 24, 16, "interleaved", "float32", dict(scaling="yarn", factor=32.0, context=4096, beta_fast=16.0, beta_slow=2.0)),
    (33, 4, 128, 64, "half", "float32", dict(divisors=np.linspace(1.0, 8.0, 32))),
    (1, 200, 256, 256, "interleaved", "float16", {}),
    (8, 130, 254, 254, "half", "float32", {}),       # over 16384 pairs a token
]


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,d,rot,layout,dtype,more", CASES)
def test_apply(gpu, torch, T, H, d, rot, layout, dtype, more):
    rng = np.random.default_rng(T + d + rot)
    base = 10000.0 if d < 128 else 1e6
    rope = gpu.Rope(d, rot=rot, layout=layout, base=base, **more)
    x = torch.from_numpy(rng.standard_normal((T, H, d), dtype=np.float32)).to(getattr(torch, dtype)).cuda()
    pos = rng.integers(0, 131072, T)
    out = rope.apply(x, torch.from_numpy(pos.astype(np.int32)).cuda(), out=torch.full_like(x, 99.0))
    f, gain = frequencies(rot, base, **more)
    want, mag = turned(x.double().cpu().numpy(), pos, f, gain, layout)
    got = out.double().cpu().numpy()
    assert (np.abs(got - want) <= bound(want, mag, dtype)).all()
    assert (got[..., rot:] == want[..., rot:]).all()


@pytest.mark.gpu
def test_far_and_negative_positions(gpu, torch):
    """The angle is as exact at 2^31 as near 0; negative positions turn back."""
    x = torch.randn((6, 4, 128), device="cuda")
    pos = np.array([0, 1, -1, 2 ** 31 - 1, -2 ** 31, 123456789])
    rope = gpu.Rope(128, base=500000.0)
    out = rope.apply(x, torch.from_numpy(pos.astype(np.int32)).cuda(), out=torch.empty_like(x))
    f, gain = frequencies(128, 500000.0)
    want, mag = turned(x.double().cpu().numpy(), pos, f, gain, "half")
    # (the reference's own angle: 2^31 turns in 64 bits of mantissa, below 1e-9)
    assert (np.abs(out.double().cpu().numpy() - want) <= bound(want, mag, "float32") + 1e-8 * mag).all()
    assert torch.equal(out[0], x[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("offset", [0, 1])
def test_strides_and_in_place(gpu, torch, dtype, offset):
    """Heads inside a wider row (also where vectors would not be aligned), in
    place, on a stream of its own; what lies beside them stays."""
    T, H, d = 37, 3, 64
    wide = torch.randn((T, 5 * d + offset), device="cuda").to(getattr(torch, dtype))
    before = wide.clone()
    x = wide[:, d + offset:d + offset + H * d].unflatten(1, (H, d))
    pos = torch.arange(T, dtype=torch.int32, device="cuda") * 1000
    rope = gpu.Rope(d, rot=32, layout="interleaved")
    want = rope.apply(x.contiguous(), pos, out=torch.empty((T, H, d), dtype=x.dtype, device="cuda"))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        rope.apply(x, pos)
    s.synchronize()
    assert torch.equal(x, want)
    assert torch.equal(wide[:, :d + offset], before[:, :d + offset])
    assert torch.equal(wide[:, d + offset + H * d:], before[:, d + offset + H * d:])


@pytest.mark.gpu
def test_nothing_and_not_finite(gpu, torch):
    rope = gpu.Rope(64)
    x = torch.randn((0, 4, 64), device="cuda")
    rope.apply(x, torch.zeros(0, dtype=torch.int32, device="cuda"))
    x = torch.randn((2, 2, 64), device="cuda")
    x[1, 0, 3] = math.inf
    x[1, 1, 5] = math.nan
    y = rope.apply(x, torch.tensor([5, 6], dtype=torch.int32, device="cuda"), out=torch.empty_like(x))
    bad = ~torch.isfinite(y)
    want = torch.zeros_like(bad)
    want[1, 0, 3] = want[1, 0, 35] = want[1, 1, 5] = want[1, 1, 37] = True       # the pair, and nothing else
    assert torch.equal(bad, want)


def test_refusals_without_gpu():
    import gs_sampler as gs
    lib = gs.load_library()
    h = ctypes.c_void_p()

    def create(**kw):
        p = dict(d=128, rot=128, layout=1, scaling=0, base=1e4, factor=1.0, context=0, beta_fast=0.0, beta_slow=0.0, gain=0.0,
                 divisors=None)
        p.update(kw)
        return lib.gs_rope_create(ctypes.byref(gs.RopeParams(**p)), ctypes.byref(h))

    assert lib.gs_rope_create(None, ctypes.byref(h)) == gs.GS_ERR_INVALID
    assert lib.gs_rope_create(ctypes.byref(gs.RopeParams()), None) == gs.GS_ERR_INVALID
    for kw in (dict(d=0), dict(d=127), dict(rot=0), dict(rot=3), dict(rot=130), dict(layout=2), dict(base=1.0),
               dict(base=math.nan), dict(base=math.inf), dict(scaling=1, factor=0.5), dict(scaling=1, factor=math.nan),
               dict(scaling=2, factor=2.0), dict(scaling=2, factor=2.0, context=4096, beta_fast=-1.0), dict(gain=-1.0),
               dict(gain=math.nan)):
        assert create(**kw) == gs.GS_ERR_INVALID, kw
    div = np.ones(64, np.float32)
    div[7] = 0.0
    assert create(divisors=div.ctypes.data) == gs.GS_ERR_INVALID
    for kw in (dict(d=514, rot=64), dict(scaling=3)):
        assert create(**kw) == gs.GS_ERR_UNSUPPORTED, kw
    assert lib.gs_rope_destroy(None) == gs.GS_ERR_INVALID
    assert lib.gs_rope_apply(None, 0, 16, 128, 16, 128, 1, 1, 16, None) == gs.GS_ERR_INVALID


@pytest.mark.gpu
def test_refusals(gpu, torch):
    rope = gpu.Rope(64)
    lib, GS = rope._lib, gpu
    x = torch.zeros((4, 2, 64), device="cuda")
    pos = torch.zeros(4, dtype=torch.int32, device="cuda")
    p = x.data_ptr()
    call = lambda *a: lib.gs_rope_apply(rope._h, *a, pos.data_ptr(), None)  # noqa: E731
    assert call(7, p, 128, p, 128, 4, 2) == GS.GS_ERR_UNSUPPORTED
    assert call(0, None, 128, p, 128, 4, 2) == GS.GS_ERR_INVALID
    assert call(0, p, 127, p, 128, 4, 2) == GS.GS_ERR_INVALID          # heads would overlap the next token
    assert call(0, p, 128, p, 130, 4, 2) == GS.GS_ERR_INVALID          # in place with another stride
    assert call(0, p + 2, 128, p, 128, 4, 2) == GS.GS_ERR_INVALID
    assert lib.gs_rope_apply(rope._h, 0, p, 128, p, 128, 4, 2, None, None) == GS.GS_ERR_INVALID
    assert call(0, None, 0, None, 0, 0, 2) == GS.GS_OK                 # nothing to do
    with pytest.raises(ValueError):
        rope.apply(torch.zeros((4, 2, 32), device="cuda"), pos)
    with pytest.raises(TypeError):
        rope.apply(x.transpose(0, 1), pos)
    with pytest.raises(TypeError):
        rope.apply(x, pos.long())
    with pytest.raises(TypeError):
        rope.apply(x.double(), pos)


@pytest.mark.gpu
def test_more_tokens_than_a_grid_is_wide(gpu, torch):
    """Over 2^24 workgroups of four tokens."""
    T, H, d, dtype = 70000003, 1, 2, "bfloat16"
    rope = gpu.Rope(d, layout="half")
    x = torch.ones((T, H, d), dtype=getattr(torch, dtype), device="cuda")
    x[:, 0, 1] = 0.0
    pos = torch.arange(T, dtype=torch.int32, device="cuda")
    out = rope.apply(x, pos, out=torch.full_like(x, 99.0))
    for at in (slice(0, 1000), slice(T // 2, T // 2 + 1000), slice(T - 1000, T)):
        a, p = x[at].double().cpu().numpy(), pos[at].cpu().numpy()
        f, gain = frequencies(d, 10000.0)
        want, mag = turned(a, p, f, gain, "half")
        assert (np.abs(out[at].double().cpu().numpy() - want) <= bound(want, mag, dtype) + 1e-8 * mag).all()
    assert float(out.float().abs().max()) < 1.01
