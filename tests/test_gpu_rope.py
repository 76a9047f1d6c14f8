"""Rotary positions with head norms (ggq_rope_dev) against their formula in 64 bits.

Bounds: the angle is reduced in 64 bits and rounded to fp32 as a fraction of a half turn, at most pi * 2^-24 off; sine, cosine
(2 units of 2^-23) and the two products and their sum round a few times more: 2^-20 of |a| + |b| holds all of it.  The norm
adds its sum of up to 512 squares (8 in a lane, then pairwise: 17 roundings), division, root and two products:
another 2^-19 of the values.  fp16 results: half a step, 2^-11 of the value or 2^-25."""
import ctypes
import math

import numpy as np
import pytest

import ggnpu_amd.lib as gl
from tests.gpu_util import dev, host, ptr, stream_handle

pytestmark = pytest.mark.gpu
EPS = 1e-6


@pytest.fixture(scope="module")
def ctx():
    import torch
    assert torch.cuda.is_available()
    c = gl.Context(0)
    yield c
    c.close()


def frequencies(rot, base, scale=1.0, factors=None, yarn=1.0, yarn_ctx=4096, fast=32.0, slow=1.0):
    out = []
    lo = rot / 2 * math.log(yarn_ctx / (fast * 2 * math.pi), base)
    hi = rot / 2 * math.log(yarn_ctx / (slow * 2 * math.pi), base)
    lo, hi = max(0, math.floor(lo)), min(rot - 1, math.ceil(hi))
    for i in range(rot // 2):
        f = scale / base ** (2 * i / rot)
        if factors is not None:
            f /= float(np.float32(factors[i]))
        if yarn > 1:
            t = min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
            f = f * (1 - t) + f / yarn * t
        out.append(f)
    return np.array(out), 1.0 + 0.1 * math.log(yarn)


def plain(x, w, pos, f, mag, rot, layout):
    x = x.astype(np.float64)
    extra = 0.0
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + EPS) * w.astype(np.float64)
        extra = 2.0 ** -19
    a, b = (slice(0, rot // 2), slice(rot // 2, rot)) if layout == 0 else (slice(0, rot, 2), slice(1, rot, 2))
    ang = pos.astype(np.float64)[:, None, None] * f
    c, s = np.cos(ang) * mag, np.sin(ang) * mag
    y, tol = x.copy(), np.abs(x) * extra
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    both = (np.abs(x[..., a]) + np.abs(x[..., b])) * mag * (2.0 ** -20 + extra)
    tol[..., a], tol[..., b] = both, both
    return y, tol + 1e-37


def case(ctx, seed, n, nq, nk, hd, rot=0, layout=0, norm=False, out_type=0, pos=None, pad=0, in_place=False, base=10000.0,
         scale=1.0, factors=None, yarn=1.0):
    import torch
    rng = np.random.default_rng(seed)
    r = rot or hd
    h = gl.Rope(ctx, hd, rot, layout, base, position_scale=scale, freq_factors=factors, yarn_factor=yarn, yarn_ctx=4096)
    f, mag = frequencies(r, base, scale, factors, yarn)
    pos = rng.integers(0, 5000, n).astype(np.int32) if pos is None else np.asarray(pos, np.int32)
    sets, keep, xs = (gl.RopeHeads * 2)(), [], []
    for i, heads in enumerate((nq, nk)):
        if not heads:
            continue
        x = (rng.standard_normal((n, heads * hd + pad)) * 3).astype(np.float32)
        w = (1 + 0.2 * rng.standard_normal(hd)).astype(np.float32) if norm else None
        dx = dev(x)
        ld = heads * hd + pad
        dy = dx if in_place else torch.full((n, ld), 7.0, dtype=torch.float16 if out_type else torch.float32, device="cuda")
        dw = dev(w) if norm else None
        s = sets[i]
        s.x, s.ldx, s.n_head, s.out, s.ldo, s.out_type = dx.data_ptr(), ld, heads, dy.data_ptr(), ld, out_type
        s.norm_w = dw.data_ptr() if norm else None
        keep.append((dx, dy, dw))
        xs.append((x, w, heads))
    dp = dev(pos)
    ctx.check(ctx.lib.ggq_rope_dev(ctx.h, h.h, sets, len(xs), ptr(dp), n, EPS, stream_handle()), "rope")
    for (x, w, heads), (_, dy, _) in zip(xs, keep):
        got = host(dy).astype(np.float64)
        want, tol = plain(x[:, : heads * hd].reshape(n, heads, hd), w, pos, f, mag, r, layout)
        if out_type:
            tol = tol + np.abs(want) * 2.0 ** -11 + 2.0 ** -25
        err = np.abs(got[:, : heads * hd].reshape(n, heads, hd) - want)
        assert (err <= tol).all(), (np.argwhere(err > tol)[:4], err.max())
        # values between the rows are left alone
        rest = got[:, heads * hd:]
        assert np.array_equal(rest, x[:, heads * hd:].astype(np.float64) if in_place else np.full_like(rest, 7.0))
    h.close()


@pytest.mark.parametrize("n,nq,nk,hd,rot,layout,norm", [
    (1, 32, 8, 64, 0, 0, False),     # one token, Llama-3.2-1B heads
    (1, 1, 0, 8, 0, 0, False),       # the smallest head, no keys
    (3, 16, 8, 128, 0, 0, True),     # Qwen3-0.6B heads with their norms
    (7, 16, 2, 256, 64, 0, True),    # a quarter of a wide head
    (5, 3, 1, 80, 32, 1, False),     # 80-wide heads, part of them, interleaved
    (4, 5, 5, 96, 0, 1, True),       # lanes that hold nothing
    (2, 2, 1, 512, 504, 0, True),    # the widest head
    (300, 12, 2, 128, 0, 0, False),  # many rows
    (2049, 2, 1, 64, 8, 1, False),   # the smallest rotated part
])
@pytest.mark.parametrize("out_type", [0, 1])
def test_rope(ctx, n, nq, nk, hd, rot, layout, norm, out_type):
    case(ctx, n + hd + out_type, n, nq, nk, hd, rot, layout, norm, out_type)


def test_rope_enough_rows_for_several_passes(ctx):
    case(ctx, 3, 1500, 32, 8, 128, norm=True)
    case(ctx, 4, 1501, 9, 4, 64, 32, 1)


@pytest.mark.parametrize("kw", [dict(base=500000.0, factors=list(np.linspace(1, 8, 32))), dict(yarn=8.0), dict(scale=0.25),
                                dict(yarn=32.0, base=1e6, factors=list(np.linspace(0.5, 3, 32)))])
def test_rope_long_context_scaling(ctx, kw):
    case(ctx, 5, 9, 4, 2, 64, pos=[0, 1, 2, 4095, 4096, 32768, 131071, 1 << 20, 7], **kw)


def test_rope_far_and_negative_positions(ctx):
    """2^31 - 1 turns' fractions come from the 64-bit product; position 0 changes nothing."""
    case(ctx, 6, 6, 4, 2, 128, pos=[0, 2 ** 31 - 1, -2 ** 31, -1, 2 ** 24 + 1, 1000003])


@pytest.mark.parametrize("norm", [False, True])
def test_rope_in_place_and_strided_rows(ctx, norm):
    case(ctx, 7, 33, 8, 2, 64, norm=norm, pad=8, in_place=True)
    case(ctx, 8, 33, 8, 2, 64, 48, 1, norm=norm, pad=24)
    case(ctx, 9, 33, 8, 2, 64, norm=norm, pad=24, out_type=1)


def test_rope_into_a_cache_slab(ctx):
    """Keys turned straight into their rows of a slab; the rest of the slab stays."""
    import torch
    rng = np.random.default_rng(0)
    hd, nk, n, at, ctx_len = 64, 2, 5, 11, 40
    k = rng.standard_normal((n, nk * hd)).astype(np.float32)
    slab = torch.full((ctx_len, nk * hd), 3.0, device="cuda")
    pos = np.arange(at, at + n, dtype=np.int32)
    h = gl.Rope(ctx, hd)
    sets = (gl.RopeHeads * 1)()
    dk, dp = dev(k), dev(pos)
    sets[0].x, sets[0].ldx, sets[0].n_head = dk.data_ptr(), nk * hd, nk
    sets[0].out, sets[0].ldo, sets[0].out_type = slab[at].data_ptr(), nk * hd, 0
    ctx.check(ctx.lib.ggq_rope_dev(ctx.h, h.h, sets, 1, ptr(dp), n, EPS, stream_handle()), "rope")
    got = host(slab)
    f, mag = frequencies(hd, 10000.0)
    want, tol = plain(k.reshape(n, nk, hd), None, pos, f, mag, hd, 0)
    assert (np.abs(got[at:at + n].reshape(n, nk, hd) - want) <= tol).all()
    assert (np.delete(got, slice(at, at + n), 0) == 3.0).all()


def test_rope_nan_stays_in_its_head(ctx):
    import torch
    x = torch.ones((2, 3, 64), device="cuda")
    x[0, 1, 5] = float("nan")
    x[1, 2, 63] = float("inf")
    w = torch.ones(64, device="cuda")
    out = torch.empty_like(x)
    h = gl.Rope(ctx, 64, 32)
    sets = (gl.RopeHeads * 1)()
    s = sets[0]
    s.x, s.ldx, s.n_head, s.out, s.ldo, s.out_type, s.norm_w = x.data_ptr(), 192, 3, out.data_ptr(), 192, 0, w.data_ptr()
    pos = torch.tensor([3, 4], dtype=torch.int32, device="cuda")
    ctx.check(ctx.lib.ggq_rope_dev(ctx.h, h.h, sets, 1, ptr(pos), 2, EPS, stream_handle()), "rope")
    bad = torch.isnan(out).any(-1).cpu()
    assert bad.tolist() == [[False, True, False], [False, False, True]]


def test_rope_refusals(ctx):
    import torch
    lib, out = ctx.lib, ctypes.c_void_p()

    def create(**kw):
        kw.setdefault("head_dim", 64)
        return lib.ggq_rope_create(ctx.h, ctypes.byref(gl.RopeParams(**kw)), ctypes.byref(out))
    for kw in (dict(head_dim=0), dict(head_dim=60), dict(head_dim=520), dict(rot_dim=72), dict(rot_dim=12), dict(rot_dim=-8),
               dict(layout=2), dict(base=-1.0), dict(base=float("nan")), dict(position_scale=float("inf")),
               dict(yarn_factor=0.5, yarn_ctx=4096), dict(yarn_factor=4.0), dict(yarn_factor=4.0, yarn_ctx=4096, yarn_beta_fast=-1.0),
               dict(yarn_factor=4.0, yarn_ctx=4096, base=1.0)):
        assert create(**kw) == gl.Status.INVALID_PARAM and not out.value, kw
    f = (ctypes.c_float * 32)(*([1.0] * 31 + [0.0]))
    assert create(freq_factors=ctypes.addressof(f)) == gl.Status.INVALID_PARAM
    h = gl.Rope(ctx, 64)
    x = torch.zeros(4096, device="cuda")
    pos = torch.zeros(4, dtype=torch.int32, device="cuda")

    def call(n_sets=1, n_tok=2, handle=None, pos_ptr=None, **kw):
        sets = (gl.RopeHeads * 2)()
        d = dict(x=x.data_ptr(), ldx=128, n_head=2, out=x.data_ptr() + 8192, ldo=128, out_type=0)
        d.update(kw)
        for k, v in d.items():
            setattr(sets[0], k, v)
        return lib.ggq_rope_dev(ctx.h, handle or h.h, sets, n_sets, pos_ptr or ptr(pos), n_tok, EPS, stream_handle())
    assert call() == gl.Status.OK and call(n_tok=0) == gl.Status.OK
    for kw in (dict(n_sets=0), dict(n_sets=3), dict(n_tok=-1), dict(ldx=127), dict(ldo=64), dict(n_head=0), dict(out_type=12),
               dict(x=x.data_ptr() + 4), dict(out=x.data_ptr() + 8196), dict(norm_w=x.data_ptr() + 8), dict(ldx=130),
               dict(ldo=130), dict(ldo=132, out_type=1), dict(x=None), dict(out=None), dict(handle=ctypes.c_void_p(16)),
               dict(out=x.data_ptr(), ldo=132), dict(out=x.data_ptr(), out_type=1)):
        assert call(**kw) == gl.Status.INVALID_PARAM, kw
    assert lib.ggq_rope_dev(ctx.h, h.h, (gl.RopeHeads * 2)(), 1, None, 1, EPS, None) == gl.Status.INVALID_PARAM
    assert lib.ggq_rope_free(ctx.h, ctypes.c_void_p(16)) == gl.Status.INVALID_PARAM
    h.close()
    with pytest.raises(ValueError):
        gl.Rope(ctx, 64, freq_factors=[1.0] * 5)


@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("far", [0, 100000])
def test_rope_angles_keep_their_bits(ctx, layout, far):
    """Pairs (1, 0) turned: the cosines and sines themselves.  An angle rounded to 32 bits as a part of half a turn is off by
    up to 2^-25 of it, uniformly: over all angles 4.1e-8 rad, root mean square, along the circle.  Sine and cosine
    rounded twice, with a function that is itself within half a unit in the mean, stay below 3e-8: the bound is between."""
    import torch
    n, hd = 1000, 256
    x = np.zeros((n, 1, hd), np.float32)
    a, b = (slice(0, hd // 2), slice(hd // 2, hd)) if layout == 0 else (slice(0, hd, 2), slice(1, hd, 2))
    x[..., a] = 1
    pos = np.arange(far, far + n, dtype=np.int32)
    h = gl.Rope(ctx, hd, 0, layout, 10000.0)
    dx, dp = dev(x), dev(pos)
    out = torch.empty((n, 1, hd), device="cuda")
    sets = (gl.RopeHeads * 1)()
    sets[0].x, sets[0].ldx, sets[0].n_head, sets[0].out, sets[0].ldo = dx.data_ptr(), hd, 1, out.data_ptr(), hd
    ctx.check(ctx.lib.ggq_rope_dev(ctx.h, h.h, sets, 1, ptr(dp), n, EPS, stream_handle()), "rope")
    got = host(out).astype(np.float64)[:, 0]
    ang = pos[:, None] * frequencies(hd, 10000.0)[0][:40]  # the pairs that turn often over these positions
    c, s = np.cos(ang), np.sin(ang)
    along = (got[:, b][:, :40] - s) * c - (got[:, a][:, :40] - c) * s
    assert np.sqrt((along ** 2).mean()) <= 3.6e-8
    h.close()
