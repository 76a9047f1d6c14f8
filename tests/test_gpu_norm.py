"""ggq_norm_dev against 64 bits: the sum rounded once, the rows rounded once, the codes those of the rows."""
import numpy as np
import pytest

import ggnpu_amd.lib as gl
from tests import step_util as su
from tests.gpu_util import host, ptr, stream_handle

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import torch
    assert torch.cuda.is_available()
    c = gl.Context(0)
    yield c
    c.close()


def t(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def padded(x, pad, fill=77.0):
    b = np.full((x.shape[0], x.shape[1] + pad), fill, np.float32)
    b[:, : x.shape[1]] = x
    return t(b)


def call(ctx, x, add=None, want_sum=False, w=None, norm_len=0, eps=1e-6, gate=None, want_out=True, act=0, pad=0, over=None):
    """dict of outputs; over: "x" or "add" (the sum goes there) or "out" (the rows go over x)."""
    import torch
    n, K = x.shape
    ld = K + pad
    bx, ba, bg = padded(x, pad), None if add is None else padded(add, pad), None if gate is None else padded(gate, pad)
    bs = {"x": bx, "add": ba}.get(over) if over in ("x", "add") else torch.full((n, ld), 5.0, device="cuda")
    bo = bx if over == "out" else torch.full((n, ld), 5.0, device="cuda")
    codes = torch.full((n, K), 99, dtype=torch.int8, device="cuda")
    scales = torch.full((n, 1 if act == 1 else max(1, K // 32)), -1.0, device="cuda")
    bw = None if w is None else t(w)
    p = gl.NormParams(n_rows=n, n_cols=K, x=bx.data_ptr(), ldx=ld, norm_len=norm_len, eps=eps, act_mode=act)
    if add is not None:
        p.add, p.ld_add = ba.data_ptr(), ld
    if want_sum:
        p.sum, p.ld_sum = bs.data_ptr(), ld
    if w is not None:
        p.norm_w = bw.data_ptr()
    if gate is not None:
        p.gate, p.ld_gate = bg.data_ptr(), ld
    if want_out:
        p.out, p.ldo = bo.data_ptr(), ld
    if act:
        p.codes, p.scales = codes.data_ptr(), scales.data_ptr()
    ctx.check(ctx.lib.ggq_norm_dev(ctx.h, p, stream_handle()), "norm")
    r = {}
    for name, b, on in (("sum", bs, want_sum), ("out", bo, want_out)):
        if on:
            h = host(b)
            r[name] = h[:, :K]
            assert (h[:, K:] == h[0, K:K + 1]).all() if pad else True  # what lies between the rows stays
    if act:
        r["codes"], r["scales"] = host(codes), host(scales)
    return r


def check(r, x, add=None, w=None, norm_len=0, eps=1e-6, gate=None, act=0):
    s, y = su.norm(x, add, w, norm_len, eps, gate)
    if "sum" in r:
        assert np.array_equal(r["sum"], s)
    out = r.get("out")
    if out is not None:
        # one rounding of what 64 bits give, which both sides have to about 2^-50
        tol = np.abs(y) * su.U32 * (1 + 2.0 ** -20) + 2.0 ** -150
        err = np.abs(out.astype(np.float64) - y)
        assert (err <= tol).all(), (np.argwhere(err > tol)[:4], err.max())
    if act and out is not None:
        q, sc = su.codes(out, 32 if act == 2 else 0)
        assert np.array_equal(r["scales"].reshape(sc.shape), sc) and np.array_equal(r["codes"], q)


def rows(rng, n, K):
    return (rng.standard_normal((n, K)) * np.where(rng.random(K) < 0.03, 20, 1)).astype(np.float32)


@pytest.mark.parametrize("K", [4, 32, 36, 252, 256, 260, 512, 516, 1000, 1024, 2048, 2052, 4096, 4100, 8192, 8196, 16384, 20000, 32768])
@pytest.mark.parametrize("n", [1, 3])
def test_widths(ctx, K, n):
    rng = np.random.default_rng(K + n)
    x, add, w = rows(rng, n, K), rows(rng, n, K), (1 + 0.2 * rng.standard_normal(K)).astype(np.float32)
    for act in (0, 1) + ((2,) if K % 32 == 0 else ()):
        check(call(ctx, x, add, True, w, act=act), x, add, w, act=act)


@pytest.mark.parametrize("K,L", [(128, 4), (128, 8), (96, 12), (512, 64), (960, 80), (4096, 128), (1152, 96), (2048, 256), (4096, 512), (2560, 20),
                                 (32768, 128), (30720, 1024)])
@pytest.mark.parametrize("gated", [False, True])
def test_heads(ctx, K, L, gated):
    rng = np.random.default_rng(K + L)
    x, w = rows(rng, 5, K), (1 + 0.2 * rng.standard_normal(L)).astype(np.float32)
    gate = (3 * rng.standard_normal((5, K))).astype(np.float32) if gated else None
    for act in (0, 1, 2):
        check(call(ctx, x, w=w, norm_len=L, gate=gate, act=act, pad=4), x, w=w, norm_len=L, gate=gate, act=act)


@pytest.mark.parametrize("over", ["x", "add", "out"])
@pytest.mark.parametrize("K", [64, 4096])
def test_in_place(ctx, over, K):
    rng = np.random.default_rng(7)
    x, add = rows(rng, 9, K), rows(rng, 9, K)
    check(call(ctx, x, add, True, over=over, act=1, pad=8), x, add, act=1)


def test_what_is_not_asked_for(ctx):
    """Codes alone equal the codes beside the rows; a sum alone; a gate without heads."""
    rng = np.random.default_rng(8)
    x, add, g = rows(rng, 33, 2048), rows(rng, 33, 2048), rows(rng, 33, 2048)
    a, b = call(ctx, x, add, act=1, want_out=False), call(ctx, x, add, act=1)
    assert np.array_equal(a["codes"], b["codes"]) and np.array_equal(a["scales"], b["scales"]) and "out" not in a
    assert np.array_equal(call(ctx, x, add, True, want_out=False)["sum"], x + add)
    check(call(ctx, x, gate=g, eps=0.5), x, gate=g, eps=0.5)


def test_many_rows_and_equal_ones(ctx):
    """Rows do not depend on each other: equal ones have equal results."""
    rng = np.random.default_rng(9)
    x = np.tile(rows(rng, 7, 260), (700, 1))
    r = call(ctx, x, act=1)
    for k in ("out", "codes"):
        assert np.array_equal(r[k], np.tile(r[k][:7], (700, 1)))
    check(r, x, act=1)


def test_zeros_and_extremes(ctx):
    x = np.zeros((6, 128), np.float32)
    x[1, 5] = 1e-38
    x[2] = 3e38          # squares beyond fp32
    x[3, ::2] = 1e-30
    x[4, 0], x[4, 1] = 3e38, 1e-30
    x[5, 3] = 1e-45
    gate = np.full((6, 128), -200.0, np.float32)  # silu next to nothing
    for act in (0, 1, 2):
        check(call(ctx, x, act=act), x, act=act)
    check(call(ctx, x, gate=gate), x, gate=gate)
    r = call(ctx, x, act=1)
    assert (r["codes"][0] == 0).all() and r["scales"][0, 0] == 1


def test_rows_that_are_not_finite_spoil_themselves_only(ctx):
    rng = np.random.default_rng(10)
    x = rows(rng, 4, 1024)
    y = x.copy()
    y[1, 3], y[2, 9] = np.inf, np.nan
    a, b = call(ctx, x, act=1), call(ctx, y, act=1)
    for r in (0, 3):
        assert np.array_equal(a["out"][r], b["out"][r]) and np.array_equal(a["codes"][r], b["codes"][r])
    assert np.isnan(b["out"][1, 3]) and np.isnan(b["out"][2]).all()


def test_refusals(ctx):
    import torch
    lib, bad = ctx.lib, gl.Status.INVALID_PARAM
    b = torch.zeros(1 << 16, device="cuda")
    q = torch.zeros(1 << 16, dtype=torch.int8, device="cuda")
    P = b.data_ptr()
    ok = dict(n_rows=2, n_cols=64, x=P, ldx=64, out=P + 4096, ldo=64, eps=1e-6)

    def st(**kw):
        return lib.ggq_norm_dev(ctx.h, gl.NormParams(**{**ok, **kw}), stream_handle())

    assert st() == 0 and st(n_rows=0, x=None) == 0
    for kw in (dict(n_rows=-1), dict(n_cols=0), dict(n_cols=66), dict(n_cols=32772, ldx=40000, ldo=40000), dict(x=None), dict(ldx=60),
               dict(ldx=66), dict(x=P + 4), dict(out=P + 4100), dict(out=None), dict(norm_len=48), dict(norm_len=2), dict(norm_len=-64),
               dict(norm_len=128), dict(eps=-1.0), dict(eps=float("nan")), dict(act_mode=3), dict(act_mode=-1), dict(act_mode=1),
               dict(act_mode=1, codes=q.data_ptr()), dict(act_mode=1, scales=P), dict(act_mode=1, codes=q.data_ptr() + 4, scales=P),
               dict(act_mode=2, n_cols=48, codes=q.data_ptr(), scales=P), dict(add=P + 8192, ld_add=32), dict(add=P + 8196, ld_add=64),
               dict(gate=P + 8192, ld_gate=0), dict(norm_w=P + 4), dict(sum=P, ld_sum=68), dict(out=P, ldo=68),
               dict(sum=P + 4096, ld_sum=64)):
        assert st(**kw) == bad, kw
        assert ctx.lib.ggq_last_error_message(ctx.h)
    torch.cuda.synchronize()


def test_more_rows_than_a_grid_dimension_holds(ctx):
    """2^26 + 3 rows of 4 values: 64 threads each are more than 2^32."""
    import torch
    n = (1 << 26) + 3
    x, out = torch.full((n, 4), 2.0, device="cuda"), torch.zeros((n, 4), device="cuda")
    at = [0, 1, (1 << 20) - 1, 1 << 20, (1 << 25) + 5, n - 2, n - 1]
    rng = np.random.default_rng(0)
    some = rng.standard_normal((len(at), 4)).astype(np.float32)
    x[at] = t(some)
    p = gl.NormParams(n_rows=n, n_cols=4, x=x.data_ptr(), ldx=4, eps=0.0, out=out.data_ptr(), ldo=4)
    ctx.check(ctx.lib.ggq_norm_dev(ctx.h, p, stream_handle()), "norm")
    want = su.norm(some, eps=0.0)[1]
    got = host(out[at])
    assert (np.abs(got - want) <= (1 + 2.0 ** -20) * su.U32 * np.abs(want)).all()
    rest = torch.ones(n, dtype=torch.bool, device="cuda")
    rest[at] = False
    assert bool((out[rest] == 1.0).all())


@pytest.mark.parametrize("cols", [256, 4096, 30000])
def test_gates_of_all_sizes(ctx, cols):
    """Gates from tiny to infinite: z / (1 + exp(-z)) of 64 bits (rounded once, half a subnormal step where that is the step)."""
    rng = np.random.default_rng(cols)
    z = np.array([-np.inf, np.inf, np.nan, -1e30, -800, -709.5, -700.1, -699.9, -104, -100, -88, -20, -1, -1e-30, -0.0, 0.0, 1e-40, 1e-8, 0.5, 3, 40,
                  699, 701, 900, 1e38], np.float32)
    gate = np.resize(z, (3, cols)).astype(np.float32)
    gate[2] = (rng.standard_normal(cols) * np.exp2(rng.integers(-20, 10, cols))).astype(np.float32)
    x = rng.standard_normal((3, cols)).astype(np.float32)
    got = call(ctx, x, gate=gate)["out"]
    with np.errstate(all="ignore"):
        want = su.norm(x, gate=gate)[1]
        f32 = want.astype(np.float32)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.isinf(got), np.isinf(f32))
    at = np.isfinite(f32)
    assert (np.abs(got[at] - want[at]) <= (1 + 2.0 ** -20) * su.U32 * np.abs(want[at]) + 2.0 ** -150).all()


@pytest.mark.parametrize("norm_len", [0, 64, 128, 96])
def test_rows_of_all_sizes_without_eps(ctx, norm_len):
    """Square sums from 1e-76 to 1e76, and of nothing: NaN as 0 / 0 is."""
    rng = np.random.default_rng(norm_len)
    x = rng.standard_normal((6, 384)).astype(np.float32) * np.float32([[1e-38], [1e-20], [1], [1e18], [1e37], [0]])
    got = call(ctx, x, norm_len=norm_len, eps=0.0)["out"]
    want = su.norm(x, norm_len=norm_len, eps=0.0)[1]
    assert np.isnan(got[5]).all()
    assert (np.abs(got[:5] - want[:5]) <= (1 + 2.0 ** -20) * su.U32 * np.abs(want[:5])).all()


@pytest.mark.parametrize("K,L", [(32768, 512), (32768, 8192), (32768, 16384), (32736, 1488)])
def test_long_groups_of_the_longest_rows(ctx, K, L):
    """Groups that are no power of two of lanes up to a wavefront's, in rows whose groups' sums take 64 KiB of LDS and what the rest takes."""
    rng = np.random.default_rng(L)
    x, w = rows(rng, 3, K), (1 + 0.2 * rng.standard_normal(L)).astype(np.float32)
    gate = (3 * rng.standard_normal((3, K))).astype(np.float32)
    for g in (None, gate):
        for act in (0, 1, 2):
            check(call(ctx, x, w=w, norm_len=L, gate=g, act=act), x, w=w, norm_len=L, gate=g, act=act)


def test_overlaps_that_are_refused(ctx):
    """The sum may go over x or add and the rows over x; nothing goes over the gate, the rows not over add or the sum."""
    import torch
    b = torch.zeros(1 << 16, device="cuda")
    P = b.data_ptr()
    ok = dict(n_rows=2, n_cols=64, x=P, ldx=64, add=P + 4096, ld_add=64, gate=P + 8192, ld_gate=64, out=P + 16384, ldo=64, sum=P + 32768, ld_sum=64, eps=1e-6)
    st = lambda **kw: ctx.lib.ggq_norm_dev(ctx.h, gl.NormParams(**{**ok, **kw}), stream_handle())  # noqa: E731
    assert st() == 0 and st(sum=P) == 0 and st(sum=P + 4096) == 0 and st(out=P) == 0
    for kw in (dict(sum=P + 8192), dict(out=P + 4096), dict(out=P + 8192), dict(out=P + 32768), dict(out=P, sum=P)):
        assert st(**kw) == gl.Status.INVALID_PARAM, kw
    torch.cuda.synchronize()


@pytest.mark.parametrize("act", [1, 2])
@pytest.mark.parametrize("K", [96, 2048, 20000])
def test_codes_are_those_of_the_quantizer(ctx, K, act):
    """Codes and scales beside the rows are what ggq_quantize_act_dev makes of these, also of rows with numbers that are not finite."""
    import torch
    rng = np.random.default_rng(K)
    x = rows(rng, 8, K)
    x[1, 5], x[2, K - 1], x[3, ::3], x[4] = np.nan, np.inf, -np.inf, 0
    x[5] *= 1e30
    gate = (3 * rng.standard_normal((8, K))).astype(np.float32)
    gate[6, 7], gate[7, 40:60] = np.inf, np.nan
    r = call(ctx, x, gate=gate, act=act, eps=0.0)
    y = t(r["out"])
    q = torch.empty((8, K), dtype=torch.int8, device="cuda")
    sc = torch.empty(r["scales"].shape, device="cuda")
    ctx.check(ctx.lib.ggq_quantize_act_dev(ctx.h, ptr(y), K, 8, K, act, ptr(q), ptr(sc), stream_handle()), "quantize")
    assert np.array_equal(r["codes"], host(q)) and np.array_equal(r["scales"], host(sc), equal_nan=True)
