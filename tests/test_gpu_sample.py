"""ggq_sample_dev against the definition in 64 bits.  A token has to be the one of the definition unless u lies within 2^-30
of a border of the running sum (no such u is used: the distance is checked first)."""
import ctypes

import numpy as np
import pytest

import ggnpu_amd.lib as gl
from tests import step_util as su
from tests.gpu_util import host, stream_handle

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import torch
    assert torch.cuda.is_available()
    c = gl.Context(0)
    yield c
    c.close()


def t(a, dtype=None):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a, dtype)).cuda()


def call(ctx, x, u, temp=None, k=None, p=None, m=None, pad=0, prob=True, offset=0):
    import torch
    n, V = x.shape
    ld = V + pad
    b = np.full(n * ld + offset, 1e30, np.float32)  # (between the rows: larger than any logit)
    b[offset:].reshape(n, ld)[:, :V] = x
    b = t(b)
    arrays = [None if a is None else t(np.broadcast_to(a, n), d) for a, d in ((temp, np.float32), (k, np.int32), (p, np.float32), (m, np.float32))]
    uu = t(np.broadcast_to(u, n), np.float32)
    tok = torch.full((n + 1,), -7, dtype=torch.int32, device="cuda")
    pr = torch.full((n + 1,), -7.0, device="cuda")
    ptr = lambda a: None if a is None else a.data_ptr()  # noqa: E731
    s = gl.SampleParams(n_rows=n, n_vocab=V, logits=b.data_ptr() + 4 * offset, ld=ld, temperature=ptr(arrays[0]), top_k=ptr(arrays[1]),
                        top_p=ptr(arrays[2]), min_p=ptr(arrays[3]), u=uu.data_ptr(), token=tok.data_ptr(), prob=pr.data_ptr() if prob else None)
    ctx.check(ctx.lib.ggq_sample_dev(ctx.h, s, stream_handle()), "sample")
    tok, pr = host(tok), host(pr)
    assert tok[n] == -7 and pr[n] == -7 and (prob or (pr == -7).all())
    return tok[:n], pr[:n]


def check(ctx, x, u, temp=None, k=None, p=None, m=None, **kw):
    n = len(x)
    tok, pr = call(ctx, x, u, temp, k, p, m, **kw)
    at = lambda a, d, i: d if a is None else np.broadcast_to(a, n)[i]  # noqa: E731
    for i in range(n):
        want, prob, near = su.sample(x[i], at(temp, 1.0, i), int(at(k, 0, i)), at(p, 1.0, i), at(m, 0.0, i), float(np.broadcast_to(u, n)[i]))
        assert near > su.BORDER, "the test's u lies on a border"
        assert tok[i] == want, (i, tok[i], want, pr[i], prob)
        if kw.get("prob", True):
            # rounded once from weights and sums within 2^-30
            assert abs(pr[i] - prob) <= prob * (su.U32 + 2.0 ** -29), (i, pr[i], prob)


def logits(rng, n, V, spread=2.5, peaks=6):
    x = rng.standard_normal((n, V)) * spread
    for i in range(n):
        x[i, rng.integers(0, V, peaks)] = x[i].max() + rng.random(peaks) * 2
    return x.astype(np.float32)


@pytest.mark.parametrize("V", [1, 2, 3, 63, 64, 65, 511, 4095, 4096, 4097, 8192, 12289, 32003, 128256])
def test_vocabularies(ctx, V):
    rng = np.random.default_rng(V)
    x = logits(rng, 4, V)
    u = rng.random(4).astype(np.float32)
    check(ctx, x, u)
    check(ctx, x, u, temp=0.7, k=5, p=0.9, m=0.02, pad=3, offset=1)
    check(ctx, x, u, temp=[0.0, 0.5, 1.3, -1.0], p=0.5)


@pytest.mark.parametrize("k", [1, 2, 40, 127, 128, 129, 1000, 5000, 40000])
@pytest.mark.parametrize("p", [None, 0.9])
def test_top_k(ctx, k, p):
    rng = np.random.default_rng(k)
    check(ctx, logits(rng, 6, 40001), rng.random(6).astype(np.float32), temp=0.9, k=k, p=p)


@pytest.mark.parametrize("spread", [0.3, 2.5, 8.0])
@pytest.mark.parametrize("p", [0.0, 0.01, 0.3, 0.8, 0.95, 0.999, 0.99999994])
def test_top_p(ctx, spread, p):
    rng = np.random.default_rng(int(spread * 10))
    x = logits(rng, 5, 30011, spread)
    u = rng.random(5).astype(np.float32)
    check(ctx, x, u, p=p)
    check(ctx, x, u, p=p, k=700, temp=1.5)


@pytest.mark.parametrize("m", [1e-8, 1e-3, 0.05, 0.5, 0.999, 1.0, 3.0])
def test_min_p(ctx, m):
    rng = np.random.default_rng(3)
    x = logits(rng, 5, 20000)
    u = rng.random(5).astype(np.float32)
    check(ctx, x, u, m=m, temp=0.8)
    check(ctx, x, u, m=m, k=300, p=0.97)


def test_each_row_has_its_own(ctx):
    rng = np.random.default_rng(4)
    n = 40
    x = logits(rng, n, 5003)
    temp = np.where(np.arange(n) % 5 == 0, 0, rng.uniform(0.2, 3, n))
    k, p, m = rng.integers(-1, 60, n), rng.uniform(0.1, 1.2, n), rng.uniform(-0.1, 0.3, n)
    check(ctx, x, rng.random(n).astype(np.float32), temp.astype(np.float32), k, p.astype(np.float32), m.astype(np.float32))


@pytest.mark.parametrize("V", [1000, 9000, 50000])
def test_equal_logits(ctx, V):
    """All alike: the head of the order is that of the indices, also where thousands of tokens share a place."""
    x = np.full((3, V), 1.25, np.float32)
    x[1, 7] = 2.0
    x[2, V // 2:] = -3.0
    u = np.array([0.3, 0.71, 0.999], np.float32)
    check(ctx, x, u)
    check(ctx, x, u, k=V // 3)
    check(ctx, x, u, p=0.25)
    check(ctx, x, u, k=V // 2 + 11, p=0.5)


def test_few_values(ctx):
    """Thousands of tokens in each of a few places (as coarse logits have them), the border inside of one."""
    rng = np.random.default_rng(5)
    x = np.round(rng.standard_normal((6, 60000)) * 1.5).astype(np.float32)
    u = rng.random(6).astype(np.float32)
    for kw in (dict(k=5000), dict(p=0.6), dict(k=20000, p=0.7), dict(m=0.3, p=0.9), dict(k=3)):
        check(ctx, x, u, **kw)


def test_crowded_values(ctx):
    """Values a last bit apart: tens of thousands of keys in one bin."""
    rng = np.random.default_rng(6)
    x = (1.0 + rng.integers(0, 1 << 16, (4, 30000)) * 2.0 ** -23).astype(np.float32)
    u = rng.random(4).astype(np.float32)
    for kw in (dict(k=9999), dict(p=0.37), dict(k=200), dict(k=25000, p=0.9)):
        check(ctx, x, u, **kw)


def test_u_at_its_ends(ctx):
    """u = 0 takes the first kept token; what is below its smallest step of 1 the last that has a weight; nonsense counts as 0."""
    rng = np.random.default_rng(7)
    x = logits(rng, 1, 7001)
    kept = lambda **kw: np.flatnonzero([su.sample(x[0], u=0, **kw)[0] == i for i in range(7001)])  # noqa: E731
    for kw in (dict(top_k=9), dict()):
        first = kept(**kw)[0]
        k = kw.get("top_k")
        for u in (0.0, -1.0, np.nan):
            assert call(ctx, x, u, k=k)[0][0] == first
        last = su.sample(x[0], u=0.99999994, **kw)[0]
        assert call(ctx, x, 0.99999994, k=k)[0][0] == last
    # above 1: the last token with a weight
    order = np.argsort(-x[0], kind="stable")[:9]
    assert call(ctx, x, 1.0, k=9)[0][0] == order.max() and call(ctx, x, 5.0, k=9)[0][0] == order.max()


def test_not_numbers_and_infinities(ctx):
    rng = np.random.default_rng(8)
    x = logits(rng, 7, 10007)
    x[0, :5000] = -np.inf
    x[1, ::3] = np.nan
    x[2] = -np.inf
    x[3] = np.nan
    x[4, 77], x[4, 9000] = np.inf, np.inf
    x[5, :] = -np.inf
    x[5, 10006] = -3e38
    x[6] *= 1e30
    u = np.array([0.2, 0.9, 0.5, 0.5, 0.7, 0.3, 0.6], np.float32)
    for kw in (dict(), dict(k=40, p=0.9), dict(m=0.1), dict(temp=0.0), dict(temp=np.float32(1e-40)), dict(p=np.nan, m=np.nan, temp=0.5)):
        if "p" in kw and np.isnan(kw["p"]):
            a, b = call(ctx, x, u, temp=0.5), call(ctx, x, u, **kw)
            assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])
        else:
            check(ctx, x, u, **kw)
    assert np.array_equal(call(ctx, x, u, temp=np.nan)[0], call(ctx, x, u, temp=0.0)[0])
    # an infinite temperature makes all alike
    y = logits(rng, 1, 1000)
    assert call(ctx, y, 0.5004, temp=np.inf)[0][0] == 500


def test_frequencies(ctx):
    """Tokens come as often as their weights say: u on a fine grid."""
    x = np.log(np.array([[0.5, 0.25, 0.125, 0.0625, 0.0625]], np.float32))
    grid = ((np.arange(4096) + 0.5) / 4096).astype(np.float32)
    tok, pr = call(ctx, np.repeat(x, 4096, 0), grid)
    assert (np.diff(tok) >= 0).all() and np.abs(np.bincount(tok) - np.array([2048, 1024, 512, 256, 256])).max() <= 1


def test_agrees_with_the_greedy_choice(ctx):
    """The token of temperature 0 is that of ggq_logits_argmax_dev on the same logits."""
    import torch
    rng = np.random.default_rng(11)
    raw = gl.encode(gl.GgmlType.Q8_0, (rng.standard_normal((3001, 256)) * 0.05).astype(np.float32))
    w = torch.zeros(raw.size + 256, dtype=torch.uint8, device="cuda")
    w[: raw.size].copy_(torch.from_numpy(raw))
    a = t(rng.standard_normal((5, 256)), np.float32)
    lg, tok = torch.empty((5, 3001), device="cuda"), torch.empty(5, dtype=torch.int32, device="cuda")
    ctx.check(ctx.lib.ggq_logits_argmax_dev(ctx.h, w.data_ptr(), int(gl.GgmlType.Q8_0), 3001, 256, a.data_ptr(), 5, 0, lg.data_ptr(),
                                            tok.data_ptr(), None, stream_handle()), "argmax")
    assert np.array_equal(call(ctx, host(lg), 0.5, temp=0.0)[0], host(tok))


def test_same_every_time_and_without_prob(ctx):
    rng = np.random.default_rng(12)
    x = logits(rng, 9, 128256)
    u = rng.random(9).astype(np.float32)
    a = call(ctx, x, u, p=0.95)
    for _ in range(3):
        b = call(ctx, x, u, p=0.95)
        assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])
    check(ctx, x, u, p=0.95, prob=False)


def test_largest_vocabulary(ctx):
    rng = np.random.default_rng(13)
    x = logits(rng, 1, 1 << 22)
    for kw in (dict(), dict(k=50, p=0.9), dict(p=0.7)):
        check(ctx, x, 0.37, **kw)


def test_refusals(ctx):
    import torch
    b = torch.zeros(4096, device="cuda")
    P = b.data_ptr()
    ok = dict(n_rows=1, n_vocab=100, logits=P, ld=100, u=P + 1024, token=P + 2048)

    def st(**kw):
        return ctx.lib.ggq_sample_dev(ctx.h, gl.SampleParams(**{**ok, **kw}), stream_handle())

    assert st() == 0 and st(n_rows=0, logits=None, u=None, token=None) == 0
    for kw in (dict(n_rows=-1), dict(n_rows=65536), dict(n_vocab=0), dict(n_vocab=(1 << 22) + 1, ld=1 << 23), dict(ld=99), dict(logits=None),
               dict(u=None), dict(token=None)):
        assert st(**kw) == gl.Status.INVALID_PARAM, kw
    assert ctx.lib.ggq_sample_dev(ctx.h, None, stream_handle()) == gl.Status.INVALID_PARAM
    torch.cuda.synchronize()


def test_no_workspace_while_capturing(ctx):
    """A context whose first call is captured has no workspace for it: refused, and the stream is fine afterwards."""
    import torch
    c = gl.Context(0)
    x, u = t(np.zeros((1, 5000), np.float32)), t(np.zeros(1, np.float32))
    tok = torch.zeros(1, dtype=torch.int32, device="cuda")
    p = gl.SampleParams(n_rows=1, n_vocab=5000, logits=x.data_ptr(), ld=5000, u=u.data_ptr(), token=tok.data_ptr())
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        st = c.lib.ggq_sample_dev(c.h, p, ctypes.c_void_p(s.cuda_stream))
        tok.zero_()
    assert st == gl.Status.ERROR and b"ggq_reserve" in c.lib.ggq_last_error_message(c.h)
    c.check(c.lib.ggq_reserve(c.h, 1 << 20), "reserve")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        st = c.lib.ggq_sample_dev(c.h, p, ctypes.c_void_p(s.cuda_stream))
    assert st == 0
    for i in (3, 4999, 0):
        x.zero_()
        x[0, i] = 50.0
        g.replay()
        torch.cuda.synchronize()
        assert int(tok[0]) == i
    c.close()


def test_logits_far_from_zero_at_low_temperatures(ctx):
    """A token and thousands of equal ones a step of fp32 below it, millions of temperatures away from 0: the border between them stays
    where 64 bits have it.  u is the fp32 number next to the border, more than 2^-30 and less than 2^-26 away from it."""
    rng = np.random.default_rng(20)
    V, rows = 9001, []
    while len(rows) < 60:
        l0 = np.float32(np.exp2(rng.uniform(3, 17)))
        l1 = np.nextafter(l0, np.float32(0), dtype=np.float32)
        n = int(rng.integers(2000, 8000))
        T = np.float32((float(l0) - float(l1)) / (np.log(n) + rng.uniform(-1, 1)))
        w = np.exp((float(l1) - float(l0)) / float(T))
        border = 1 / (1 + n * w)
        u = np.float32(border)
        if 2.0 ** -30 < abs(float(u) - border) < 2.0 ** -26:
            x = np.full(V, -np.inf, np.float32)
            x[7:7 + n], x[rng.integers(0, 7)] = l1, l0
            rows.append((x, T, u))
    x, T, u = (np.array([r[i] for r in rows], np.float32) for i in range(3))
    check(ctx, x, u, temp=T)
    check(ctx, x, u, temp=T, p=0.99999994)
    check(ctx, x, u, temp=T, k=8999, m=1e-6)


@pytest.mark.parametrize("T", [1e-40, 1e-25, 1e-12, 1e-9])
def test_equal_logits_far_from_zero(ctx, T):
    """Logits so many temperatures away from 0 that only equal ones have a weight."""
    rng = np.random.default_rng(21)
    x = rng.standard_normal((6, 9000)).astype(np.float32) * 10
    x[:, 8999] = x[:, 17] = x[:, 5000] = x.max() + 3
    x[3:] -= 1000
    u = np.array([0.1, 0.5, 0.9] * 2, np.float32)
    for kw in (dict(), dict(k=2), dict(p=0.5), dict(m=0.5), dict(k=100, p=0.9)):
        check(ctx, x, u, temp=np.float32(T), **kw)


def test_min_p_above_one_keeps_the_first_token(ctx):
    """No weight is above 1: the first token is left, also where others equal it (few of them and many, with and without other filters)."""
    rng = np.random.default_rng(22)
    x = rng.standard_normal((3, 9001)).astype(np.float32)
    x[0, [40, 7000]] = 9.0
    x[1, 100:5000] = 9.0
    x[2, [3, 8000]] = np.inf
    for m in (1.0000001, 2.0, np.inf):
        for kw in (dict(), dict(k=3), dict(p=0.9), dict(k=3000, p=0.99)):
            tok, pr = call(ctx, x, 0.99, m=m, **kw)
            assert tok.tolist() == [40, 100, 3] and (pr == 1).all(), (m, kw)
    tok, pr = call(ctx, x, 0.99, m=1.0)  # (1 itself: all that equal it)
    assert tok.tolist() == [7000, 100 + int(np.float32(0.99) * np.float64(4900)), 8000]


def test_min_p_at_an_infinite_temperature(ctx):
    """All weights are 1: min_p up to 1 keeps every token."""
    x = np.random.default_rng(23).standard_normal((1, 1000)).astype(np.float32)
    for m in (1e-30, 0.5, 1.0):
        assert call(ctx, x, 0.5004, temp=np.inf, m=m)[0][0] == 500
        assert call(ctx, x, 0.5004, temp=np.inf, m=m, k=900, p=0.999)[0][0] == su.sample(x[0], np.inf, 900, 0.999, 0.0, 0.5004)[0]
    assert call(ctx, x, 0.5004, temp=np.inf, m=2.0)[0][0] == x[0].argmax()


@pytest.mark.parametrize("T,m,top", [("0x1.d816cep-1", "0x1.b73bf4p-4", "0x1.078324p+1"), ("0x1.5530b2p-1", "0x1.a5ba9ep-4", "0x1.83d4dcp+0"),
                                     ("0x1.76bf42p-1", "0x1.e081bcp-4", "0x1.918706p+0")])
def test_min_p_whose_border_is_at_zero(ctx, T, m, top):
    """T ln(min_p) is minus the largest logit to within 2^-53: hundreds of millions of numbers around 0 have that difference from it
    in 64 bits."""
    T, m, top = (np.float32(float.fromhex(v)) for v in (T, m, top))
    x = np.full((2, 5000), -5, np.float32)
    x[0, [9, 40, 41, 42]] = top, 1e-10, -1e-10, 0.01
    x[1, 1000:3000], x[1, 3000:4000], x[1, 77] = 1e-10, -1e-10, top
    w = np.exp((1e-10 - float(top)) / float(T))
    tok, pr = call(ctx, x, 0.99999994, temp=T, m=m)
    assert tok.tolist() == [42, 2999]
    tok, pr = call(ctx, x, 0.99999994, temp=T, m=m, k=4000)
    assert tok.tolist() == [42, 2999] and abs(pr[1] - w / (1 + 2000 * w)) <= pr[1] * (su.U32 + 2.0 ** -29)


def test_min_p_borders(ctx):
    """What min_p keeps, logit by logit, beside the largest ones of all sizes: the number at the border and its neighbours."""
    rng = np.random.default_rng(24)
    rows, temp, mins = [], [], []
    for _ in range(200):
        top = np.float32(rng.choice([-1, 1]) * np.exp2(rng.uniform(-20, 20)))
        T, m = np.float32(np.exp2(rng.uniform(-8, 8))), np.float32(np.exp2(rng.uniform(-20, 0)))
        at = float(top) + float(T) * np.log(float(m))
        near = [np.float32(at)]
        for _ in range(4):
            near = [np.nextafter(near[0], np.float32(-np.inf))] + near + [np.nextafter(near[-1], np.float32(np.inf))]
        # (a number whose weight is min_p's to within 2^-45 may be on either side)
        near = [v for v in near if v <= top and abs((float(v) - float(top)) / float(T) - np.log(float(m))) > 2.0 ** -45 * max(1.0, abs(np.log(float(m))))]
        x = np.full(300, -np.inf, np.float32)
        x[0], x[100:100 + len(near)] = top, near
        rows.append(x), temp.append(T), mins.append(m)
    x, temp, mins = np.array(rows), np.array(temp), np.array(mins)
    with np.errstate(all="ignore"):
        keep = (x.astype(np.float64) - x[:, :1]) / temp[:, None].astype(np.float64) >= np.log(mins.astype(np.float64))[:, None]
    keep[:, 0] = True
    last = np.where(keep, np.arange(300), -1).max(1)
    assert np.array_equal(call(ctx, x, 0.99999994, temp=temp, m=mins)[0], last)
