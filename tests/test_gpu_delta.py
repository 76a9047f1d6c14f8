"""ggq_delta_rule_dev against the recurrence in 64 bits, within the bounds that step_util.delta derives; row by row and in
parts of 16 rows."""
import ctypes

import numpy as np
import pytest

import ggnpu_amd.lib as gl
from tests import step_util as su
from tests.attn_util import check
from tests.gpu_util import host, stream_handle

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


def padded(x, pad, fill=9.0):
    n = x.shape[0]
    b = np.full((n, x[0].size + pad if n else 1), fill, np.float32)
    if n:
        b[:, : x[0].size] = x.reshape(n, -1)
    return b


class Case:
    def __init__(self, seed, lens, kh, vh, kd, vd, raw=False, before=0, behind=0, slots=None, slot=None, long_memory=False):
        """`before` and `behind`: rows of no sequence."""
        rng = np.random.default_rng(seed)
        self.lens, self.dims = list(lens), (kh, vh, kd, vd)
        n = before + sum(lens) + behind
        self.off = np.concatenate([[before], before + np.cumsum(lens)]).astype(np.int32)
        f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
        self.q, self.k, self.v = f(n, kh, kd), f(n, kh, kd), f(n, vh, vd)
        self.raw = raw
        if raw:
            self.gate, self.beta = f(n, vh), 2 * f(n, vh)
            self.rate, self.bias = -np.exp(f(vh)), f(vh)
        else:
            self.gate = -np.exp(f(n, vh) - (5 if long_memory else 1)).astype(np.float32)
            self.beta = (1 / (1 + np.exp(-f(n, vh)))).astype(np.float32)
            self.rate = self.bias = None
            for x in ("q", "k"):
                y = getattr(self, x)
                setattr(self, x, (y / np.linalg.norm(y, axis=-1, keepdims=True)).astype(np.float32))
        self.slots = slots or len(lens) + 1
        self.slot = np.asarray(rng.permutation(self.slots)[: len(lens)] if slot is None else slot, np.int32)
        self.state = f(self.slots, vh, vd, kd)

    def call(self, ctx, in_place=False, pad=0, flags=None, eps=1e-6, scale=0.0, rows=None, use_off=True, use_slot=True, stream=None, gap=0):
        import torch
        kh, vh, kd, vd = self.dims
        n = len(self.q)
        b = {x: t(padded(getattr(self, x), pad)) for x in ("q", "k", "v")}
        g, be = t(padded(self.gate, gap)), t(padded(self.beta, gap))
        rate, bias = (None if x is None else t(x) for x in (self.rate, self.bias))
        st = t(self.state)
        so = st if in_place else torch.full_like(st, 7.0)
        out = torch.full((max(n, 1), vh * vd + pad), 7.0, device="cuda")
        off, slot = t(self.off), t(self.slot)
        P = lambda x: None if x is None else x.data_ptr()  # noqa: E731
        fl = (gl.DELTA_BETA_SIGMOID | gl.DELTA_QK_NORM if self.raw else 0) if flags is None else flags
        p = gl.DeltaRuleParams(n_k_head=kh, n_v_head=vh, k_dim=kd, v_dim=vd, q=P(b["q"]), ldq=kh * kd + pad, k=P(b["k"]), ldk=kh * kd + pad,
                               v=P(b["v"]), ldv=vh * vd + pad, gate=P(g), ld_gate=vh + gap, beta=P(be), ld_beta=vh + gap, gate_rate=P(rate),
                               gate_bias=P(bias), flags=fl, eps=eps, scale=scale, state=P(st), state_out=P(so), n_slots=self.slots,
                               slot=P(slot) if use_slot else None, n_seq=len(self.lens), n_rows=n if rows is None else rows,
                               row_off=P(off) if use_off else None, out=P(out), ldo=vh * vd + pad)
        ctx.check(ctx.lib.ggq_delta_rule_dev(ctx.h, p, stream_handle() if stream is None else stream), "delta rule")
        o = host(out)
        assert (o[:, vh * vd:] == 7).all()
        return o[:n, : vh * vd].reshape(n, vh, vd), host(so)

    def check(self, o, so, in_place=False, flags=None, eps=1e-6, scale=0.0, seqs=None):
        fl = (gl.DELTA_BETA_SIGMOID | gl.DELTA_QK_NORM if self.raw else 0) if flags is None else flags
        g, b = su.gates(self.gate, self.beta, self.rate, self.bias, bool(fl & gl.DELTA_BETA_SIGMOID))
        rows, slots = np.zeros(len(self.q), bool), np.zeros(self.slots, bool)
        for i in range(len(self.lens)) if seqs is None else seqs:
            a, e, s = self.off[i], self.off[i + 1], self.slot[i]
            out, S, tol, S_tol = su.delta(self.q[a:e], self.k[a:e], self.v[a:e], g[a:e], b[a:e], self.state[s], bool(fl & gl.DELTA_QK_NORM),
                                          eps, scale)
            check(o[a:e], out, tol)
            check(so[s], S, S_tol)
            rows[a:e], slots[s] = True, True
        if seqs is None:
            assert (o[~rows] == 7).all()  # rows and slots of no sequence stay
            assert np.array_equal(so[~slots], self.state[~slots]) if in_place else (so[~slots] == 7).all()


@pytest.fixture(params=["rows", "parts"])
def form(request, monkeypatch):
    monkeypatch.setenv("GGQ_DELTA_PARTS", "1" if request.param == "parts" else "0")
    return request.param


@pytest.mark.parametrize("kd", [64, 128, 256])
@pytest.mark.parametrize("vd", [16, 48, 64, 128])
@pytest.mark.parametrize("raw", [False, True])
def test_widths(ctx, form, kd, vd, raw):
    c = Case(kd + vd, [37], 1, 2, kd, vd, raw)
    c.check(*c.call(ctx))


@pytest.mark.parametrize("kh,vh", [(1, 1), (2, 2), (1, 3), (3, 15), (5, 10), (16, 32), (1, 8)])
def test_heads(ctx, form, kh, vh):
    c = Case(kh * vh, [5, 18], kh, vh, 64, 16, raw=True)
    c.check(*c.call(ctx))


@pytest.mark.parametrize("lens", [[1], [2], [15], [16], [17], [31, 32, 33], [0, 1, 0, 16, 5, 0], [48], [200], [1, 150, 1, 1, 64]])
def test_lengths(ctx, form, lens):
    c = Case(sum(lens) + len(lens), lens, 2, 4, 64, 32, before=3, behind=2)
    c.check(*c.call(ctx))


def test_wide_values(ctx, form):
    c = Case(1, [20], 1, 1, 128, 512)
    c.check(*c.call(ctx))


def test_single_tokens(ctx, form):
    """One row a sequence with offsets and without, many sequences (a workgroup takes more columns then), with and without slots."""
    for n, vh in ((3, 2), (70, 32)):
        c = Case(n, [1] * n, 2, vh, 128, 128, raw=True, slots=n + 5)
        a = c.call(ctx)
        c.check(*a, seqs=range(min(n, 4)))
        b = c.call(ctx, use_off=False)
        if form == "rows":
            assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])
        c.slot = np.arange(n, dtype=np.int32)
        x, y = c.call(ctx, use_slot=False), c.call(ctx)
        assert np.array_equal(x[0], y[0]) and np.array_equal(x[1], y[1])


def test_in_place_and_strides(ctx, form):
    c = Case(5, [40, 3, 0, 29], 2, 4, 128, 32, raw=True, before=1, behind=4)
    a, b = c.call(ctx), c.call(ctx, in_place=True, pad=12, gap=3)
    c.check(*a)
    c.check(*b, in_place=True)
    used = c.slot
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1][used], b[1][used])


def test_parts_of_a_sequence_follow_each_other(ctx, form):
    """A prompt in calls of 23, 1, 16 and 30 rows: the state carries what the rows before left."""
    c = Case(6, [70], 1, 2, 64, 64, long_memory=True)
    g, b = su.gates(c.gate, c.beta)
    out, S, tol, S_tol = su.delta(c.q, c.k, c.v, g, b, c.state[c.slot[0]])
    at, got = 0, []
    for n in (23, 1, 16, 30):
        d = Case(6, [70], 1, 2, 64, 64, long_memory=True)
        d.state, d.lens, d.off, d.slot = c.state.copy(), [n], np.array([at, at + n], np.int32), c.slot
        o, so = d.call(ctx, in_place=True)
        got.append(o[at:at + n])
        c.state = so
        at += n
    check(np.concatenate(got), out, tol)
    check(c.state[c.slot[0]], S, S_tol)


def test_forms_agree(ctx, monkeypatch):
    """The two forms on a prompt of several hundred rows, both within the bound; without forcing, long prompts go in parts."""
    c = Case(7, [333], 1, 2, 128, 64, raw=True)
    r = []
    for v in ("0", "1", ""):
        monkeypatch.setenv("GGQ_DELTA_PARTS", v)
        r.append(c.call(ctx))
        c.check(*r[-1])
    assert np.array_equal(r[1][0], r[2][0]) and not np.array_equal(r[0][0], r[1][0])


@pytest.mark.parametrize("env", ["", "2"])
@pytest.mark.parametrize("lens,vh", [([1] * 9 + [90] + [3, 16, 17, 0, 33, 8, 9], 2), ([1] * 40 + [200], 2), ([4] * 30, 4), ([1, 30, 1], 32), ([0] * 5, 2),
                                     ([70] + [1] * 70, 32), ([17] * 12 + [1] * 30, 32)])
def test_short_and_long_sequences_in_one_call(ctx, monkeypatch, env, lens, vh):
    """Short ones go row by row and long ones in parts, each once; forced and by the rule."""
    monkeypatch.setenv("GGQ_DELTA_PARTS", env)
    c = Case(len(lens) + vh, lens, 2, vh, 64, 32, raw=True, before=2, behind=3)
    a = c.call(ctx)
    c.check(*a)
    b = c.call(ctx, in_place=True)
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1][c.slot], b[1][c.slot])


def test_long_sequences_among_many(ctx, monkeypatch):
    """More sequences than are looked through in one turn, the long ones in several turns, one with a slot that does not exist."""
    monkeypatch.setenv("GGQ_DELTA_PARTS", "2")
    lens = [1] * 1300
    for i in (0, 5, 511, 512, 700, 1024, 1299):
        lens[i] = 20 + i % 7
    c = Case(21, lens, 1, 1, 64, 16)
    c.slot[700] = -1
    o, so = c.call(ctx)
    c.check(o, so, seqs=[0, 1, 5, 510, 511, 512, 513, 1023, 1024, 1025, 1298, 1299])
    assert (o[c.off[700]:c.off[701]] == 7).all()


def test_decays_of_all_sizes(ctx, form):
    """Nothing forgotten, everything forgotten (also by -infinity), and long runs after large decays: differences of sums keep their bits."""
    c = Case(8, [60], 1, 4, 64, 32)
    c.gate[:, 0] = 0.0
    c.gate[:, 1] = -1e-3
    c.gate[::7, 1] = -90.0
    c.gate[:, 2] = -2.5
    c.gate[::5, 3], c.gate[1::5, 3], c.gate[2::5, 3] = -np.inf, -1e30, -3e-4
    c.check(*c.call(ctx))


def test_steps_at_their_ends(ctx, form):
    """b = 0 keeps the state (but for the decay), b = 1 replaces what it gave for the key; equal keys in a row."""
    c = Case(9, [40], 1, 2, 64, 16)
    c.beta[:, 0], c.beta[:, 1] = 0.0, 1.0
    c.k[1::2] = c.k[::2]
    c.gate[:] = 0
    c.check(*c.call(ctx))


def test_flags_one_by_one(ctx, form):
    c = Case(10, [21], 1, 2, 64, 16, raw=True)
    c.k /= 20  # (without the norm: keys shorter than 1)
    for flags in (gl.DELTA_BETA_SIGMOID, gl.DELTA_BETA_SIGMOID | gl.DELTA_QK_NORM):
        c.check(*c.call(ctx, flags=flags, eps=0.01, scale=0.3), flags=flags, eps=0.01, scale=0.3)
    c.bias = None
    c.check(*c.call(ctx))
    c.beta = np.abs(np.tanh(c.beta))
    c.check(*c.call(ctx, flags=gl.DELTA_QK_NORM), flags=gl.DELTA_QK_NORM)


def test_values_of_all_sizes(ctx, form):
    """Rows a million times larger beside small ones, in columns of their own and in all."""
    c = Case(11, [50], 1, 2, 128, 32)
    c.v[::9] *= 1e6
    c.v[:, :, 5] *= 1e-6
    c.state[:, 0] *= 1e3
    c.check(*c.call(ctx))


def test_slots_that_do_not_exist(ctx, form):
    """Such a sequence is passed over, the others are not."""
    c = Case(12, [20, 20, 20, 20], 1, 2, 64, 16, slots=4, slot=[2, -1, 0, 4])
    o, so = c.call(ctx)
    c.check(o, so, seqs=[0, 2])
    assert (o[20:40] == 7).all() and (o[60:80] == 7).all() and (so[1] == 7).all() and (so[3] == 7).all()


def test_not_finite_rows_spoil_their_sequence_only(ctx, form):
    c = Case(13, [20, 35, 20], 1, 2, 64, 16)
    a = c.call(ctx)
    c.v[30], c.k[33, 0, 3] = np.nan, np.inf
    b = c.call(ctx)
    for s in (0, 2):
        r = slice(c.off[s], c.off[s + 1])
        assert np.array_equal(a[0][r], b[0][r]) and np.array_equal(a[1][c.slot[s]], b[1][c.slot[s]])
    assert np.array_equal(a[0][20:28 if form == "rows" else 20], b[0][20:28 if form == "rows" else 20])
    assert np.isnan(b[1][c.slot[1]]).all()


def test_same_every_time(ctx, form):
    c = Case(14, [100, 1, 77], 4, 8, 128, 128, raw=True)
    a = c.call(ctx)
    for _ in range(3):
        b = c.call(ctx)
        assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


def test_offsets_are_held_inside_the_rows(ctx, form):
    """Offsets beyond n_rows end there."""
    c = Case(15, [20, 40], 1, 1, 64, 16)
    o, so = c.call(ctx, rows=50)
    assert (o[50:] == 7).all()
    c.lens, c.off = [20, 30], np.array([0, 20, 50], np.int32)
    c.check(o, so, seqs=[0, 1])


def test_without_workspace_row_by_row(ctx):
    """A capture for which nothing is set aside takes the form without workspace: the same result within the bound."""
    import torch
    c = Case(16, [90], 1, 2, 64, 32)
    x = gl.Context(0)
    s = torch.cuda.Stream()
    kh, vh, kd, vd = c.dims
    b = {n: t(getattr(c, n)) for n in ("q", "k", "v", "gate", "beta", "state", "off", "slot")}
    so, out = torch.zeros_like(b["state"]), torch.full((90, vh * vd), 7.0, device="cuda")
    p = gl.DeltaRuleParams(n_k_head=kh, n_v_head=vh, k_dim=kd, v_dim=vd, q=b["q"].data_ptr(), ldq=kh * kd, k=b["k"].data_ptr(), ldk=kh * kd,
                           v=b["v"].data_ptr(), ldv=vh * vd, gate=b["gate"].data_ptr(), ld_gate=vh, beta=b["beta"].data_ptr(), ld_beta=vh,
                           state=b["state"].data_ptr(), state_out=so.data_ptr(), n_slots=c.slots, slot=b["slot"].data_ptr(), n_seq=1, n_rows=90,
                           row_off=b["off"].data_ptr(), out=out.data_ptr(), ldo=vh * vd)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        st = x.lib.ggq_delta_rule_dev(x.h, p, ctypes.c_void_p(s.cuda_stream))
    assert st == 0
    for _ in range(3):
        out.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        c.check(host(out).reshape(90, vh, vd), host(so), seqs=[0])
    x.close()


def test_refusals(ctx):
    import torch
    b = torch.zeros(1 << 16, device="cuda")
    P = b.data_ptr()
    i32 = torch.zeros(8, dtype=torch.int32, device="cuda")
    ok = dict(n_k_head=1, n_v_head=2, k_dim=64, v_dim=16, q=P, ldq=64, k=P, ldk=64, v=P, ldv=32, gate=P, ld_gate=2, beta=P, ld_beta=2,
              state=P, state_out=P + 65536, n_slots=1, n_seq=1, n_rows=1, out=P + 131072, ldo=32)

    def st(**kw):
        return ctx.lib.ggq_delta_rule_dev(ctx.h, gl.DeltaRuleParams(**{**ok, **kw}), stream_handle())

    assert st() == 0 and st(n_seq=0) == 0 and st(n_slots=0) == 0 and st(n_rows=0, q=None, k=None, v=None, gate=None, beta=None, out=None) == 0
    for kw in (dict(n_k_head=0), dict(n_v_head=0), dict(n_k_head=2, n_v_head=3), dict(k_dim=96), dict(k_dim=0), dict(v_dim=0), dict(v_dim=24),
               dict(v_dim=528, ldv=2000, ldo=2000), dict(ldq=60), dict(ldk=60), dict(ldv=28), dict(ldo=28), dict(ld_gate=1), dict(ld_beta=1),
               dict(ldq=66), dict(ldq=1 << 25), dict(ldo=34), dict(q=None), dict(k=None), dict(v=None), dict(gate=None), dict(beta=None),
               dict(out=None), dict(state=None), dict(state_out=None), dict(q=P + 4), dict(state=P + 8), dict(out=P + 12), dict(flags=4),
               dict(flags=-1), dict(n_seq=-1), dict(n_seq=65536), dict(n_rows=-1), dict(n_rows=(1 << 27) + 1), dict(n_slots=-1), dict(eps=-1.0), dict(eps=float("nan")),
               dict(scale=float("inf")), dict(gate_bias=P), dict(n_v_head=65536)):
        assert st(**kw) == gl.Status.INVALID_PARAM, kw
        assert ctx.lib.ggq_last_error_message(ctx.h)
    assert i32 is not None
    torch.cuda.synchronize()


@pytest.mark.parametrize("what", ["v", "v infinite", "one column of v", "k", "k infinite", "beta", "gate", "beta infinite"])
@pytest.mark.parametrize("row", [0, 7, 15, 16, 37, 49])
def test_a_row_that_is_not_finite_does_not_reach_back(ctx, form, what, row):
    """Rows before it keep their results, also those that are solved together with it, and so do columns without it; what comes after
    it is not finite."""
    c = Case(40, [3, 50, 20], 1, 2, 64, 48)
    clean = c.call(ctx)
    at, end, odd = 3 + row, 53, [5] if what == "one column of v" else list(range(48))
    bad = np.inf if "infinite" in what else np.nan
    if what == "one column of v":
        c.v[at, :, 5] = bad
    elif what[0] == "k":
        c.k[at, 0, 3] = bad
    else:
        {"v": c.v, "b": c.beta, "g": c.gate}[what[0]][at] = bad
    o, so = c.call(ctx)
    out, S, tol, S_tol = su.delta(*(x[3:at] for x in (c.q, c.k, c.v, c.gate, c.beta)), c.state[c.slot[1]])
    check(o[3:at], out, tol)
    assert not np.isfinite(o[at:end][:, :, odd]).any() and not np.isfinite(so[c.slot[1]][:, odd]).any()
    for s in (0, 2):
        r = slice(c.off[s], c.off[s + 1])
        assert np.array_equal(o[r], clean[0][r]) and np.array_equal(so[c.slot[s]], clean[1][c.slot[s]])
    if what == "one column of v":
        rest = [d for d in range(48) if d != 5]
        x, y = c.v.copy(), c.v.copy()
        y[at, :, 5] = 0
        c.v = y
        want, S, tol, S_tol = su.delta(*(z[3:end] for z in (c.q, c.k, c.v, c.gate, c.beta)), c.state[c.slot[1]])
        check(o[3:end][:, :, rest], want[:, :, rest], tol[:, :, rest])
        check(so[c.slot[1]][:, rest], S[:, rest], S_tol[:, rest])


def test_a_query_that_is_not_finite_spoils_its_row_only(ctx, form):
    c = Case(41, [40], 1, 2, 64, 16)
    a = c.call(ctx)
    c.q[21, 0, 9] = np.nan
    b = c.call(ctx)
    rest = [r for r in range(40) if r != 21]
    assert np.array_equal(a[0][rest], b[0][rest]) and np.array_equal(a[1], b[1]) and np.isnan(b[0][21]).all()


@pytest.mark.parametrize("env", ["", "1", "2"])
def test_not_finite_rows_of_many_sequences(ctx, monkeypatch, env):
    """Long and short sequences, states in place, one state that is not finite from the start, several workgroups' worth of columns."""
    monkeypatch.setenv("GGQ_DELTA_PARTS", env)
    lens = [90, 1, 40, 5, 33, 64] + [1] * 20
    c = Case(42, lens, 2, 4, 128, 32)
    at = {0: 20, 2: 39, 3: 2, 5: 0}
    for s, i in at.items():
        c.v[c.off[s] + i, 1, 3] = np.nan
    c.state[c.slot[4], 2, 7, 11] = np.nan
    o, so = c.call(ctx, in_place=True)
    for s in range(len(lens)):
        a, e = c.off[s], c.off[s + 1]
        v, S0 = c.v[a:e].copy(), c.state[c.slot[s]].copy()
        spoilt, late = np.zeros((e - a, 4, 32), bool), np.zeros((4, 32), bool)
        if s in at:
            spoilt[at[s]:, 1, 3], late[1, 3], v[at[s], 1, 3] = True, True, 0
        if s == 4:
            spoilt[:, 2, 7], late[2, 7], S0[2, 7] = True, True, 0
        want, S, tol, S_tol = su.delta(c.q[a:e], c.k[a:e], v, c.gate[a:e], c.beta[a:e], S0)
        if s in at:  # (the rows before it)
            x = su.delta(c.q[a:a + at[s]], c.k[a:a + at[s]], c.v[a:a + at[s]], c.gate[a:a + at[s]], c.beta[a:a + at[s]], S0)
            want[:at[s]], tol[:at[s]] = x[0], x[2]
        got, gS = o[a:e], so[c.slot[s]]
        assert np.isnan(got[spoilt]).all() and np.isnan(gS[late]).all()
        check(got[~spoilt], want[~spoilt], tol[~spoilt])
        check(gS[~late], S[~late], S_tol[~late])
