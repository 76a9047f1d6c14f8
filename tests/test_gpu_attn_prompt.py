"""Causal attention of packed prompts (ggq_attention_prompt_dev) against 64 bits, each value within the bound that
attn_util.attention derives."""
import numpy as np
import pytest

import ggnpu_amd.lib as gl
from tests import attn_util as au
from tests.gpu_util import host, stream_handle

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    import torch
    assert torch.cuda.is_available()
    c = gl.Context(0)
    yield c
    c.close()


@pytest.fixture(params=["", "0", "1"], ids=["rule", "valu", "mfma"])
def ctx(gpu, request, monkeypatch):
    """Every test on the route of the rule and on both routes (GGQ_PROMPT_MFMA, read at every call)."""
    monkeypatch.setenv("GGQ_PROMPT_MFMA", request.param)
    return gpu


def t(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def inputs(rng, rows, keys, n_head, n_kv, hd, type=0, pad=0, qscale=1.0):
    dt = np.float16 if type else np.float32
    q = (rng.standard_normal((rows, n_head * hd + pad)) * qscale).astype(np.float32)
    k = rng.standard_normal((keys, n_kv * hd + pad)).astype(dt)
    v = (rng.standard_normal((keys, n_kv * hd + pad)) * np.exp2(rng.integers(-3, 4, (keys, 1)))).astype(dt)
    return q, k, v


def call(ctx, q, k, v, n_head, n_kv, hd, type, q_off, kv_off, window=0, scale=0.0, out=None, n_rows=None):
    import torch
    dq, dk, dv = t(q), t(k), t(v)
    out = torch.full(q.shape, 5.0, device="cuda") if out is None else out
    qo, ko = t(np.asarray(q_off, np.int32)), None if kv_off is None else t(np.asarray(kv_off, np.int32))
    p = gl.AttnPromptParams(type=type, n_head=n_head, n_kv_head=n_kv, head_dim=hd, q=dq.data_ptr(), ldq=q.shape[1],
                            k=dk.data_ptr(), ldk=k.shape[1], v=dv.data_ptr(), ldv=v.shape[1], out=out.data_ptr(), ldo=q.shape[1],
                            n_rows=q.shape[0], n_kv_rows=k.shape[0], n_seq=len(q_off) - 1, q_off=qo.data_ptr(),
                            kv_off=None if ko is None else ko.data_ptr(), window=window, scale=scale)
    ctx.check(ctx.lib.ggq_attention_prompt_dev(ctx.h, p, stream_handle()), "prompt attention")
    return host(out)


def verify(got, q, k, v, n_head, n_kv, hd, q_off, kv_off, window=0, scale=0.0, rows=None):
    """All rows, or the listed ones of each sequence (the 64-bit form takes its time)."""
    kv_off = q_off if kv_off is None else kv_off
    seen = np.zeros(len(q), bool)
    for s in range(len(q_off) - 1):
        n, m = q_off[s + 1] - q_off[s], kv_off[s + 1] - kv_off[s]
        kk = k[kv_off[s]:kv_off[s + 1], : n_kv * hd].reshape(m, n_kv, hd)
        vv = v[kv_off[s]:kv_off[s + 1], : n_kv * hd].reshape(m, n_kv, hd)
        seen[q_off[s]:q_off[s + 1]] = True
        for i in range(n) if rows is None else [r for r in rows if r < n]:
            r = q_off[s] + i
            want, tol = au.attention(q[r:r + 1, : n_head * hd].reshape(1, n_head, hd), kk, vv, m - n + i, window, scale or None)
            au.check(got[r:r + 1, : n_head * hd].reshape(1, n_head, hd), want, tol)
    assert (got[~seen] == 5).all() and (got[:, n_head * hd:] == 5).all()


def run(ctx, seed, q_off, kv_off, n_head, n_kv, hd, type=0, window=0, scale=0.0, pad=0, qscale=1.0, rows=None, behind=0):
    rng = np.random.default_rng(seed)
    keys = (q_off if kv_off is None else kv_off)[-1]
    q, k, v = inputs(rng, q_off[-1] + behind, keys + behind, n_head, n_kv, hd, type, pad, qscale)
    got = call(ctx, q, k, v, n_head, n_kv, hd, type, q_off, kv_off, window, scale)
    verify(got, q, k, v, n_head, n_kv, hd, q_off, kv_off, window, scale, rows)
    return got


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("type", [0, 1])
@pytest.mark.parametrize("n_head,n_kv", [(4, 1), (6, 2)])
def test_prompt_heads_and_types(ctx, hd, type, n_head, n_kv):
    run(ctx, hd + type, [0, 70], None, n_head, n_kv, hd, type)


@pytest.mark.parametrize("n_head,n_kv", [(1, 1), (5, 5), (7, 1), (16, 2), (16, 1), (24, 1), (33, 3)])
def test_prompt_head_ratios(ctx, n_head, n_kv):
    run(ctx, n_head, [0, 37], None, n_head, n_kv, 64)


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 129, 300])
def test_prompt_lengths(ctx, n):
    run(ctx, n, [0, n], None, 4, 2, 64)
    run(ctx, n + 1, [0, n], None, 3, 1, 128, 1)


def test_prompt_long(ctx):
    run(ctx, 1, [0, 2500], None, 8, 2, 64, rows=[0, 1, 63, 64, 1000, 2047, 2048, 2300, 2499])
    run(ctx, 2, [0, 1700], None, 2, 1, 128, 1, rows=[0, 65, 255, 256, 1023, 1500, 1699])


@pytest.mark.parametrize("type", [0, 1])
def test_prompt_packed(ctx, type):
    """Ragged prompts, empty ones among them, rows behind the last sequence left alone."""
    run(ctx, 5, [0, 1, 1, 66, 66, 66, 200, 233], None, 6, 2, 64, type, behind=5)
    run(ctx, 6, [0, 17, 18, 150], None, 4, 4, 128, type, pad=16)


def test_prompt_first_row_not_at_zero(ctx):
    """The first sequence starts behind row 0: rows in front of it stay, too."""
    run(ctx, 8, [3, 20, 45], [5, 22, 90], 4, 2, 64)


@pytest.mark.parametrize("type", [0, 1])
def test_prompt_chunks_of_a_cache(ctx, type):
    """A prompt's next chunk: fewer rows than keys; a single row; more rows than keys, whose first ones see nothing."""
    run(ctx, 7, [0, 40, 41, 60, 63], [0, 300, 417, 427, 427], 8, 2, 64, type)
    run(ctx, 9, [0, 3], [0, 5000], 4, 1, 128, type)
    run(ctx, 10, [0, 1], [0, 9000], 8, 2, 64, type)


@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 200])
def test_prompt_window(ctx, window):
    run(ctx, window, [0, 150, 180], [0, 150, 400], 4, 2, 64, window=window)
    run(ctx, window, [0, 300], None, 3, 1, 128, 1, window=window)


def test_prompt_chunk_equals_whole(ctx):
    """Rows of a later chunk see what they see in the whole prompt."""
    rng = np.random.default_rng(20)
    q, k, v = inputs(rng, 200, 200, 4, 2, 64)
    a = call(ctx, q, k, v, 4, 2, 64, 0, [0, 200], None)
    b = call(ctx, q[150:], k, v, 4, 2, 64, 0, [0, 50], [0, 200])
    verify(b, q[150:], k, v, 4, 2, 64, [0, 50], [0, 200])
    assert np.abs(a[150:] - b).max() <= 1e-5 * np.abs(v).max()


@pytest.mark.parametrize("type", [0, 1])
def test_prompt_unseen_keys_never_count(ctx, type):
    """Keys and values a row does not see may hold anything: its result stays within the bound of its own inputs (the
    32 positions that share a power of two may round otherwise).  Behind a sequence not even that."""
    rng = np.random.default_rng(11)
    n, n_head, n_kv, hd = 100, 4, 2, 64
    q, k, v = inputs(rng, n, n + 40, n_head, n_kv, hd, type)
    clean = call(ctx, q, k, v, n_head, n_kv, hd, type, [0, n], [0, n])
    for bad in (np.nan, np.inf, -np.inf, 6e4) + (() if type else (1e12, -3e38)):
        k2, v2 = k.copy(), v.copy()
        k2[60:, ::7], v2[60:, ::5] = bad, bad  # rows 0 .. 59 see none of it; nor does anyone positions n ..
        got = call(ctx, q, k2, v2, n_head, n_kv, hd, type, [0, n], [0, n])
        for i in (0, 31, 32, 45, 59):
            want, tol = au.attention(q[i:i + 1].reshape(1, n_head, hd), k[:n].reshape(n, n_kv, hd), v[:n].reshape(n, n_kv, hd), i)
            au.check(got[i:i + 1].reshape(1, n_head, hd), want, tol)
        if not np.isfinite(bad):
            assert not np.isfinite(got[60:]).all()
        k2, v2 = k.copy(), v.copy()
        k2[n:], v2[n:] = bad, bad  # behind the sequence
        assert np.array_equal(call(ctx, q, k2, v2, n_head, n_kv, hd, type, [0, n], [0, n]), clean)


@pytest.mark.parametrize("type", [0, 1])
def test_prompt_values_that_are_not_finite(ctx, type):
    """A row that sees an infinity or a NaN value has it in that value's place, as the sum of products has."""
    rng = np.random.default_rng(12)
    n, n_head, n_kv, hd = 90, 2, 1, 64
    q, k, v = inputs(rng, n, n, n_head, n_kv, hd, type)
    v[20, 3], v[70, 9], v[75, 9], v[30, 40] = np.inf, np.inf, -np.inf, np.nan
    got = call(ctx, q, k, v, n_head, n_kv, hd, type, [0, n], None).reshape(n, n_head, hd)
    assert np.isfinite(got[:20]).all()
    assert (got[20:, :, 3] == np.inf).all() and np.isnan(got[30:, :, 40]).all()
    assert (got[70:75, :, 9] == np.inf).all() and np.isnan(got[75:, :, 9]).all()
    keep = np.ones(hd, bool)
    keep[[3, 9, 40]] = False
    assert np.isfinite(got[:, :, keep]).all()
    want = np.where(np.isfinite(v), v, 0).astype(v.dtype)
    for i in (0, 25, 69, 70, 89):
        w, tol = au.attention(q[i:i + 1].reshape(1, n_head, hd), k.reshape(n, 1, hd), want.reshape(n, 1, hd), i)
        au.check(got[i:i + 1][..., keep], w[..., keep], tol[..., keep])


def test_prompt_sizes_of_values(ctx):
    """Rows, keys and values of very different sizes: outliers of 2^12 in some, everything at 1e-15 or 1e15 in others."""
    rng = np.random.default_rng(13)
    n, n_head, n_kv, hd = 200, 4, 1, 128
    q, k, v = inputs(rng, n, n, n_head, n_kv, hd)
    k[5] *= 8
    v[17] *= 4096
    q[:, ::9] *= 0.01
    for qs, ks, vs in ((1, 1, 1), (1e15, 1e-15, 1e15), (1e-15, 1e15, 1e-15), (1, 1, 1e-30)):
        a, b, c = (q * np.float32(qs)).astype(np.float32), (k * np.float32(ks)).astype(np.float32), (v * np.float32(vs)).astype(np.float32)
        got = call(ctx, a, b, c, n_head, n_kv, hd, 0, [0, n], None)
        verify(got, a, b, c, n_head, n_kv, hd, [0, n], None, rows=[0, 16, 17, 18, 100, 199])


def test_prompt_peaked_scores_and_scale(ctx):
    run(ctx, 14, [0, 130], None, 4, 2, 64, qscale=30.0)
    run(ctx, 15, [0, 130], None, 4, 2, 64, scale=0.7)
    run(ctx, 16, [0, 130], None, 4, 2, 64, 1, scale=-0.1)


def test_prompt_is_repeatable(ctx):
    a = run(ctx, 17, [0, 500, 900], None, 8, 2, 128, rows=[0, 399])
    assert np.array_equal(a, run(ctx, 17, [0, 500, 900], None, 8, 2, 128, rows=[0, 399]))


def test_prompt_many_sequences(ctx):
    """More sequences than threads of a workgroup, many of them empty."""
    rng = np.random.default_rng(18)
    n = rng.integers(0, 5, 600)
    off = np.concatenate([[0], np.cumsum(n)]).tolist()
    run(ctx, 19, off, None, 2, 1, 64)


@pytest.mark.parametrize("splits", ["1", "2", "5", "1000"])
def test_prompt_split_counts(gpu, monkeypatch, splits):
    """Any number of parts of the positions (GGQ_PROMPT_SPLITS), empty ones among them, rows of no sequence left alone."""
    monkeypatch.setenv("GGQ_PROMPT_MFMA", "1")
    monkeypatch.setenv("GGQ_PROMPT_SPLITS", splits)
    run(gpu, 30, [0, 40, 41, 41, 60], [0, 300, 700, 710, 729], 6, 2, 64, 0, behind=3)
    run(gpu, 31, [2, 90], [0, 260], 4, 1, 128, 1, window=100)
    run(gpu, 32, [0, 20], [0, 7], 2, 2, 64)


def test_prompt_not_finite_queries_and_keys_stay_in_their_rows(ctx):
    rng = np.random.default_rng(33)
    n, n_head, n_kv, hd = 80, 4, 2, 64
    q, k, v = inputs(rng, n, n, n_head, n_kv, hd)
    q2, k2 = q.copy(), k.copy()
    q2[11, 64 * 2 + 5] = np.nan  # row 11, head 2
    q2[12, 3] = np.inf  # row 12, head 0
    k2[50, 64 + 7] = np.nan  # key 50 of kv head 1: heads 2 and 3 from row 50 on
    got = call(ctx, q2, k2, v, n_head, n_kv, hd, 0, [0, n], None).reshape(n, n_head, hd)
    assert np.isnan(got[11, 2]).all() and not np.isfinite(got[12, 0]).any() and np.isnan(got[50:, 2:]).all()
    good = np.ones((n, n_head), bool)
    good[11, 2] = good[12, 0] = False
    good[50:, 2:] = False
    want, tol = au.attention(q.reshape(n, n_head, hd), k.reshape(n, n_kv, hd), v.reshape(n, n_kv, hd), 0)
    au.check(got[good], want[good], tol[good])


def test_prompt_refusals(ctx):
    import torch
    x = torch.zeros(8192, device="cuda")
    off = t(np.array([0, 1], np.int32))

    def go(**kw):
        d = dict(type=0, n_head=4, n_kv_head=2, head_dim=64, q=x.data_ptr(), ldq=256, k=x.data_ptr() + 4096, ldk=128,
                 v=x.data_ptr() + 8192, ldv=128, out=x.data_ptr() + 16384, ldo=256, n_rows=1, n_kv_rows=1, n_seq=1,
                 q_off=off.data_ptr())
        d.update(kw)
        return ctx.lib.ggq_attention_prompt_dev(ctx.h, gl.AttnPromptParams(**d), stream_handle())
    assert go() == gl.Status.OK and go(n_rows=0, q=None) == gl.Status.OK and go(n_seq=0) == gl.Status.OK
    for kw in (dict(type=12), dict(n_head=3), dict(n_head=0), dict(n_kv_head=0), dict(head_dim=96), dict(ldq=255), dict(ldo=128),
               dict(ldk=64), dict(ldv=127), dict(ldq=258), dict(ldk=130), dict(type=1, ldk=132), dict(n_rows=-1), dict(n_kv_rows=-1),
               dict(n_seq=-1), dict(window=-1), dict(scale=float("nan")), dict(q=None), dict(k=None), dict(v=None), dict(out=None),
               dict(q_off=None), dict(q=x.data_ptr() + 4), dict(k=x.data_ptr() + 8), dict(v=x.data_ptr() + 4), dict(out=x.data_ptr() + 8)):
        assert go(**kw) == gl.Status.INVALID_PARAM, kw
    assert ctx.lib.ggq_attention_prompt_dev(ctx.h, None, stream_handle()) == gl.Status.INVALID_PARAM
