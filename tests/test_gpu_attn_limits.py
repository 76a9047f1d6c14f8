"""Prompt attention where it could go wrong unseen: calls that follow each other without a wait, against themselves and
against 64 bits; windows of any size, values and keys of any size that a row does not see, on the route of the rule and on both
routes."""
import numpy as np
import pytest

import ggnpu_amd.lib as gl
from tests import attn_util as au
from tests.gpu_util import host, stream_handle
from tests.test_gpu_attn_prompt import call as attend, inputs, run, t

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
    monkeypatch.setenv("GGQ_PROMPT_MFMA", request.param)
    return gpu


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("type", [0, 1])
@pytest.mark.parametrize("n_head,n_kv,q_off,kv_off,window", [
    (8, 8, [0, 369], None, 0),
    (2, 2, [0, 700, 1200], None, 0),
    (4, 1, [0, 40, 41, 100], [0, 900, 2100, 2200], 0),
    (5, 1, [0, 300], None, 14),  # wavefronts that skip the first units
    (16, 2, [0, 205], [0, 413], 82),
    (6, 2, [0, 3, 20, 22], [0, 3, 20, 22], 0),  # one unit, or less
])
def test_prompt_calls_in_a_row(gpu, monkeypatch, hd, type, n_head, n_kv, q_off, kv_off, window):
    """Two inputs in turn through one workspace, nothing waited for between the calls: every result is its input's first
    one bit for bit, and that one within the bound of 64 bits."""
    import torch
    monkeypatch.setenv("GGQ_PROMPT_MFMA", "1")
    rng = np.random.default_rng(hd + type)
    ko = q_off if kv_off is None else kv_off
    qo, kvo = t(np.array(q_off, np.int32)), t(np.array(ko, np.int32))
    data = [inputs(rng, q_off[-1], ko[-1], n_head, n_kv, hd, type) for _ in range(2)]
    on_gpu = [[t(x) for x in d] for d in data]

    def call(i, out):
        q, k, v = on_gpu[i]
        p = gl.AttnPromptParams(type=type, n_head=n_head, n_kv_head=n_kv, head_dim=hd, q=q.data_ptr(), ldq=n_head * hd,
                                k=k.data_ptr(), ldk=n_kv * hd, v=v.data_ptr(), ldv=n_kv * hd, out=out.data_ptr(), ldo=n_head * hd,
                                n_rows=q_off[-1], n_kv_rows=ko[-1], n_seq=len(q_off) - 1, q_off=qo.data_ptr(),
                                kv_off=kvo.data_ptr(), window=window)
        gpu.check(gpu.lib.ggq_attention_prompt_dev(gpu.h, p, stream_handle()), "prompt attention")

    outs = [torch.zeros((q_off[-1], n_head * hd), device="cuda") for _ in range(24)]
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        call(i % 2, out)
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        assert torch.equal(out, outs[i % 2]), i
    for i in (0, 1):
        q, k, v = data[i]
        got = host(outs[i])
        for s in range(len(q_off) - 1):
            n, m = q_off[s + 1] - q_off[s], ko[s + 1] - ko[s]
            kk, vv = (x[ko[s]:ko[s + 1]].reshape(m, n_kv, hd) for x in (k, v))
            for r in {0, n // 3, n // 2, n - 1}:
                want, tol = au.attention(q[q_off[s] + r].reshape(1, n_head, hd), kk, vv, m - n + r, window)
                au.check(got[q_off[s] + r].reshape(1, n_head, hd), want, tol)


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 8])
def test_prompt_windows_of_any_size(ctx, window):
    """A window far above every length is none, also where the first rows come before all keys."""
    run(ctx, 40, [0, 20], [0, 7], 4, 2, 64, window=window)
    run(ctx, 41, [0, 30, 50, 53], [0, 5, 25, 90], 3, 1, 128, 1, window=window)
    run(ctx, 42, [0, 1010], [0, 1000], 4, 1, 64, window=window, rows=[0, 8, 9, 10, 11, 500, 1009])
    run(ctx, 43, [0, 300], [0, 200], 4, 2, 256, window=window, rows=[0, 98, 99, 100, 101, 131, 132, 299])


@pytest.mark.parametrize("window", [1, 33])
def test_prompt_windows_and_rows_that_see_nothing(ctx, window):
    run(ctx, 46, [0, 90, 100, 140], [0, 50, 50, 200], 4, 2, 64, window=window)
    run(ctx, 47, [0, 90], [0, 50], 3, 1, 256, 1, window=window)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_prompt_unseen_values_beside_zero_rows(ctx, hd):
    """Value rows of zeros among the seen ones, values of any size among the unseen ones of the same 32 positions."""
    rng = np.random.default_rng(44)
    n, n_head, n_kv = 100, 4, 2
    q, k, v = inputs(rng, n, n, n_head, n_kv, hd)
    v[[0, 40, 95]] = 0
    v[64:70] = 0  # rows 64 .. 69 see nothing but zeros of their last 32 positions
    for bad in (1e4, 1e6, 1e12, -3e38):
        v2 = v.copy()
        v2[[59, 70, 99], ::5] = bad
        got = attend(ctx, q, k, v2, n_head, n_kv, hd, 0, [0, n], [0, n])
        for i in (0, 1, 31, 32, 40, 41, 58):
            want, tol = au.attention(q[i:i + 1].reshape(1, n_head, hd), k.reshape(n, n_kv, hd), v.reshape(n, n_kv, hd), i)
            au.check(got[i:i + 1].reshape(1, n_head, hd), want, tol)
        # a window whose rows see the large value no more: positions 60 .. 69 for row 69, among them six rows of zeros
        got = attend(ctx, q, k, v2, n_head, n_kv, hd, 0, [0, n], [0, n], window=10)
        for i in (58, 69, 82, 97):
            want, tol = au.attention(q[i:i + 1].reshape(1, n_head, hd), k.reshape(n, n_kv, hd), v.reshape(n, n_kv, hd), i, 10)
            au.check(got[i:i + 1].reshape(1, n_head, hd), want, tol)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_prompt_unseen_keys_beside_small_ones(ctx, hd):
    """Small keys under large queries, keys of any size among the unseen ones of the same 32 positions."""
    rng = np.random.default_rng(45)
    n, n_head, n_kv = 100, 4, 2
    q, k, v = inputs(rng, n, n, n_head, n_kv, hd)
    for size in (1.0, 1e10, 1e18):
        qs, ks = (q * np.float32(size)).astype(np.float32), (k * np.float32(1 / size)).astype(np.float32)
        for bad in (1e6, 1e20, -3e38):
            k2 = ks.copy()
            k2[59:, ::7] = bad
            got = attend(ctx, qs, k2, v, n_head, n_kv, hd, 0, [0, n], [0, n])
            for i in (0, 31, 32, 45, 58):
                want, tol = au.attention(qs[i:i + 1].reshape(1, n_head, hd), ks.reshape(n, n_kv, hd), v.reshape(n, n_kv, hd), i)
                au.check(got[i:i + 1].reshape(1, n_head, hd), want, tol)


def weighted(q, k, v, scale, floor):
    """fp64 attention of one row over all of k, v (one head) and the bound of each value: the score of a position is off by
    (hd / 4 + 8) roundings of its own sum of magnitudes, which its weight and the sum of weights take over; the sum over positions
    adds 32 + n / 16 roundings of its magnitudes; a weight is off by `floor` of the largest at most besides."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    s = k @ q * scale
    p = np.exp(s - s.max())
    p /= p.sum()
    ds = au.U32 * (k.shape[1] / 4 + 8) * (np.abs(k) @ np.abs(q)) * scale
    out = p @ v
    return out, (p * (ds + au.U32 * (32 + len(k) / 16))) @ np.abs(v) + p @ ds * np.abs(out) + floor * np.abs(v).sum(0) + 1e-37


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("type", [0, 1])
@pytest.mark.parametrize("where", [[0], [5], [40], [98], range(0, 32), range(32, 64), range(64, 96), [3, 31, 32, 60, 64, 90],
                                   [*range(0, 32), 40, 70, 96]])
def test_prompt_large_values_of_little_weight(ctx, hd, type, where):
    """Values of up to 2^100 (fp16: 2^12 beside 2^-6) that a row sees with a weight of next to nothing, before, among and
    behind the ones that make its result."""
    rng = np.random.default_rng(hd + len(where) + where[0])
    n, n_head = 100, 2
    u = rng.standard_normal(hd)
    u *= np.sqrt(hd) / np.linalg.norm(u)
    q = (np.tile(u, (n, n_head)) * (1 + 0.1 * rng.random((n, 1)))).astype(np.float32)
    for bits, nats in ((14, 12), (18, 14), (18, 30)) if type else ((20, 15), (24, 25), (40, 40), (70, 55), (100, 80)):
        k = 0.3 * rng.standard_normal((n, hd))
        v = rng.standard_normal((n, hd)) * (2.0 ** -6 if type else 1.0)
        for i in where:
            k[i] = -u / np.sqrt(hd) * nats
            v[i] *= 2.0 ** bits
        k, v = (x.astype(np.float16 if type else np.float32) for x in (k, v))
        got = attend(ctx, q, k, v, n_head, 1, hd, type, [0, n], [0, n])
        for i in (33, 63, 64, 97, 99):
            want, tol = weighted(q[i, :hd], k[:i + 1], v[:i + 1], hd ** -0.5, 2.0 ** -36 if type else 0.0)
            for h in range(n_head):
                au.check(got[i, h * hd:(h + 1) * hd], want, tol)


@pytest.mark.parametrize("hd,bound", [(64, 3.3e-6), (128, 4.1e-6), (256, 5.5e-6)])
def test_prompt_scores_add_small_products_first(gpu, monkeypatch, hd, bound):
    """Scores of 44 whose products all have one sign, told from the weights of two keys.  The products of the fp16 parts
    are added 16 values a step: with the small ones first, only the hd / 16 steps of hi times hi round at the size of the
    sum.  Emulated in 64 bits with a rounding to fp32 a step (two, if the step adds in halves), the difference of two scores
    is then off by 2.3 (2.8), 2.7 (3.6) and 3.5 (4.8) e-6, root mean square, and by 3.7, 4.7 and 6.2 e-6 at the least with
    hi times hi in between."""
    monkeypatch.setenv("GGQ_PROMPT_MFMA", "1")
    rng = np.random.default_rng(55)
    n, heads = 512, 8
    c = 44 * hd ** -0.5
    q = (1 + 0.2 * rng.standard_normal((n, heads * hd))).astype(np.float32)
    k = (c * (1 + 0.2 * rng.standard_normal((2 * n, heads * hd)))).astype(np.float32)
    v = np.zeros((2 * n, heads * hd), np.float32)
    v[0::2] = 1
    got = attend(gpu, q, k, v, heads, heads, hd, 0, np.arange(n + 1), 2 * np.arange(n + 1)).reshape(n, heads, hd)[..., 0].astype(np.float64)
    s = (k.reshape(n, 2, heads, hd).astype(np.float64) * q.reshape(n, 1, heads, hd)).sum(-1) * hd ** -0.5
    d = s[:, 0] - s[:, 1]
    assert 40 < s.mean() < 48 and np.abs(d).max() < 6
    err = np.log(got / (1 - got)) - d
    assert np.sqrt((err ** 2).mean()) <= bound
