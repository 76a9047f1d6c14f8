"""The attention operators where calls could meet: captured and eager calls that need workspace in flight together, threads of
one context; and 256-wide prompts, whose units, wavefronts and schedule are their own, in parts, chunks, windows, captures
and groups of heads."""
import threading

import numpy as np
import pytest

import ggnpu_amd.lib as gl
from tests import attn_util as au
from tests.gpu_util import host
from tests.test_gpu_attn_prompt import run, t
from tests.test_gpu_attn_together import Layer, _buffers, _token_step, stream

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import torch
    assert torch.cuda.is_available()
    c = gl.Context(0)
    yield c
    c.close()


def _generator(seed):
    import torch
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


def _prompt_of(lay, rows, gen):
    """Buffers of a prompt whose offsets split it in two."""
    import torch
    q, k, v = (torch.randn((rows, h, lay.hd), device="cuda", generator=gen) for h in (lay.n_head, lay.n_kv, lay.n_kv))
    return q, k, v, torch.empty_like(q), t(np.array([0, rows // 3, rows], np.int32))


@pytest.mark.parametrize("hd", [64, 256])
def test_graphs_and_streams_with_planes_and_parts(ctx, monkeypatch, hd):
    """Two captured and two eager pairs of calls, each on a stream of its own and all in flight together; every prompt
    goes through planes and every cache call through parts, so that a shared buffer would show."""
    import torch
    monkeypatch.setenv("GGQ_PROMPT_MFMA", "1")
    monkeypatch.setenv("GGQ_KV_SPLITS", "9")
    gen = _generator(50)
    lays = [Layer(ctx, 1, 1, 4096, 8, 2, hd, 4, 8, seed=i) for i in range(4)]
    bufs = [_buffers(x, 1, 60 + i) for i, x in enumerate(lays)]
    prompts = [_prompt_of(x, 400 + 90 * i, gen) for i, x in enumerate(lays)]
    for x in lays:
        k, v = (torch.randn((4000, 2, hd), device="cuda", generator=gen) for _ in range(2))
        x.len.fill_(4000)
        x.store(k, v, t(np.array([0, 4000], np.int32)), stream())

    def work(i, s):
        q, k, v, out, off = prompts[i]
        lays[i].prompt(q, k, v, out, off, off, s)
        lays[i].decode(bufs[i]["q"], bufs[i]["out"], s)
        lays[i].prompt(q, k, v, out, off, off, s)
    want = []
    for i in range(4):
        work(i, stream())
        torch.cuda.synchronize()
        want.append((bufs[i]["out"].clone(), prompts[i][3].clone()))
    q, k, v, _, _ = prompts[3]
    n = q.shape[0]
    for r in (0, n // 3 - 1):
        w, tol = au.attention(host(q)[r:r + 1], host(k), host(v), r)
        au.check(host(want[3][1])[r:r + 1], w, tol)
    streams = [torch.cuda.Stream() for _ in range(4)]
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for i in range(2):
        with torch.cuda.graph(graphs[i], stream=streams[i]):
            work(i, streams[i].cuda_stream)
    for _ in range(6):
        for i in range(4):
            bufs[i]["out"].zero_()
            prompts[i][3].zero_()
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
            work(i + 2, streams[i + 2].cuda_stream)
        torch.cuda.synchronize()
        for i in range(4):
            assert torch.equal(bufs[i]["out"], want[i][0]) and torch.equal(prompts[i][3], want[i][1]), i


def test_threads_with_planes_and_parts(ctx, monkeypatch):
    """Threads of one context, each on its stream, whose calls all take workspace."""
    import torch
    monkeypatch.setenv("GGQ_PROMPT_MFMA", "1")
    monkeypatch.setenv("GGQ_KV_SPLITS", "7")
    gen = _generator(51)
    lays = [Layer(ctx, 2, 2, 1024, 8, 2, 128, 4, 4, seed=i) for i in range(3)]
    data, prompts, want, errs = [], [], [], []
    for i, x in enumerate(lays):
        x.len.copy_(t(np.array([1500, 41 + i], np.int32)))
        k, v = (torch.randn((1541 + i, 2, 128), device="cuda", generator=gen) for _ in range(2))
        b = _buffers(x, 2, 30 + i)
        x.store(k, v, t(np.array([0, 1500, 1541 + i], np.int32)), stream())
        p = _prompt_of(x, 300 + 60 * i, gen)
        _token_step(x, b, stream())
        x.prompt(*p[:4], p[4], p[4], stream())
        torch.cuda.synchronize()
        want.append((b["out"].clone(), p[3].clone()))
        data.append(b)
        prompts.append(p)

    def go(i):
        try:
            s = torch.cuda.Stream()
            for _ in range(20):
                p = prompts[i]
                lays[i].prompt(*p[:4], p[4], p[4], s.cuda_stream)
                _token_step(lays[i], data[i], s.cuda_stream)
            s.synchronize()
        except Exception as e:  # noqa: BLE001
            errs.append(e)
    torch.cuda.synchronize()
    ts = [threading.Thread(target=go, args=(i,)) for i in range(3)]
    for x in ts:
        x.start()
    for x in ts:
        x.join()
    assert not errs
    for b, p, (a, c) in zip(data, prompts, want):
        assert torch.equal(b["out"], a) and torch.equal(p[3], c)


@pytest.fixture(params=["", "1"], ids=["rule", "mfma"])
def route(request, monkeypatch):
    monkeypatch.setenv("GGQ_PROMPT_MFMA", request.param)


@pytest.mark.parametrize("type", [0, 1])
@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 64, 65, 127, 129, 300])
def test_wide_heads_lengths(ctx, route, n, type):
    run(ctx, n, [0, n], None, 3, 1, 256, type, rows=[0, n // 2, n - 2, n - 1] if n > 2 else None)


@pytest.mark.parametrize("type", [0, 1])
@pytest.mark.parametrize("window", [0, 1, 33, 64, 200])
def test_wide_heads_windows_and_chunks(ctx, route, window, type):
    run(ctx, window, [0, 40, 41, 60, 63], [0, 300, 417, 427, 427], 8, 2, 256, type, window=window, rows=[0, 9, 10, 18, 39])
    run(ctx, window + 1, [3, 20, 145], [5, 22, 190], 2, 2, 256, type, window=window, behind=2, pad=8, rows=[0, 16, 70, 124])


@pytest.mark.parametrize("splits", ["1", "2", "5", "1000"])
@pytest.mark.parametrize("type", [0, 1])
def test_wide_heads_parts(ctx, monkeypatch, splits, type):
    monkeypatch.setenv("GGQ_PROMPT_MFMA", "1")
    monkeypatch.setenv("GGQ_PROMPT_SPLITS", splits)
    run(ctx, 30, [0, 40, 41, 41, 60], [0, 300, 700, 710, 729], 6, 2, 256, type, behind=3, rows=[0, 18, 39])
    run(ctx, 31, [2, 90], [0, 260], 4, 1, 256, type, window=100, rows=[0, 50, 87])


@pytest.mark.parametrize("splits", ["1", "3"])
def test_wide_heads_in_groups(ctx, monkeypatch, splits):
    """More than 256 MB of planes: the kv heads go in groups of six."""
    monkeypatch.setenv("GGQ_PROMPT_SPLITS", splits)
    run(ctx, 52, [0, 3], [0, 20011], 8, 8, 256, 0, rows=[0, 2])


@pytest.mark.parametrize("type", [0, 1])
def test_wide_heads_captured(ctx, monkeypatch, type):
    """Captured once; inputs and offsets change between the replays, and each equals the eager call bit for bit."""
    import torch
    monkeypatch.setenv("GGQ_PROMPT_MFMA", "1")
    gen = _generator(53)
    lay = Layer(ctx, 1, 1, 32, 8, 2, 256, 4, 4)
    rows = 300
    q, k, v, out, off = _prompt_of(lay, rows, gen)
    if type:
        k, v = k.half(), v.half()
    ref = torch.empty_like(out)
    lay.prompt(q, k, v, ref, off, off, stream(), type)
    torch.cuda.synchronize()
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        lay.prompt(q, k, v, out, off, off, s.cuda_stream, type)
    for i in range(5):
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, device="cuda", generator=gen))
        off.copy_(t(np.array([0, 1 + 7 * i, rows - i], np.int32)))
        out.zero_()
        ref.zero_()
        torch.cuda.synchronize()
        g.replay()
        lay.prompt(q, k, v, ref, off, off, stream(), type)
        torch.cuda.synchronize()
        assert torch.equal(out, ref), i
        r = 1 + 7 * i
        w, tol = au.attention(host(q)[r:r + 1], host(k)[r:], host(v)[r:], 0)
        au.check(host(out)[r:r + 1], w, tol)


def _cache(ctx, n_pages, page_len, n_kv, hd, kt, vt, table, lens, max_len):
    import ctypes

    import torch
    size = ctx.lib.ggq_kv_page_bytes(ctypes.byref(gl.KvCache(None, 0, page_len, n_kv, hd, kt, vt)))
    mem = torch.full((n_pages, size), 0x22, dtype=torch.uint8, device="cuda")
    tab, ln = t(np.asarray(table, np.int32)), t(np.asarray(lens, np.int32))
    keep = (mem, tab, ln)
    return (gl.KvCache(mem.data_ptr(), n_pages, page_len, n_kv, hd, kt, vt),
            gl.KvSeqs(len(lens), len(table[0]), max_len, tab.data_ptr(), ln.data_ptr()), keep)


def test_pages_that_several_sequences_read(ctx):
    """A common start of two pages and one of its own for each of three sequences; one of them twice in the call."""
    import torch
    n_kv, hd, page = 2, 128, 64
    gen = _generator(54)
    k, v = (torch.randn((5 * page, n_kv, hd), device="cuda", generator=gen) for _ in range(2))
    cache, seqs, keep = _cache(ctx, 6, page, n_kv, hd, 8, 4, [[4, 0, 2, 5, 1]], [5 * page], 5 * page)
    ld = n_kv * hd
    off = t(np.array([0, 5 * page], np.int32))
    ctx.check(ctx.lib.ggq_kv_store_dev(ctx.h, cache, seqs, off.data_ptr(), 5 * page, k.data_ptr(), ld, v.data_ptr(), ld, 0, stream()), "store")
    lens = [150, 130, 192, 150]
    table, ln = t(np.array([[4, 0, 2], [4, 0, 5], [4, 0, 1], [4, 0, 2]], np.int32)), t(np.array(lens, np.int32))
    shared = gl.KvSeqs(4, 3, 192, table.data_ptr(), ln.data_ptr())
    q, out = torch.randn((4, 4, hd), device="cuda", generator=gen), torch.empty((4, 4, hd), device="cuda")
    q[3] = q[0]
    ctx.check(ctx.lib.ggq_attention_kv_dev(ctx.h, cache, shared, q.data_ptr(), 4 * hd, 4, 0.0, 0, out.data_ptr(), 4 * hd, stream()), "a")
    kk, vv = au.kv_quantize(host(k), 8)[0], au.kv_quantize(host(v), 4)[0]
    got = host(out)
    for s, last in enumerate((2, 3, 4, 2)):
        at = np.concatenate([np.arange(2 * page), np.arange(last * page, (last + 1) * page)])[:lens[s]]
        want, tol = au.attention(host(q)[s:s + 1], kk[at], vv[at], lens[s] - 1)
        au.check(got[s:s + 1], want, tol)
    assert np.array_equal(got[0], got[3])
    k2, v2 = (torch.full((sum(lens), n_kv, hd), 5.0, device="cuda") for _ in range(2))
    off = t(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32))
    ctx.check(ctx.lib.ggq_kv_load_dev(ctx.h, cache, shared, off.data_ptr(), sum(lens), k2.data_ptr(), ld, v2.data_ptr(), ld, 0, stream()), "l")
    at = np.concatenate([np.concatenate([np.arange(2 * page), np.arange(x * page, (x + 1) * page)])[:n] for x, n in zip((2, 3, 4, 2), lens)])
    assert np.array_equal(host(k2), kk[at].astype(np.float32)) and np.array_equal(host(v2), vv[at].astype(np.float32))


def test_more_rows_than_positions(ctx):
    """Rows of a sequence beyond its length have positions below 0: nothing is stored or loaded for them."""
    import torch
    n_kv, hd, page = 1, 64, 32
    gen = _generator(55)
    k, v = (torch.randn((60, n_kv, hd), device="cuda", generator=gen) for _ in range(2))
    cache, seqs, keep = _cache(ctx, 4, page, n_kv, hd, 4, 4, [[2, 0], [1, 3]], [10, -3], 64)
    off = t(np.array([0, 40, 60], np.int32))
    mem = keep[0]
    before = host(mem)
    ctx.check(ctx.lib.ggq_kv_store_dev(ctx.h, cache, seqs, off.data_ptr(), 60, k.data_ptr(), 64, v.data_ptr(), 64, 0, stream()), "store")
    after = host(mem)
    assert np.array_equal(after[[0, 1, 3]], before[[0, 1, 3]])
    K, V = au.kv_unpack(after, n_kv, page, hd, 4, 4)
    K0, V0 = au.kv_unpack(before, n_kv, page, hd, 4, 4)
    assert np.array_equal(K[2, :10], au.kv_quantize(host(k)[30:40], 4)[0]) and np.array_equal(K[2, 10:], K0[2, 10:])
    assert np.array_equal(V[2, :10], au.kv_quantize(host(v)[30:40], 4)[0]) and np.array_equal(V[2, 10:], V0[2, 10:])
    k2, v2 = (torch.full((60, n_kv, hd), 5.0, device="cuda") for _ in range(2))
    ctx.check(ctx.lib.ggq_kv_load_dev(ctx.h, cache, seqs, off.data_ptr(), 60, k2.data_ptr(), 64, v2.data_ptr(), 64, 0, stream()), "load")
    assert (host(k2)[:30] == 5).all() and (host(k2)[40:] == 5).all() and (host(v2)[:30] == 5).all() and (host(v2)[40:] == 5).all()
    assert np.array_equal(host(k2)[30:40], K[2, :10].astype(np.float32)) and np.array_equal(host(v2)[30:40], V[2, :10].astype(np.float32))
