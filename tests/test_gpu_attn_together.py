"""The operators between the q/k/v and the output projections as they are used together: a prompt and its next tokens
through rotary positions, cache and attention; captured and replayed; on several streams at once; far into large
buffers; without workspace."""
import ctypes
import threading

import numpy as np
import pytest

import ggnpu_amd.lib as gl
from tests import attn_util as au
from tests.gpu_util import host, ptr

pytestmark = pytest.mark.gpu
EPS = 1e-6


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


class Layer:
    """One layer's cache and the calls around it; every buffer is allocated once, so that calls can be captured."""

    def __init__(self, ctx, n_seq, per, page_len, n_head, n_kv, hd, kt, vt, seed=0, rot=0, norm=True):
        import torch
        rng = np.random.default_rng(seed)
        self.ctx, self.n_seq, self.n_head, self.n_kv, self.hd = ctx, n_seq, n_head, n_kv, hd
        self.page_len, self.kt, self.vt = page_len, kt, vt
        n_pages = n_seq * per + 1
        size = gl.load_library().ggq_kv_page_bytes(ctypes.byref(gl.KvCache(None, 0, page_len, n_kv, hd, kt, vt)))
        self.pool = torch.zeros((n_pages, size), dtype=torch.uint8, device="cuda")
        self.cache = gl.KvCache(self.pool.data_ptr(), n_pages, page_len, n_kv, hd, kt, vt)
        self.table_np = rng.permutation(n_pages)[: n_seq * per].reshape(n_seq, per).astype(np.int32)
        self.table = t(self.table_np)
        self.len = torch.zeros(n_seq, dtype=torch.int32, device="cuda")
        self.seqs = gl.KvSeqs(n_seq, per, per * page_len, self.table.data_ptr(), self.len.data_ptr())
        self.rope = gl.Rope(ctx, hd, rot, gl.RopeLayout.HALF, 10000.0)
        self.w = t((1 + 0.1 * rng.standard_normal(hd)).astype(np.float32)) if norm else None

    def turn(self, q, k, q_out, k_out, pos, stream):
        sets = (gl.RopeHeads * 2)()
        for s, x, o in ((sets[0], q, q_out), (sets[1], k, k_out)):
            n = x.shape[1]
            s.x, s.ldx, s.n_head, s.out, s.ldo, s.out_type = x.data_ptr(), n * self.hd, n, o.data_ptr(), n * self.hd, 0
            s.norm_w = self.w.data_ptr() if self.w is not None else None
        self.ctx.check(self.ctx.lib.ggq_rope_dev(self.ctx.h, self.rope.h, sets, 2, ptr(pos), q.shape[0], EPS, stream), "rope")

    def store(self, k, v, off, stream):
        ld = self.n_kv * self.hd
        self.ctx.check(self.ctx.lib.ggq_kv_store_dev(self.ctx.h, self.cache, self.seqs, None if off is None else ptr(off), k.shape[0],
                                                     ptr(k), ld, ptr(v), ld, 0, stream), "store")

    def load(self, k, v, off, stream):
        ld = self.n_kv * self.hd
        self.ctx.check(self.ctx.lib.ggq_kv_load_dev(self.ctx.h, self.cache, self.seqs, ptr(off), k.shape[0], ptr(k), ld, ptr(v), ld, 0,
                                                    stream), "load")

    def decode(self, q, out, stream):
        ld = self.n_head * self.hd
        self.ctx.check(self.ctx.lib.ggq_attention_kv_dev(self.ctx.h, self.cache, self.seqs, ptr(q), ld, self.n_head, 0.0, 0, ptr(out),
                                                         ld, stream), "decode")

    def prompt(self, q, k, v, out, q_off, kv_off, stream, type=0):
        ld, lk = self.n_head * self.hd, self.n_kv * self.hd
        p = gl.AttnPromptParams(type=type, n_head=self.n_head, n_kv_head=self.n_kv, head_dim=self.hd, q=q.data_ptr(), ldq=ld,
                                k=k.data_ptr(), ldk=lk, v=v.data_ptr(), ldv=lk, out=out.data_ptr(), ldo=ld, n_rows=q.shape[0],
                                n_kv_rows=k.shape[0], n_seq=q_off.numel() - 1, q_off=q_off.data_ptr(), kv_off=kv_off.data_ptr())
        self.ctx.check(self.ctx.lib.ggq_attention_prompt_dev(self.ctx.h, p, stream), "prompt")

    def values(self):
        k, v = au.kv_unpack(host(self.pool), self.n_kv, self.page_len, self.hd, self.kt, self.vt)
        return [[x[self.table_np[s]].reshape(-1, self.n_kv, self.hd) for x in (k, v)] for s in range(self.n_seq)]


def stream():
    import torch
    return torch.cuda.current_stream().cuda_stream


def test_prompts_then_tokens(ctx):
    """Two prompts of different lengths: turned, attended, stored; a second chunk of the first against the cache read
    back; then four tokens of both over the cache.  Each stage against 64 bits on the stage's own inputs."""
    import torch
    lay = Layer(ctx, 2, 3, 64, 8, 2, 128, 8, 4, rot=64)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    new = lambda n, h: torch.randn((n, h, 128), device="cuda", generator=gen)  # noqa: E731
    lens = [70, 33]
    off = t(np.array([0, 70, 103], np.int32))
    q, k, v = new(103, 8), new(103, 2), new(103, 2)
    pos = t(np.concatenate([np.arange(70), np.arange(33)]).astype(np.int32))
    qr, kr, out = torch.empty_like(q), torch.empty_like(k), torch.empty_like(q)
    lay.turn(q, k, qr, kr, pos, stream())
    lay.prompt(qr, kr, v, out, off, off, stream())
    lay.len.copy_(t(np.array(lens, np.int32)))
    lay.store(kr, v, off, stream())
    Q, K, V, O = host(qr), host(kr), host(v), host(out)
    for a, b in ((0, 70), (70, 103)):
        want, tol = au.attention(Q[a:b], K[a:b], V[a:b], 0)
        au.check(O[a:b], want, tol)
    for s, (a, b) in enumerate(((0, 70), (70, 103))):
        kk, vv = lay.values()[s]
        assert np.array_equal(kk[: b - a], au.kv_quantize(K[a:b], 8)[0]) and np.array_equal(vv[: b - a], au.kv_quantize(V[a:b], 4)[0])
    # a second chunk of 25 rows of the first sequence, against its 95 positions read back
    q2, k2, v2 = new(25, 8), new(25, 2), new(25, 2)
    qr2, kr2, out2 = torch.empty_like(q2), torch.empty_like(k2), torch.empty_like(q2)
    lay.turn(q2, k2, qr2, kr2, t(np.arange(70, 95, dtype=np.int32)), stream())
    lay.len.copy_(t(np.array([95, 33], np.int32)))
    lay.store(kr2, v2, t(np.array([0, 25, 25], np.int32)), stream())
    kall, vall = (torch.empty((95, 2, 128), device="cuda") for _ in range(2))
    lay.load(kall, vall, t(np.array([0, 95, 95], np.int32)), stream())
    lay.prompt(qr2, kall, vall, out2, t(np.array([0, 25], np.int32)), t(np.array([0, 95], np.int32)), stream())
    kk, vv = lay.values()[0]
    assert np.array_equal(host(kall), kk[:95].astype(np.float32)) and np.array_equal(host(vall), vv[:95].astype(np.float32))
    want, tol = au.attention(host(qr2), kk[:95], vv[:95], 70)
    au.check(host(out2), want, tol)
    # tokens
    lens = [95, 33]
    for _ in range(4):
        lens = [n + 1 for n in lens]
        lay.len.copy_(t(np.array(lens, np.int32)))
        q, k, v = new(2, 8), new(2, 2), new(2, 2)
        qr, kr, out = torch.empty_like(q), torch.empty_like(k), torch.empty_like(q)
        lay.turn(q, k, qr, kr, t(np.array([n - 1 for n in lens], np.int32)), stream())
        lay.store(kr, v, None, stream())
        lay.decode(qr, out, stream())
        got, Q = host(out), host(qr)
        for s, n in enumerate(lens):
            kk, vv = lay.values()[s]
            assert np.array_equal(kk[n - 1], au.kv_quantize(host(kr)[s], 8)[0])
            want, tol = au.attention(Q[s:s + 1], kk[:n], vv[:n], n - 1)
            au.check(got[s:s + 1], want, tol)


def _token_step(lay, b, s):
    lay.turn(b["q"], b["k"], b["qr"], b["kr"], b["pos"], s)
    lay.store(b["kr"], b["v"], None, s)
    lay.decode(b["qr"], b["out"], s)


def _buffers(lay, n, seed):
    import torch
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    b = {x: torch.randn((n, h, lay.hd), device="cuda", generator=gen) for x, h in (("q", lay.n_head), ("k", lay.n_kv), ("v", lay.n_kv))}
    b["qr"], b["kr"], b["out"] = torch.empty_like(b["q"]), torch.empty_like(b["k"]), torch.empty_like(b["q"])
    b["pos"] = torch.zeros(n, dtype=torch.int32, device="cuda")
    return b


def test_captured_token_steps(ctx):
    """A token step captured once and replayed as the sequences grow (lengths and positions on the device), eager work
    between the replays; every replay equals the eager step on an equal cache bit for bit."""
    import torch
    a, b = (Layer(ctx, 3, 5, 1024, 8, 2, 128, 4, 4, seed=5) for _ in range(2))
    gen = torch.Generator(device="cuda")
    gen.manual_seed(9)
    lens = np.array([4000, 37, 1023], np.int32)
    total = int(lens.sum())
    k, v = (torch.randn((total, 2, 128), device="cuda", generator=gen) for _ in range(2))
    off = t(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32))
    for x in (a, b):
        x.len.copy_(t(lens))
        x.store(k, v, off, stream())
    ba, bb = _buffers(a, 3, 1), _buffers(b, 3, 1)
    _token_step(a, ba, stream())  # sizes the workspace (and writes the last position of a; b gets the same)
    _token_step(b, bb, stream())
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        _token_step(a, ba, s.cuda_stream)
    for i in range(5):
        new = [torch.randn((3, h, 128), device="cuda", generator=gen) for h in (8, 2, 2)]
        for x, buf in ((a, ba), (b, bb)):
            x.len.copy_(t(lens + 1 + i))
            buf["pos"].copy_(t(lens + i))
            for n, val in zip(("q", "k", "v"), new):
                buf[n].copy_(val)
        torch.cuda.synchronize()
        g.replay()
        _token_step(b, bb, stream())
        torch.cuda.synchronize()
        assert torch.equal(ba["out"], bb["out"]) and torch.equal(a.pool, b.pool), i
    kk, vv = b.values()[0]
    want, tol = au.attention(host(bb["qr"])[:1], kk[:4005], vv[:4005], 4004)
    au.check(host(bb["out"])[:1], want, tol)


@pytest.mark.parametrize("rows,route", [(40, ""), (300, "1")])
def test_captured_prompts(ctx, monkeypatch, rows, route):
    """Prompt attention captured on both routes; offsets rewritten between replays."""
    import torch
    monkeypatch.setenv("GGQ_PROMPT_MFMA", route)
    lay = Layer(ctx, 1, 1, 32, 8, 2, 64, 4, 4)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(2)
    q, k, v = (torch.randn((rows, h, 64), device="cuda", generator=gen) for h in (8, 2, 2))
    off = t(np.array([0, rows // 3, rows], np.int32))
    out, ref = torch.empty_like(q), torch.empty_like(q)
    lay.prompt(q, k, v, ref, off, off, stream())
    torch.cuda.synchronize()
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        lay.prompt(q, k, v, out, off, off, s.cuda_stream)
    for i in range(4):
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, device="cuda", generator=gen))
        off.copy_(t(np.array([0, 1 + 7 * i, rows - i], np.int32)))
        out.zero_()
        ref.zero_()
        torch.cuda.synchronize()
        g.replay()
        lay.prompt(q, k, v, ref, off, off, stream())
        torch.cuda.synchronize()
        assert torch.equal(out, ref), i


def test_capture_without_workspace():
    """A fresh context has nothing set aside for captures: cache attention runs in one part, prompts without planes."""
    import torch
    c = gl.Context(0)
    try:
        lay = Layer(c, 1, 1, 4096, 8, 2, 64, 4, 4)
        gen = torch.Generator(device="cuda")
        gen.manual_seed(3)
        n = 3000
        k, v = (torch.randn((n, 2, 64), device="cuda", generator=gen) for _ in range(2))
        lay.len.fill_(n)
        lay.store(k, v, t(np.array([0, n], np.int32)), stream())
        q, out = torch.randn((1, 8, 64), device="cuda", generator=gen), torch.empty((1, 8, 64), device="cuda")
        pq, pout = torch.randn((700, 8, 64), device="cuda", generator=gen), torch.empty((700, 8, 64), device="cuda")
        off = t(np.array([0, 700], np.int32))
        torch.cuda.synchronize()
        s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            lay.decode(q, out, s.cuda_stream)
            lay.prompt(pq, k, v, pout, off, off, s.cuda_stream)
        for _ in range(3):
            out.zero_()
            pout.zero_()
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
        kk, vv = lay.values()[0]
        want, tol = au.attention(host(q), kk[:n], vv[:n], n - 1)
        au.check(host(out), want, tol)
        K, V, Q = host(k)[:700], host(v)[:700], host(pq)
        for i in (0, 63, 64, 500, 699):
            want, tol = au.attention(Q[i:i + 1], K, V, i)
            au.check(host(pout)[i:i + 1], want, tol)
    finally:
        c.close()


def test_two_graphs_and_two_streams_at_once(ctx):
    """Two captured calls that need workspace and two eager ones, all in flight together on four streams of one context."""
    import torch
    lays = [Layer(ctx, 1, 1, 8192, 8, 2, 64, 4, 8, seed=i) for i in range(4)]
    bufs = [_buffers(x, 1, 20 + i) for i, x in enumerate(lays)]
    gen = torch.Generator(device="cuda")
    gen.manual_seed(4)
    prompts = []
    for i, x in enumerate(lays):
        k, v = (torch.randn((8000, 2, 64), device="cuda", generator=gen) for _ in range(2))
        x.len.fill_(8000)
        x.store(k, v, t(np.array([0, 8000], np.int32)), stream())
        n = 400 + 50 * i
        q = torch.randn((n, 8, 64), device="cuda", generator=gen)
        prompts.append((q, k[:n].contiguous(), v[:n].contiguous(), torch.empty_like(q), t(np.array([0, n], np.int32))))

    def work(i, s):
        lays[i].decode(bufs[i]["q"], bufs[i]["out"], s)
        q, k, v, out, off = prompts[i]
        lays[i].prompt(q, k, v, out, off, off, s)
    want = []
    for i in range(4):
        work(i, stream())
        torch.cuda.synchronize()
        want.append((bufs[i]["out"].clone(), prompts[i][3].clone()))
    streams = [torch.cuda.Stream() for _ in range(4)]
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for i in range(2):
        with torch.cuda.graph(graphs[i], stream=streams[i]):
            work(i, streams[i].cuda_stream)
    for _ in range(5):
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


def test_threads_share_a_context(ctx):
    import torch
    lays = [Layer(ctx, 2, 2, 256, 8, 2, 128, 4, 4, seed=i) for i in range(3)]
    gen = torch.Generator(device="cuda")
    gen.manual_seed(6)
    data, want, got, errs = [], [], [None] * 3, []
    for i, x in enumerate(lays):
        x.len.copy_(t(np.array([300, 41 + i], np.int32)))
        k, v = (torch.randn((341 + i, 2, 128), device="cuda", generator=gen) for _ in range(2))
        b = _buffers(x, 2, 30 + i)
        off = t(np.array([0, 300, 341 + i], np.int32))
        x.store(k, v, off, stream())
        _token_step(x, b, stream())
        torch.cuda.synchronize()
        want.append(b["out"].clone())
        data.append(b)

    def run(i):
        try:
            import torch
            s = torch.cuda.Stream()
            for _ in range(20):
                _token_step(lays[i], data[i], s.cuda_stream)
            s.synchronize()
            got[i] = data[i]["out"]
        except Exception as e:  # noqa: BLE001
            errs.append(e)
    ts = [threading.Thread(target=run, args=(i,)) for i in range(3)]
    for x in ts:
        x.start()
    for x in ts:
        x.join()
    assert not errs
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_pages_beyond_4_gib(ctx):
    """A pool of 5 GB whose last pages are in use."""
    import torch
    n_kv, hd, page_len = 2, 256, 1024
    size = gl.load_library().ggq_kv_page_bytes(ctypes.byref(gl.KvCache(None, 0, page_len, n_kv, hd, 8, 8)))
    n_pages = (5 << 30) // size
    pool = torch.empty((n_pages, size), dtype=torch.uint8, device="cuda")
    cache = gl.KvCache(pool.data_ptr(), n_pages, page_len, n_kv, hd, 8, 8)
    table = np.array([[n_pages - 1, 0], [3, n_pages - 2]], np.int32)
    dt, ln = t(table), t(np.array([1500, 1100], np.int32))
    seqs = gl.KvSeqs(2, 2, 1500, dt.data_ptr(), ln.data_ptr())
    gen = torch.Generator(device="cuda")
    gen.manual_seed(7)
    k, v = (torch.randn((2600, n_kv, hd), device="cuda", generator=gen) for _ in range(2))
    off = t(np.array([0, 1500, 2600], np.int32))
    lib = ctx.lib
    ctx.check(lib.ggq_kv_store_dev(ctx.h, cache, seqs, ptr(off), 2600, ptr(k), 512, ptr(v), 512, 0, stream()), "store")
    k2, v2 = torch.empty_like(k), torch.empty_like(v)
    ctx.check(lib.ggq_kv_load_dev(ctx.h, cache, seqs, ptr(off), 2600, ptr(k2), 512, ptr(v2), 512, 0, stream()), "load")
    kk, vv = au.kv_quantize(host(k), 8)[0], au.kv_quantize(host(v), 8)[0]
    assert np.array_equal(host(k2), kk.astype(np.float32)) and np.array_equal(host(v2), vv.astype(np.float32))
    q, out = torch.randn((2, 4, hd), device="cuda", generator=gen), torch.empty((2, 4, hd), device="cuda")
    ctx.check(lib.ggq_attention_kv_dev(ctx.h, cache, seqs, ptr(q), 1024, 4, 0.0, 0, ptr(out), 1024, stream()), "attention")
    for s, (a, b) in enumerate(((0, 1500), (1500, 2600))):
        want, tol = au.attention(host(q)[s:s + 1], kk[a:b], vv[a:b], b - a - 1)
        au.check(host(out)[s:s + 1], want, tol)


@pytest.mark.parametrize("route", ["0", "1"])
def test_rows_beyond_4_gib(ctx, monkeypatch, route):
    """Rows 16 MB apart: offsets pass 32 bits within the call (and 2^31 elements in the fp32 slab)."""
    import torch
    monkeypatch.setenv("GGQ_PROMPT_MFMA", route)
    n, ld = 300, 4 << 20
    gen = torch.Generator(device="cuda")
    gen.manual_seed(8)
    big = torch.empty(n * ld + 4096, device="cuda")
    rows = big[: n * ld].view(n, ld)
    q, k, v = (torch.randn((n, w), device="cuda", generator=gen) for w in (256, 64, 64))
    rows[:, :256], rows[:, 256:320], rows[:, 320:384] = q, k, v
    off = t(np.array([0, n], np.int32))
    p = gl.AttnPromptParams(type=0, n_head=4, n_kv_head=1, head_dim=64, q=big.data_ptr(), ldq=ld, k=big.data_ptr() + 1024, ldk=ld,
                            v=big.data_ptr() + 1280, ldv=ld, out=big.data_ptr() + 1536, ldo=ld, n_rows=n, n_kv_rows=n, n_seq=1,
                            q_off=off.data_ptr())
    ctx.check(ctx.lib.ggq_attention_prompt_dev(ctx.h, p, stream()), "prompt")
    got = host(rows[:, 384:640]).reshape(n, 4, 64)
    Q, K, V = host(q).reshape(n, 4, 64), host(k).reshape(n, 1, 64), host(v).reshape(n, 1, 64)
    for i in (0, 130, 255, 256, 299):
        want, tol = au.attention(Q[i:i + 1], K, V, i)
        au.check(got[i:i + 1], want, tol)


def test_planes_in_groups_of_heads(ctx, monkeypatch):
    """More than 256 MB of planes: the kv heads go in groups, with and without parts of the positions."""
    import torch
    n_kv, hd, keys, rows = 14, 128, 20011, 70
    gen = torch.Generator(device="cuda")
    gen.manual_seed(10)
    q = torch.randn((rows, n_kv, hd), device="cuda", generator=gen)
    k, v = (torch.randn((keys, n_kv, hd), device="cuda", generator=gen) for _ in range(2))
    qo, ko = t(np.array([0, rows], np.int32)), t(np.array([0, keys], np.int32))
    for splits in ("1", "3"):
        monkeypatch.setenv("GGQ_PROMPT_SPLITS", splits)
        out = torch.empty_like(q)
        p = gl.AttnPromptParams(type=0, n_head=n_kv, n_kv_head=n_kv, head_dim=hd, q=q.data_ptr(), ldq=n_kv * hd, k=k.data_ptr(),
                                ldk=n_kv * hd, v=v.data_ptr(), ldv=n_kv * hd, out=out.data_ptr(), ldo=n_kv * hd, n_rows=rows,
                                n_kv_rows=keys, n_seq=1, q_off=qo.data_ptr(), kv_off=ko.data_ptr())
        ctx.check(ctx.lib.ggq_attention_prompt_dev(ctx.h, p, stream()), "prompt")
        got = host(out)
        for h in (0, 11, 12, 13):
            kk, vv = host(k[:, h:h + 1]), host(v[:, h:h + 1])
            for i in (0, 69):
                want, tol = au.attention(host(q)[i:i + 1, h:h + 1], kk, vv, keys - rows + i)
                au.check(got[i:i + 1, h:h + 1], want, tol)
