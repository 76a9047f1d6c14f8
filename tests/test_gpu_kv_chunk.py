"""ggq_attention_kv_rows_dev against 64 bits within the bound that attn_util.attention derives: by tiles over the records and
by planes of operands."""
import ctypes
import os

import numpy as np
import pytest

import ggnpu_amd.lib as gl
from tests import attn_util as au
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


@pytest.fixture(params=["tiles", "planes"])
def form(request, monkeypatch):
    monkeypatch.setenv("GGQ_KV_PLANES", "1" if request.param == "planes" else "0")
    return request.param


def row_of(q, k, v, scale, planes):
    """One row over all of k, v (it sees them all): attn_util.attention, and for the form by planes what its weights lose.

    A weight is kept times 2^11 as the sum of two fp16 numbers, so one that is small beside the largest is off by half the smallest fp16
    step, 2^-25: 2^-36 of the weight whose product with its position's largest value is largest, and up to 2^8 times as much where the
    position's values lie that far below the largest ones of their 32 positions.  So a position whose value is not zero adds up to
    2^-28 of that product (what fp32 has not, where the large weights' positions hold zeros: MXFP4 has many)."""
    want, tol = au.attention(q, k, v, len(k) - 1, 0, scale)
    if planes and len(k):
        G = q.shape[1] // k.shape[1]
        for h in range(q.shape[1]):
            kk, vv = k[:, h // G], np.abs(v[:, h // G])
            s = kk @ q[0, h].astype(np.float64) * (q.shape[2] ** -0.5 if scale is None else scale)
            with np.errstate(invalid="ignore"):
                p = np.exp(s - s.max())
                tol[0, h] += 2.0 ** -28 * (p / p.sum() * vv.max(1)).max() * (vv != 0).sum(0)
    return want, tol


class Case:
    """Sequences of lens positions whose last rows[s] are queries; before/behind: rows of no sequence."""

    def __init__(self, seed, lens, rows, n_head, n_kv, hd, kt, vt, page_len=64, before=0, behind=0, more=0, kscale=1.0):
        rng = np.random.default_rng(seed)
        self.lens, self.rows, self.heads, self.n_kv, self.hd, self.kt, self.vt, self.page_len = lens, rows, n_head, n_kv, hd, kt, vt, page_len
        per = max(1, -(-max(lens) // page_len)) + more
        n_pages = len(lens) * per + 2
        k, v = (rng.standard_normal((n_pages, page_len, n_kv, hd)) * np.exp2(rng.integers(-3, 4, (n_pages, page_len, n_kv, hd // 32))).repeat(32, -1)
                for _ in range(2))
        self.pool = au.kv_pack(k * kscale, v, n_kv, page_len, kt, vt)
        self.table = rng.permutation(n_pages)[: len(lens) * per].reshape(-1, per).astype(np.int32)
        self.off = np.concatenate([[before], before + np.cumsum(rows)]).astype(np.int32)
        n = before + sum(rows) + behind
        self.q = rng.standard_normal((n, n_head, hd)).astype(np.float32)

    def call(self, ctx, window=0, scale=0.0, pad=0, max_len=None, use_off=True, n_rows=None, pool=None):
        import torch
        n, width = len(self.q), self.heads * self.hd
        b = np.full((n, width + pad), 3.0, np.float32)
        b[:, :width] = self.q.reshape(n, -1)
        q, out = t(b), torch.full((n, width + pad), 7.0, device="cuda")
        mem = t(self.pool) if pool is None else pool
        table, lens, off = t(self.table), t(np.asarray(self.lens, np.int32)), t(self.off)
        c = gl.KvCache(mem.data_ptr(), len(self.pool), self.page_len, self.n_kv, self.hd, self.kt, self.vt)
        s = gl.KvSeqs(len(self.lens), self.table.shape[1], max(1, max(self.lens)) if max_len is None else max_len, table.data_ptr(), lens.data_ptr())
        ctx.check(ctx.lib.ggq_attention_kv_rows_dev(ctx.h, c, s, ptr(off) if use_off else None, n if n_rows is None else n_rows, ptr(q), width + pad,
                                                    self.heads, scale, window, ptr(out), width + pad, stream_handle()), "chunk")
        o = host(out)
        assert (o[:, width:] == 7).all()
        return o[:, :width].reshape(n, self.heads, self.hd)

    def seq_values(self, s):
        K, V = au.kv_unpack(self.pool, self.n_kv, self.page_len, self.hd, self.kt, self.vt)
        pages = self.table[s]
        there = (pages >= 0) & (pages < len(self.pool))
        k, v = (x[np.where(there, pages, 0)].reshape(-1, self.n_kv, self.hd) for x in (K, V))
        return k, v, np.repeat(there, self.page_len)

    def check(self, o, window=0, scale=None, max_len=None):
        inside = np.zeros(len(o), bool)
        for s, n in enumerate(self.lens):
            a, e = self.off[s], self.off[s + 1]
            k, v, there = self.seq_values(s)
            lim = min(n, len(k), n if max_len is None else max_len)
            first = n - (e - a)
            for i in range(e - a):
                hi = min(first + i + 1, lim)
                lo = max(0, first + i + 1 - window) if window else 0
                at = np.arange(lo, max(lo, hi))
                at = at[there[at]] if len(at) else at
                # (one row at its keys: they are all that it sees)
                want, tol = row_of(self.q[a + i:a + i + 1], k[at], v[at], scale, os.environ.get("GGQ_KV_PLANES") != "0")
                au.check(o[a + i:a + i + 1], want, tol)
            inside[a:e] = True
        assert (o[~inside] == 7).all()


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("kt,vt", [(4, 4), (8, 4), (4, 8), (8, 8)])
def test_formats(ctx, form, hd, kt, vt):
    c = Case(hd + kt, [150, 33], [21, 7], 4, 2, hd, kt, vt)
    c.check(c.call(ctx))


@pytest.mark.parametrize("n_head,n_kv", [(1, 1), (3, 1), (4, 4), (10, 2), (7, 1), (16, 2), (24, 1)])
def test_head_ratios(ctx, form, n_head, n_kv):
    c = Case(n_head, [70], [13], n_head, n_kv, 64, 8, 4)
    c.check(c.call(ctx))


@pytest.mark.parametrize("lens,rows", [([1], [1]), ([31], [31]), ([32], [2]), ([33], [33]), ([64, 65, 1, 300], [3, 64, 1, 9]), ([5, 0, 40], [5, 0, 4]),
                                       ([128], [128]), ([97, 97, 97], [0, 5, 0]), ([700], [40])])
@pytest.mark.parametrize("page_len", [32, 96])
def test_lengths(ctx, form, lens, rows, page_len):
    c = Case(sum(lens), lens, rows, 4, 2, 128, 8, 8, page_len, before=2, behind=3, more=1)
    c.check(c.call(ctx))


@pytest.mark.parametrize("window", [1, 31, 32, 33, 100, 5000, 2147483647])
def test_windows(ctx, form, window):
    c = Case(window % 97, [250, 40, 130], [50, 40, 1], 4, 1, 64, 4, 8)
    c.check(c.call(ctx, window=window), window=window)


@pytest.mark.parametrize("splits", ["1", "2", "5", "100"])
def test_parts_of_the_positions(ctx, form, monkeypatch, splits):
    monkeypatch.setenv("GGQ_KV_SPLITS" if form == "tiles" else "GGQ_PROMPT_SPLITS", splits)
    c = Case(3, [400, 90, 333], [6, 20, 3], 6, 2, 128, 4, 4)
    c.check(c.call(ctx))
    c.check(c.call(ctx, window=60), window=60)


def test_one_row_a_sequence_equals_the_token_call(ctx):
    """Without offsets a row is a sequence's token: zeros for a sequence without positions."""
    c = Case(4, [65, 1, 0, 200], [1, 1, 1, 1], 8, 2, 128, 8, 4)
    a, b = c.call(ctx, use_off=False), c.call(ctx)
    assert np.array_equal(a, b)
    c.check(a)
    assert (a[2] == 0).all()


def test_rows_before_position_zero(ctx, form):
    """More rows than positions: the first ones see nothing."""
    c = Case(5, [10, 3], [25, 3], 2, 1, 64, 8, 8)
    o = c.call(ctx)
    assert (o[:15] == 0).all()
    c.check(o)


def test_pages_that_do_not_exist(ctx, form):
    c = Case(6, [300, 64], [30, 8], 4, 2, 128, 8, 4, page_len=32)
    c.table[0, 3], c.table[0, 6], c.table[1, :] = -1, len(c.pool), -5
    o = c.call(ctx)
    c.check(o)
    assert (o[30:38] == 0).all()


def test_max_len_bounds_what_is_read(ctx, form):
    c = Case(7, [200], [20], 2, 1, 64, 4, 4)
    c.check(c.call(ctx, max_len=190), max_len=190)
    c.check(c.call(ctx, max_len=0), max_len=0)


def test_scale_strides_peaked_scores(ctx, form):
    c = Case(8, [120], [40], 4, 2, 128, 8, 8, kscale=6.0)
    c.check(c.call(ctx, scale=0.25, pad=8), scale=0.25)
    c.check(c.call(ctx, scale=-0.1), scale=-0.1)


def test_hidden_positions_may_hold_anything(ctx, form):
    """Codes of NaN and scales of 255 behind the sequences' ends, in front of their windows, and at later rows' positions."""
    c = Case(9, [75, 64], [20, 10], 4, 2, 128, 8, 4, page_len=32)
    clean = c.call(ctx, window=30)
    v0, ks, vs, end = au.kv_record(128, 8, 4)
    for s, n in enumerate(c.lens):
        for pos in [p for p in range(c.table.shape[1] * 32) if p >= n or p < n - c.rows[s] + 1 - 30]:
            rec = c.pool[c.table[s, pos // 32]].reshape(c.n_kv, 1, end)
            p = pos % 32
            kb, _, ksc = au.kv_places(128, 8, False)
            vb, _, vsc = au.kv_places(128, 4, True)
            rec[:, :, kb[p]] = 0x7F
            rec[:, :, ks + ksc[p]] = 255
            rec[:, :, vs + vsc[p]] = 255
    dirty = c.call(ctx, window=30)
    assert np.array_equal(clean, dirty)


def test_a_value_that_is_nan_spoils_no_row_that_does_not_see_it(ctx, form):
    c = Case(10, [90], [40], 2, 1, 64, 8, 8, page_len=32)
    clean = c.call(ctx)
    v0, ks, vs, end = au.kv_record(64, 8, 8)
    pos = 70  # seen by rows 20 .. 39
    rec = c.pool[c.table[0, pos // 32]].reshape(1, 1, end)
    rec[:, :, vs + au.kv_places(64, 8, True)[2][pos % 32, 1]] = 255
    o = c.call(ctx)
    assert np.array_equal(o[:20], clean[:20])


def test_scales_far_apart(ctx, form):
    """Positions and blocks of very different sizes, among them ones that the rows do not see."""
    rng = np.random.default_rng(11)
    c = Case(11, [200], [30], 4, 2, 128, 8, 8, page_len=32)
    k, v = (rng.standard_normal((len(c.pool), 32, 2, 128)) for _ in range(2))
    k *= np.exp2(rng.integers(-12, 1, (len(c.pool), 32, 2, 1)))
    v *= np.exp2(rng.integers(-30, 31, (len(c.pool), 32, 2, 1)))
    c.pool = au.kv_pack(k, v, 2, 32, 8, 8)
    c.check(c.call(ctx))


def test_long_cache_few_rows(ctx, form):
    c = Case(12, [6001, 2500], [5, 1], 8, 2, 128, 4, 4, page_len=256)
    c.check(c.call(ctx))


def test_many_sequences(ctx, form):
    """More of them than threads look at in one turn, most without rows."""
    rng = np.random.default_rng(13)
    lens = rng.integers(0, 40, 600).tolist()
    rows = [int(min(n, 2)) if i % 50 == 0 else 0 for i, n in enumerate(lens)]
    c = Case(13, lens, rows, 2, 1, 64, 4, 4, page_len=32, before=1)
    c.check(c.call(ctx))


def test_offsets_are_held_inside_the_rows(ctx, form):
    c = Case(14, [50, 60], [10, 30], 2, 1, 64, 8, 8)
    o = c.call(ctx, n_rows=35)
    c.off, c.rows = np.array([0, 10, 35], np.int32), [10, 25]
    c.check(o)


def test_same_every_time(ctx, form):
    c = Case(15, [900, 333], [100, 50], 8, 2, 128, 8, 4)
    a = c.call(ctx)
    for _ in range(3):
        assert np.array_equal(a, c.call(ctx))


def test_the_rule_takes_planes_for_prompts(ctx, monkeypatch):
    """Unforced calls equal the forced ones of the form that the rule chooses."""
    big, small = Case(16, [1400], [1100], 8, 2, 128, 4, 4), Case(17, [700], [8], 8, 2, 128, 4, 4)
    a, b = big.call(ctx), small.call(ctx)
    monkeypatch.setenv("GGQ_KV_PLANES", "0")
    assert np.array_equal(b, small.call(ctx))
    x = big.call(ctx)
    rows = [0, 1, 31, 500, 1099]
    k, v, _ = big.seq_values(0)
    for r in rows:
        for planes, o in ((True, a), (False, x)):
            au.check(o[r:r + 1], *row_of(big.q[r:r + 1], k[: 301 + r], v[: 301 + r], None, planes))


def test_a_cache_beyond_four_gigabytes(ctx):
    """Pages whose byte offsets do not fit 32 bits."""
    import torch
    n_kv, hd, page_len = 8, 256, 256
    size = gl.load_library().ggq_kv_page_bytes(ctypes.byref(gl.KvCache(None, 0, page_len, n_kv, hd, 8, 8)))
    n_pages = (5 << 30) // size
    mem = torch.empty((n_pages, size), dtype=torch.uint8, device="cuda")
    c = Case(18, [400], [6], 16, n_kv, hd, 8, 8, page_len)
    small = c.pool
    where = np.array([n_pages - 1, n_pages // 2, 3, 7], np.int32)[: len(small)]
    for i, w in enumerate(where):
        mem[int(w)].copy_(t(small[i]))
    for v in ("0", "1"):
        os.environ["GGQ_KV_PLANES"] = v
        try:
            table = c.table.copy()
            c.pool = np.zeros((n_pages, 1), np.uint8)  # (its length is the pool's)
            c.table = where[table]
            o = c.call(ctx, pool=mem)
        finally:
            c.pool, c.table = small, table
            del os.environ["GGQ_KV_PLANES"]
        c.check(o)


def test_refusals(ctx):
    import torch
    mem, i32 = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda"), torch.zeros(16, dtype=torch.int32, device="cuda")
    f = torch.zeros(1 << 16, device="cuda")
    P = f.data_ptr()

    def cache(**kw):
        return gl.KvCache(**{**dict(pages=mem.data_ptr(), n_pages=2, page_len=32, n_kv_head=1, head_dim=64, k_type=8, v_type=8), **kw})

    def seqs(**kw):
        return gl.KvSeqs(**{**dict(n_seq=1, table_len=1, max_len=32, pages=i32.data_ptr(), len=i32.data_ptr()), **kw})

    def st(c=None, s=None, off=i32.data_ptr(), n_rows=1, q=P, ldq=128, n_head=2, scale=0.0, window=0, out=P + 4096, ldo=128):
        return ctx.lib.ggq_attention_kv_rows_dev(ctx.h, c or cache(), s or seqs(), off, n_rows, q, ldq, n_head, scale, window, out, ldo, stream_handle())

    assert st() == 0 and st(n_rows=0, q=None, out=None) == 0 and st(s=seqs(n_seq=0)) == 0 and st(off=None) == 0
    for kw in (dict(c=cache(head_dim=80)), dict(c=cache(page_len=48)), dict(c=cache(k_type=5)), dict(c=cache(pages=None)), dict(c=cache(n_pages=0)),
               dict(c=cache(pages=mem.data_ptr() + 8)), dict(s=seqs(n_seq=-1)), dict(s=seqs(n_seq=65536)), dict(s=seqs(table_len=0)),
               dict(s=seqs(max_len=-1)), dict(s=seqs(pages=None)), dict(s=seqs(len=None)), dict(n_rows=-1), dict(q=None), dict(out=None),
               dict(q=P + 4), dict(out=P + 4), dict(ldq=127), dict(ldq=126), dict(ldq=130), dict(ldo=124), dict(ldo=130), dict(n_head=0),
               dict(c=cache(n_kv_head=2), n_head=3), dict(n_head=65536), dict(scale=float("nan")), dict(window=-1), dict(n_rows=2147483647, n_head=64), dict(n_rows=1 << 28)):
        assert st(**kw) == gl.Status.INVALID_PARAM, kw
    torch.cuda.synchronize()


def infinite_at(c, s, pos, keys=True, byte=254, code=None):
    """Position pos of sequence s reads back as infinite, keys (if they are meant) and values: the largest code under 2^127, or another."""
    v0, ks, vs, end = au.kv_record(c.hd, c.kt, c.vt)
    rec = c.pool[c.table[s, pos // c.page_len]].reshape(c.n_kv, c.page_len // 32, end)[:, pos % c.page_len // 32]
    p = pos % 32
    for bits, value, at, sc in ((c.kt, False, 0, ks), (c.vt, True, v0, vs)):
        if not (keys or value):
            continue
        places, _, scale = au.kv_places(c.hd, bits, value)
        rec[:, at + places[p]] = (0x77 if bits == 4 else 0x7E) if code is None else code
        rec[:, sc + scale[p]] = byte


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("kt,vt", [(8, 4), (4, 8), (8, 8)])
def test_hidden_positions_may_be_infinite(ctx, form, hd, kt, vt):
    """Behind the sequences' ends, in front of their windows, and at the positions of later rows of the same tile."""
    c = Case(30, [75, 64], [20, 10], 4, 2, hd, kt, vt, page_len=32)
    clean, kept = c.call(ctx, window=30), c.pool.copy()

    def check(rows):
        dirty = c.call(ctx, window=30)
        if form == "tiles":
            assert np.array_equal(clean[rows], dirty[rows])
        for r in rows:  # (by planes hidden values have a say in the powers of two, which is a matter of roundings)
            s = int(r >= 20)
            end = c.lens[s] - c.rows[s] + r - c.off[s] + 1
            k, v, _ = c.seq_values(s)
            au.check(dirty[r:r + 1], *row_of(c.q[r:r + 1], k[max(0, end - 30):end], v[max(0, end - 30):end], None, form == "planes"))

    for s, n in enumerate(c.lens):
        for pos in [p for p in range(c.table.shape[1] * 32) if p >= n or p < n - c.rows[s] + 1 - 30]:
            infinite_at(c, s, pos)
    check(range(30))
    # seen by some of a tile's rows: the others keep theirs
    c.pool = kept
    infinite_at(c, 0, 75 - 8)  # rows 12 .. 19
    infinite_at(c, 1, 64 - 10 + 1 - 30)  # row 0 of the second, by the window
    check([r for r in range(30) if not (12 <= r < 20 or r == 20)])


@pytest.mark.parametrize("kt,vt,byte,code", [(8, 4, 254, 0x77), (8, 4, 254, 0x44), (8, 4, 253, 0x66), (8, 8, 254, 0x7E), (8, 8, 247, 0x78), (8, 8, 250, 0xE1),
                                             (4, 8, 253, 0x48)])
def test_infinite_values_do_not_vanish(ctx, form, kt, vt, byte, code):
    """A row that sees one is not finite, in both forms; rows that do not see it keep theirs.  (The codes are the largest, and those
    that just pass 2^128.)"""
    c = Case(31, [90], [40], 2, 1, 64, kt, vt, page_len=32)
    clean = c.call(ctx)
    infinite_at(c, 0, 70, keys=False, byte=byte, code=code)  # seen by rows 20 .. 39
    assert (np.abs(c.seq_values(0)[1][70]) >= 2.0 ** 128).all()
    o = c.call(ctx)
    assert np.isfinite(o[:20]).all() and not np.isfinite(o[20:]).any()
    if form == "tiles":
        assert np.array_equal(o[:20], clean[:20])


def test_the_rule_takes_planes_beyond_both_limits(ctx, monkeypatch):
    """512 rows of four heads a kv head over 4000 positions: an unforced call is the one by planes, bit for bit."""
    monkeypatch.delenv("GGQ_KV_PLANES", raising=False)
    c = Case(32, [4000], [512], 32, 8, 128, 4, 4)
    a = c.call(ctx)
    monkeypatch.setenv("GGQ_KV_PLANES", "1")
    assert np.array_equal(a, c.call(ctx))
    monkeypatch.setenv("GGQ_KV_PLANES", "0")
    b = c.call(ctx)
    assert not np.array_equal(a, b)
    k, v, _ = c.seq_values(0)
    for r in (0, 300, 511):
        n = 4000 - 512 + r + 1
        for planes, o in ((True, a), (False, b)):
            au.check(o[r:r + 1], *row_of(c.q[r:r + 1], k[:n], v[:n], None, planes))


def test_planes_without_workspace_become_tiles(ctx, monkeypatch):
    """A captured call of such a size in a context with nothing set aside goes by tiles, in one part: the same results within the bound
    at every replay."""
    import torch
    monkeypatch.delenv("GGQ_KV_PLANES", raising=False)
    c = Case(33, [4000], [512], 32, 8, 128, 4, 4)
    k, v, _ = c.seq_values(0)
    mem, table, lens, off, q = t(c.pool), t(c.table), t(np.asarray(c.lens, np.int32)), t(c.off), t(c.q)
    out = torch.empty_like(q)
    x, s, g = gl.Context(0), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    cache = gl.KvCache(mem.data_ptr(), len(c.pool), c.page_len, c.n_kv, c.hd, c.kt, c.vt)
    seqs = gl.KvSeqs(1, c.table.shape[1], 4000, table.data_ptr(), lens.data_ptr())
    with torch.cuda.graph(g, stream=s):
        st = x.lib.ggq_attention_kv_rows_dev(x.h, cache, seqs, ptr(off), 512, ptr(q), 32 * 128, 32, 0.0, 0, ptr(out), 32 * 128,
                                             ctypes.c_void_p(s.cuda_stream))
    assert st == 0
    for _ in range(3):
        out.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        o = host(out)
        for r in (0, 129, 511):
            n = 4000 - 512 + r + 1
            au.check(o[r:r + 1], *row_of(c.q[r:r + 1], k[:n], v[:n], None, False))
    x.close()
