"""The quantized KV cache: rows into its pages and back (ggq_kv_store_dev, ggq_kv_load_dev), against the formats'
definition value for value, and the attention over it (ggq_attention_kv_dev) against 64 bits within the bound that
attn_util.attention derives."""
import ctypes

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


class Pool:
    """A pool of pages on the GPU with its page tables; `fill` is the byte that unwritten places hold."""

    def __init__(self, n_pages, page_len, n_kv, hd, kt, vt, fill=0, data=None):
        import torch
        self.shape = (n_kv, page_len, hd, kt, vt)
        size = gl.load_library().ggq_kv_page_bytes(ctypes.byref(gl.KvCache(None, 0, page_len, n_kv, hd, kt, vt)))
        assert size == n_kv * page_len // 32 * au.kv_record(hd, kt, vt)[-1]
        self.mem = torch.full((n_pages, size), fill, dtype=torch.uint8, device="cuda") if data is None else t(data)
        self.desc = gl.KvCache(self.mem.data_ptr(), n_pages, page_len, n_kv, hd, kt, vt)

    def seqs(self, table, lens, max_len=None):
        self.table, self.lens = t(np.asarray(table, np.int32)), t(np.asarray(lens, np.int32))
        return gl.KvSeqs(len(lens), np.asarray(table).shape[1], max(1, max(lens)) if max_len is None else max_len,
                         self.table.data_ptr(), self.lens.data_ptr())

    def values(self):
        n_kv, page_len, hd, kt, vt = self.shape
        return au.kv_unpack(host(self.mem), n_kv, page_len, hd, kt, vt)


def rows(rng, n, n_kv, hd, dtype=np.float32):
    x = rng.standard_normal((n, n_kv, hd)) * np.exp2(rng.integers(-6, 7, (n, n_kv, hd // 32))).repeat(32, -1)
    return x.astype(dtype)


def table_of(rng, n_seq, per, n_pages):
    return rng.permutation(n_pages)[: n_seq * per].reshape(n_seq, per).astype(np.int32)


def store(ctx, pool, seqs, off, k, v, pad=0):
    n, width = k.shape[0], k.shape[1] * k.shape[2]
    bufs = []
    for x in (k, v):
        b = np.full((n, width + pad), 9, x.dtype)
        b[:, :width] = x.reshape(n, width)
        bufs.append(t(b))
    o = None if off is None else t(np.asarray(off, np.int32))
    ctx.check(ctx.lib.ggq_kv_store_dev(ctx.h, pool.desc, seqs, None if o is None else ptr(o), n, ptr(bufs[0]), width + pad,
                                       ptr(bufs[1]), width + pad, int(k.dtype == np.float16), stream_handle()), "store")
    return bufs, o


def load(ctx, pool, seqs, off, n, dtype=np.float32, pad=0):
    import torch
    n_kv, _, hd = pool.shape[0], pool.shape[1], pool.shape[2]
    width = n_kv * hd
    bufs = [torch.full((n, width + pad), 5.0, dtype=torch.float16 if dtype == np.float16 else torch.float32, device="cuda")
            for _ in range(2)]
    o = None if off is None else t(np.asarray(off, np.int32))
    ctx.check(ctx.lib.ggq_kv_load_dev(ctx.h, pool.desc, seqs, None if o is None else ptr(o), n, ptr(bufs[0]), width + pad,
                                      ptr(bufs[1]), width + pad, int(dtype == np.float16), stream_handle()), "load")
    return [host(b) for b in bufs]


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("kt,vt", [(4, 4), (8, 4), (4, 8), (8, 8)])
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_store_then_load(ctx, hd, kt, vt, dtype):
    """Ragged sequences, new rows behind old positions, pages that end among them; everything else stays."""
    rng = np.random.default_rng(hd + kt + 10 * vt)
    n_kv, page_len = 3, 96
    lens, new = [1, 97, 250, 64, 33], [1, 97, 31, 0, 33]
    table = table_of(rng, 5, 3, 18)
    pool = Pool(18, page_len, n_kv, hd, kt, vt, fill=0x33)
    seqs = pool.seqs(table, lens)
    off = np.concatenate([[0], np.cumsum(new)])
    n = off[-1] + 2  # two rows of no sequence
    k, v = rows(rng, n, n_kv, hd, dtype), rows(rng, n, n_kv, hd, dtype)
    before = pool.values()
    store(ctx, pool, seqs, off, k, v, pad=8)
    want = [x.copy() for x in before]
    for s, (ln, nw) in enumerate(zip(lens, new)):
        for i in range(nw):
            pos, r = ln - nw + i, off[s] + i
            for x, src, bits in ((want[0], k, kt), (want[1], v, vt)):
                x[table[s, pos // page_len], pos % page_len] = au.kv_quantize(src[r].astype(np.float64), bits)[0]
    for got, w in zip(pool.values(), want):
        assert np.array_equal(got, w)
    got = load(ctx, pool, seqs, off, n, dtype, pad=16)
    for g, src, bits in zip(got, (k, v), (kt, vt)):
        w = au.kv_quantize(src[: off[-1]].astype(np.float64), bits)[0].astype(dtype)
        assert np.array_equal(g[: off[-1], : n_kv * hd].reshape(w.shape), w)
        assert (g[off[-1]:] == 5).all() and (g[:, n_kv * hd:] == 5).all()
    # whole sequences, among them positions stored above
    whole = np.concatenate([[0], np.cumsum(lens)])
    got = load(ctx, pool, seqs, whole, whole[-1])
    for g, w in zip(got, want):
        w = np.concatenate([w[table[s]].reshape(-1, n_kv, hd)[:ln] for s, ln in enumerate(lens)])
        assert np.array_equal(g.reshape(w.shape), w.astype(np.float32))


@pytest.mark.parametrize("bits", [4, 8])
def test_store_rounds_to_the_nearest_code(ctx, bits):
    """Every code's value, every middle between two codes and its fp32 neighbours, at scales from the least to the largest;
    blocks at the edge of a scale."""
    mags = au.E2M1 if bits == 4 else au.E4M3
    mid = ((mags[1:] + mags[:-1]) / 2).astype(np.float32)
    edge = np.float32(7.0 if bits == 4 else 464.0)
    one = np.concatenate([mags, mid, np.nextafter(mid, np.float32(0)), np.nextafter(mid, np.float32(1e9))]).astype(np.float32)
    one = one[one <= edge]
    out = []
    for top in (edge, mags[-1], np.nextafter(edge / 2, np.float32(1e9))):
        for part in np.array_split(one[one <= top], -(-len(one) // 31)):
            b = np.zeros(32, np.float32)
            b[: len(part)], b[31] = part, top
            out += [b, -b]
    base = np.stack(out)
    x = np.concatenate([base * np.float32(2.0) ** e for e in (-126, -125, -60, 0, 50, 118)])
    tiny = np.float32(2.0) ** np.arange(-149, -117, dtype=np.float32)  # among them fp32's smallest
    x = np.concatenate([x, tiny[None], -tiny[None], np.zeros((1, 32), np.float32), np.full((1, 32), 3.4e38, np.float32)])
    x = np.concatenate([x, np.zeros((-len(x) % 2, 32), np.float32)]).astype(np.float32)
    n = len(x) // 2
    k = x.reshape(n, 1, 64)
    pool = Pool(1, -(-n // 32) * 32, 1, 64, bits, bits)
    seqs = pool.seqs([[0]], [n])
    store(ctx, pool, seqs, [0, n], k, k)
    want = au.kv_quantize(k.astype(np.float64), bits)[0]
    for got in pool.values():
        assert np.array_equal(got[0, :n], want)
    with np.errstate(over="ignore"):  # 3.4e38 rounds to 2^128 in 4 bits
        want = want.astype(np.float32)
    for got in load(ctx, pool, seqs, [0, n], n):
        assert np.array_equal(got.reshape(want.shape), want)


@pytest.mark.parametrize("bits", [4, 8])
def test_store_values_that_are_not_finite(ctx, bits):
    rng = np.random.default_rng(3)
    k = rows(rng, 40, 2, 128)
    k[3, 0, 7], k[5, 1, 64], k[39, 1, 127] = np.nan, np.inf, -np.inf
    pool = Pool(2, 64, 2, 128, bits, bits)
    seqs = pool.seqs([[1]], [40])
    store(ctx, pool, seqs, [0, 40], k, k)
    want = au.kv_quantize(k.astype(np.float64), bits)[0]
    assert np.isnan(want).sum() == 96
    for got in load(ctx, pool, seqs, [0, 40], 40):
        assert np.array_equal(got.reshape(want.shape), want.astype(np.float32), equal_nan=True)


def test_one_row_a_sequence_and_missing_pages(ctx):
    """A batch's new tokens; a sequence of no length, one behind its table, one on a page that does not exist."""
    rng = np.random.default_rng(4)
    n_kv, hd = 2, 64
    pool = Pool(6, 32, n_kv, hd, 4, 4, fill=0x11)
    table = np.array([[0, 1], [2, -1], [3, 77], [4, 5], [1, 5]], np.int32)
    lens = [33, 40, 64, 0, 65]
    seqs = pool.seqs(table, lens)
    k, v = rows(rng, 5, n_kv, hd), rows(rng, 5, n_kv, hd)
    want = pool.values()
    store(ctx, pool, seqs, None, k, v)
    want[0][1, 0], want[1][1, 0] = au.kv_quantize(k[0], 4)[0], au.kv_quantize(v[0], 4)[0]
    for got, w in zip(pool.values(), want):
        assert np.array_equal(got, w)
    got = load(ctx, pool, seqs, None, 5)
    for g, src in zip(got, (k, v)):
        assert np.array_equal(g[0].reshape(n_kv, hd), au.kv_quantize(src[0], 4)[0].astype(np.float32))
        assert (g[1:] == 5).all()


def test_many_sequences_and_empty_ones(ctx):
    """More sequences than threads of a workgroup, most without new rows."""
    rng = np.random.default_rng(5)
    n_seq, n_kv, hd = 700, 1, 64
    new = (rng.random(n_seq) < 0.2).astype(int) * rng.integers(1, 4, n_seq)
    new[-1] = 3
    lens = new + rng.integers(0, 20, n_seq)
    off = np.concatenate([[0], np.cumsum(new)])
    table = rng.permutation(n_seq).astype(np.int32)[:, None]
    pool = Pool(n_seq, 32, n_kv, hd, 8, 4)
    seqs = pool.seqs(table, lens)
    k, v = rows(rng, off[-1], n_kv, hd), rows(rng, off[-1], n_kv, hd)
    store(ctx, pool, seqs, off, k, v)
    gk, gv = load(ctx, pool, seqs, off, off[-1])
    assert np.array_equal(gk.reshape(k.shape), au.kv_quantize(k, 8)[0].astype(np.float32))
    assert np.array_equal(gv.reshape(v.shape), au.kv_quantize(v, 4)[0].astype(np.float32))
    vals = pool.values()[0]
    for s in (0, 255, 256, 699):
        for i in range(new[s]):
            assert np.array_equal(vals[table[s, 0], lens[s] - new[s] + i], au.kv_quantize(k[off[s] + i], 8)[0])


def attend(ctx, seed, lens, n_head, n_kv, hd, kt, vt, page_len, window=0, max_len=None, qscale=1.0, scale=0.0, pad=0, table_more=0,
           nan_behind=True):
    """One call against the 64-bit form; the places behind each length hold NaN scales."""
    import torch
    rng = np.random.default_rng(seed)
    n_seq = len(lens)
    per = max(1, -(-max(lens) // page_len)) + table_more
    n_pages = n_seq * per + 2
    k = rows(rng, n_pages * page_len, n_kv, hd).reshape(n_pages, page_len, n_kv, hd)
    v = rows(rng, n_pages * page_len, n_kv, hd).reshape(n_pages, page_len, n_kv, hd)
    k /= np.abs(k).max((0, 1, 2)) / 3  # scores of the size that attention has
    table = table_of(rng, n_seq, per, n_pages)
    if nan_behind:
        for s, ln in enumerate(lens):
            for pos in range(ln, per * page_len):
                k[table[s, pos // page_len], pos % page_len, :, 3] = np.nan
                v[table[s, pos // page_len], pos % page_len, :, ::32] = np.nan
    pool = Pool(n_pages, page_len, n_kv, hd, kt, vt, data=au.kv_pack(k, v, n_kv, page_len, kt, vt))
    seqs = pool.seqs(table, lens, max_len)
    q = (rng.standard_normal((n_seq, n_head * hd + pad)) * qscale).astype(np.float32)
    dq = t(q)
    out = torch.full((n_seq, n_head * hd + pad), 5.0, device="cuda")
    ctx.check(ctx.lib.ggq_attention_kv_dev(ctx.h, pool.desc, seqs, ptr(dq), n_head * hd + pad, n_head, scale, window, ptr(out),
                                           n_head * hd + pad, stream_handle()), "cache attention")
    got = host(out)
    assert (got[:, n_head * hd:] == 5).all()
    K, V = pool.values()
    for s, ln in enumerate(lens):
        n = min(ln, max_len) if max_len is not None else ln
        kk, vv = (x[table[s]].reshape(-1, n_kv, hd)[:n] for x in (K, V))
        want, tol = au.attention(q[s:s + 1, : n_head * hd].reshape(1, n_head, hd), kk, vv, ln - 1, window, scale or None)
        au.check(got[s, : n_head * hd].reshape(1, n_head, hd), want, tol)
    return got


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("kt,vt", [(4, 4), (8, 4), (4, 8), (8, 8)])
@pytest.mark.parametrize("n_head,n_kv", [(8, 2), (6, 1)])
def test_attention_formats_and_heads(ctx, hd, kt, vt, n_head, n_kv):
    attend(ctx, hd + kt + vt, [1, 31, 33, 200, 0], n_head, n_kv, hd, kt, vt, 64)


@pytest.mark.parametrize("n_head,n_kv", [(1, 1), (3, 1), (4, 4), (10, 2), (7, 1), (16, 2), (9, 1), (16, 1), (24, 1), (14, 2)])
def test_attention_head_ratios(ctx, n_head, n_kv):
    attend(ctx, n_head, [70, 5], n_head, n_kv, 64, 4, 4, 32)


@pytest.mark.parametrize("lens,page_len,table_more", [
    ([1], 32, 0), ([32], 32, 0), ([4097], 32, 0), ([5000], 5024, 0), ([2047, 1, 0, 900], 96, 1),
    ([20000], 256, 2), ([3000] * 3 + [17], 3008, 0)])
def test_attention_lengths(ctx, lens, page_len, table_more):
    attend(ctx, sum(lens), lens, 8, 2, 64, 4, 4, page_len, table_more=table_more)


@pytest.mark.parametrize("window", [1, 31, 32, 33, 500, 5000])
def test_attention_window(ctx, window):
    attend(ctx, window, [1, 32, 33, 2100, 0], 8, 2, 128, 8, 4, 64, window=window)


def test_attention_max_len_bounds_what_is_read(ctx):
    """Lengths above max_len: the row stays where it is, positions from max_len on are not seen."""
    attend(ctx, 1, [100, 300], 4, 2, 64, 4, 4, 64, max_len=120, nan_behind=False)
    attend(ctx, 2, [100, 300], 4, 2, 64, 4, 4, 64, max_len=120, window=200, nan_behind=False)


def test_attention_peaked_scores_strides_scale(ctx):
    attend(ctx, 3, [700, 64], 8, 2, 64, 8, 8, 64, qscale=30.0)
    attend(ctx, 4, [700, 64], 8, 2, 128, 4, 4, 64, qscale=1e-3, scale=2.0, pad=12)
    attend(ctx, 5, [300], 8, 2, 64, 4, 8, 64, scale=-0.3)


def test_attention_nan_in_the_cache_is_seen(ctx):
    """A NaN block of a visible position reaches its kv head's rows, and those only."""
    import torch
    rng = np.random.default_rng(8)
    k, v = rows(rng, 64, 2, 64), rows(rng, 64, 2, 64)
    v[10, 1, 40] = np.nan
    pool = Pool(1, 64, 2, 64, 4, 4)
    seqs = pool.seqs([[0]], [40])
    store(ctx, pool, seqs, [0, 40], k[:40], v[:40])
    q = t(rng.standard_normal((1, 4, 64)).astype(np.float32))
    out = torch.empty((1, 4, 64), device="cuda")
    ctx.check(ctx.lib.ggq_attention_kv_dev(ctx.h, pool.desc, seqs, ptr(q), 256, 4, 0.0, 0, ptr(out), 256, stream_handle()), "a")
    bad = np.isnan(host(out))[0]
    assert not bad[:2].any() and bad[2:, 32:].all() and not bad[2:, :32].any()


def test_attention_pages_that_do_not_exist(ctx):
    """Positions of such pages are passed over; a sequence of nothing else gives zeros."""
    import torch
    rng = np.random.default_rng(9)
    k, v = rows(rng, 128, 1, 64).reshape(4, 32, 1, 64), rows(rng, 128, 1, 64).reshape(4, 32, 1, 64)
    pool = Pool(4, 32, 1, 64, 4, 4, data=au.kv_pack(k, v, 1, 32, 4, 4))
    table = np.array([[2, -5, 1], [-1, 4, 1 << 30]], np.int32)
    seqs = pool.seqs(table, [90, 96])
    q = rng.standard_normal((2, 4, 64)).astype(np.float32)
    dq = t(q)
    out = torch.full((2, 4, 64), 5.0, device="cuda")
    ctx.check(ctx.lib.ggq_attention_kv_dev(ctx.h, pool.desc, seqs, ptr(dq), 256, 4, 0.0, 0, ptr(out), 256, stream_handle()), "a")
    K, V = pool.values()
    kk, vv = (np.concatenate([x[2], x[1][:26]]) for x in (K, V))
    want, tol = au.attention(q[:1], kk, vv, 57)
    got = host(out)
    au.check(got[:1], want, tol)
    assert (got[1] == 0).all()


def test_attention_is_repeatable_and_splits_do_not_overlap(ctx):
    a = attend(ctx, 11, [9001, 8000], 8, 2, 128, 4, 4, 256)
    b = attend(ctx, 11, [9001, 8000], 8, 2, 128, 4, 4, 256)
    assert np.array_equal(a, b)


@pytest.mark.parametrize("splits", ["1", "2", "7", "100000"])
def test_attention_split_counts(ctx, monkeypatch, splits):
    """Any number of parts (GGQ_KV_SPLITS, read at every call), empty ones among them, gives the same result."""
    monkeypatch.setenv("GGQ_KV_SPLITS", splits)
    attend(ctx, 21, [1500, 40, 0, 700], 8, 2, 64, 4, 8, 96)
    attend(ctx, 22, [900, 33], 12, 2, 128, 8, 4, 64, window=300)


def test_no_sequences(ctx):
    pool = Pool(1, 32, 1, 64, 4, 4)
    seqs = gl.KvSeqs(0, 1, 0, None, None)
    lib = ctx.lib
    assert lib.ggq_attention_kv_dev(ctx.h, pool.desc, seqs, None, 64, 1, 0.0, 0, None, 64, None) == gl.Status.OK
    assert lib.ggq_kv_store_dev(ctx.h, pool.desc, seqs, None, 3, None, 64, None, 64, 0, None) == gl.Status.OK


def test_refusals(ctx):
    import torch
    lib = ctx.lib
    mem = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")
    tab, ln = t(np.zeros((1, 1), np.int32)), t(np.ones(1, np.int32))
    x = torch.zeros(4096, device="cuda")

    def cache(**kw):
        d = dict(pages=mem.data_ptr(), n_pages=1, page_len=32, n_kv_head=2, head_dim=64, k_type=4, v_type=8)
        d.update(kw)
        return gl.KvCache(**d)

    def seqs(**kw):
        d = dict(n_seq=1, table_len=1, max_len=32, pages=tab.data_ptr(), len=ln.data_ptr())
        d.update(kw)
        return gl.KvSeqs(**d)

    def st(c=None, s=None, n=1, k=None, ldk=128, v=None, ldv=128, ty=0, fn=lib.ggq_kv_store_dev):
        return fn(ctx.h, c or cache(), s or seqs(), None, n, x.data_ptr() if k is None else k, ldk,
                  x.data_ptr() if v is None else v, ldv, ty, stream_handle())

    def at(c=None, s=None, q=None, ldq=256, n_head=4, scale=0.0, window=0, out=None, ldo=256):
        return lib.ggq_attention_kv_dev(ctx.h, c or cache(), s or seqs(), x.data_ptr() if q is None else q, ldq, n_head, scale, window,
                                        x.data_ptr() + 8192 if out is None else out, ldo, stream_handle())
    bad = gl.Status.INVALID_PARAM
    assert st() == gl.Status.OK and at() == gl.Status.OK and st(fn=lib.ggq_kv_load_dev, k=x.data_ptr() + 4096) == gl.Status.OK
    for kw in (dict(pages=None), dict(pages=mem.data_ptr() + 8), dict(n_pages=0), dict(page_len=48), dict(page_len=0),
               dict(n_kv_head=0), dict(head_dim=96), dict(head_dim=512), dict(k_type=5), dict(v_type=0)):
        assert st(c=cache(**kw)) == bad and at(c=cache(**kw)) == bad, kw
        assert not kw.keys() & {"page_len", "n_kv_head", "head_dim", "k_type", "v_type"} or \
            lib.ggq_kv_page_bytes(ctypes.byref(cache(**kw))) == 0
    for kw in (dict(n_seq=-1), dict(n_seq=65536), dict(table_len=0), dict(table_len=1 << 27), dict(max_len=-1), dict(pages=None),
               dict(len=None)):
        assert st(s=seqs(**kw)) == bad and at(s=seqs(**kw)) == bad, kw
    for kw in (dict(n=-1), dict(k=0), dict(v=0), dict(k=x.data_ptr() + 4), dict(ldk=127), dict(ldv=64), dict(ldk=130),
               dict(ty=1, ldv=132), dict(ty=8)):
        assert st(**kw) == bad, kw
        assert st(fn=lib.ggq_kv_load_dev, **kw) == bad, kw
    for kw in (dict(q=0), dict(out=0), dict(q=x.data_ptr() + 4), dict(ldq=255), dict(ldq=258), dict(ldo=200), dict(n_head=3),
               dict(n_head=0), dict(scale=float("nan")), dict(scale=float("inf")), dict(window=-1)):
        assert at(**kw) == bad, kw
    assert lib.ggq_kv_store_dev(ctx.h, None, seqs(), None, 1, ptr(x), 128, ptr(x), 128, 0, None) == bad
    assert lib.ggq_attention_kv_dev(ctx.h, cache(), None, ptr(x), 256, 4, 0.0, 0, ptr(x), 256, None) == bad
    assert st(n=0) == gl.Status.OK
