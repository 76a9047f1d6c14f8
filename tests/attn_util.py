"""Plain 64-bit forms of the attention operators around the KV cache, from the definitions in include/ggq.h, and
error bounds for their tests."""
import numpy as np

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
# e4m3: code c < 127 has exponent c >> 3 (0: subnormal) and three bits of mantissa
E4M3 = np.array([(c & 7) * 2.0 ** -9 if c < 8 else (8 + (c & 7)) * 2.0 ** ((c >> 3) - 10) for c in range(127)])
U32 = 2.0 ** -24  # half a step of fp32, relative


def kv_quantize(x, bits):
    """(values, codes without zeros' signs, scale bytes) of x [..., head_dim], blocks of 32."""
    mags, edge = (E2M1, 7.0) if bits == 4 else (E4M3, 464.0)
    b = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, 32)
    bad = ~np.isfinite(b).all(-1)
    top = np.where(np.isfinite(b), np.abs(b), 0).max(-1)
    e = np.full(top.shape, 999)
    with np.errstate(divide="ignore"):
        g = np.where(top > 0, np.floor(np.log2(np.maximum(top, 1e-300) / edge)), -200.0).astype(int)
    for d in (-1, 0, 1):  # the smallest exponent that holds the block, around the logarithm's
        ok = top <= edge * np.exp2((g + d).astype(float))
        e = np.where(ok & (e == 999), g + d, e)
    e = np.maximum(e, -126)
    assert (e < 999).all()
    y = np.abs(np.where(bad[..., None], 0, b)) * np.exp2(-e[..., None].astype(float))
    mid = (mags[1:] + mags[:-1]) / 2
    lo, hi = np.searchsorted(mid, y, side="left"), np.searchsorted(mid, y, side="right")
    i = np.where((hi != lo) & (lo % 2 == 1), hi, lo)  # a tie: the even one of lo and lo + 1
    v = np.where(b < 0, -1, 1) * mags[i] * np.exp2(e[..., None].astype(float))
    v = np.where(bad[..., None], np.nan, v)
    codes = i + np.where((b < 0) & (i > 0), 8 if bits == 4 else 128, 0)
    codes = np.where(bad[..., None], 0, codes)
    return v.reshape(x.shape), codes.reshape(x.shape).astype(np.uint8), np.where(bad, 255, e + 127).astype(np.uint8)


def kv_record(hd, kt, vt):
    k, v = 32 * hd * kt // 8, 32 * hd * vt // 8
    return k, k + v, k + v + hd, k + v + 2 * hd  # V codes, K scales, V scales, end


def kv_places(hd, bits, value):
    """Byte and half of position p, value d; byte of the scale of position p, block c."""
    p, d = np.mgrid[0:32, 0:hd]
    if value:
        lane, n = 16 * (p % 16 // 4) + d // (hd // 16), (4 * (p // 16) + p % 4) * (hd // 16) + d % (hd // 16)
    else:
        lane, n = 16 * (d // (hd // 4)) + p % 16, (p // 16) * (hd // 4) + d % (hd // 4)
    b = n * bits // 8
    p, c = np.mgrid[0:32, 0:hd // 32]
    sc = (4 * c + p % 16 // 4) * 8 + 4 * (p // 16) + p % 4 if value else (16 * c + p % 16) * 2 + p // 16
    return 1024 * (b // 16) + 16 * lane + b % 16, n % 2, sc


def kv_values(codes, scales, bits):
    mag = np.concatenate([E2M1, -E2M1]) if bits == 4 else np.concatenate([E4M3, [np.nan], -E4M3, [np.nan]])
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(float) - 127))
    return mag[codes] * np.repeat(s, 32, axis=-1)


def kv_unpack(pages, n_kv, page_len, hd, kt, vt):
    """fp64 K and V [n_pages][page_len][n_kv][hd] of a pool of pages (bytes)."""
    v0, ks, vs, end = kv_record(hd, kt, vt)
    rec = pages.reshape(len(pages), n_kv, page_len // 32, end)
    out = []
    for bits, value, at, sc in ((kt, False, 0, ks), (vt, True, v0, vs)):
        byte, half, scale = kv_places(hd, bits, value)
        codes = rec[..., at + byte]
        if bits == 4:
            codes = np.where(half == 1, codes >> 4, codes & 15)
        x = kv_values(codes, rec[..., sc + scale], bits)
        out.append(x.reshape(len(pages), n_kv, page_len, hd).transpose(0, 2, 1, 3))
    return out


def kv_pack(k, v, n_kv, page_len, kt, vt):
    """Pool bytes of K and V [n_pages][page_len][n_kv][hd]."""
    n_pages, hd = k.shape[0], k.shape[-1]
    v0, ks, vs, end = kv_record(hd, kt, vt)
    rec = np.zeros((n_pages, n_kv, page_len // 32, end), np.uint8)
    for x, bits, value, at, sc in ((k, kt, False, 0, ks), (v, vt, True, v0, vs)):
        _, codes, scales = kv_quantize(x, bits)
        byte, half, scale = kv_places(hd, bits, value)
        codes = codes.transpose(0, 2, 1, 3).reshape(n_pages, n_kv, -1, 32, hd)
        scales = scales.transpose(0, 2, 1, 3).reshape(n_pages, n_kv, -1, 32, hd // 32)
        if bits == 4:
            for h in (0, 1):
                w = half == h
                rec[..., (at + byte)[w]] |= codes[..., w] << (4 * h)
        else:
            rec[..., at + byte] = codes
        rec[..., sc + scale] = scales
    return rec.reshape(n_pages, -1)


def attention(q, k, v, first, window=0, scale=None):
    """fp64 attention of rows q [rows][heads][hd] over k, v [positions][kv heads][hd], row i at position first + i,
    and the bound of an fp32 kernel's error of each value.

    The bound: scores are sums of hd fp32 products, off by (hd / 4 + 8) roundings of the sum of their magnitudes at
    most (four products a step of a lane's chain, the matrix cores' steps take more at once); the relative error of a weight
    is that of the exponent, numerator and denominator each; the sum over positions adds a rounding a step of 16 positions and those
    of the splits, relative to the sum of magnitudes."""
    rows, heads, hd = q.shape
    scale = hd ** -0.5 if scale is None else scale
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    out, tol = np.zeros((rows, heads, hd)), np.zeros((rows, heads, hd))
    G = heads // k.shape[1]
    for i in range(rows):
        e = min(first + i + 1, len(k))
        b = max(0, first + i + 1 - window) if window else 0
        if e <= b:
            continue
        for h in range(heads):
            kk, vv = k[b:e, h // G], v[b:e, h // G]
            s = kk @ q[i, h] * scale
            with np.errstate(invalid="ignore"):
                p = np.exp(s - s.max())
                p /= p.sum()
                ds = U32 * (hd / 4 + 8) * (np.abs(kk) @ np.abs(q[i, h])).max() * abs(scale)
                out[i, h] = p @ vv
                tol[i, h] = (2 * ds + U32 * (32 + (e - b) / 16)) * (p @ np.abs(vv)) + 1e-37
    return out, tol


def check(got, want, tol):
    """Every value within its bound; NaN where NaN is wanted, and nowhere else."""
    got = np.asarray(got, np.float64)
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan), (np.argwhere(np.isnan(got) != nan)[:5], nan.sum())
    err = np.abs(np.where(nan, 0, got - want))
    bad = err > np.where(nan, 0, tol)
    assert not bad.any(), (np.argwhere(bad)[:5], err[bad][:5], np.asarray(tol)[bad][:5], int(bad.sum()))
