"""Plain 64-bit forms of the operators around a layer's matmuls (norms with int8 rows, sampling, the gated delta rule),
from the definitions in include/ggq.h, and error bounds for their tests."""
import numpy as np

U32 = 2.0 ** -24  # half a step of fp32, relative


# ------------------------------------------------------------------- norms

def norm(x, add=None, w=None, norm_len=0, eps=1e-6, gate=None):
    """(sum as fp32, y in 64 bits) of fp32 rows."""
    with np.errstate(all="ignore"):
        s = x if add is None else x + add  # one rounding
        h = s.astype(np.float64).reshape(len(s), -1, norm_len or s.shape[1])
        y = h / np.sqrt((h * h).mean(-1, keepdims=True) + np.float64(np.float32(eps)))
        if w is not None:
            y = y * w.astype(np.float64)
        y = y.reshape(s.shape)
        if gate is not None:
            z = gate.astype(np.float64)
            y = y * (z / (1 + np.exp(-z)))
    return s, y


def codes(y, block=0):
    """int8 codes and scales of fp32 rows, each step in fp32 (block 32, or 0: the row)."""
    b = y.reshape(len(y), -1, block or y.shape[1])
    top = np.abs(b).max(-1, keepdims=True)
    sc = np.where(top > 0, top / np.float32(127), np.float32(1)).astype(np.float32)
    q = np.clip(np.rint(b * (np.float32(1) / sc)), -128, 127)
    return q.reshape(y.shape).astype(np.int8), sc[..., 0]


# ---------------------------------------------------------------- sampling

BORDER = 2.0 ** -30  # how near to a border of the running sum u has to be before a token may be the next one


def sample(x, t=1.0, top_k=0, top_p=1.0, min_p=0.0, u=0.0):
    """(token, prob, distance of u to the nearest border, of the sum) of one row."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    if not (x > -np.inf).any():
        return 0, 0.0, 1.0
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    if not t > 0:
        return int(order[0]), 1.0, 1.0
    top = x[order[0]]
    with np.errstate(all="ignore"):
        # (a difference of infinities is none)
        w = np.exp(np.where(x[order] == top, 0.0, (x[order] - top) / np.float64(np.float32(t))))
    n = top_k if 0 < top_k < len(w) else len(w)
    if top_p < 1:
        want = max(0.0, float(np.float32(top_p))) * w[:n].sum()
        n = min(n, int(np.searchsorted(np.cumsum(w[:n]), want)) + 1)
    if min_p > 0:
        n = max(1, min(n, int((w >= min(1.0, float(np.float32(min_p)))).sum())))
    at = np.argsort(order[:n])
    ids, w = order[:n][at], w[:n][at]
    w = np.where(w < 2.0 ** -60, 0.0, w)
    c = np.cumsum(w)
    u = float(np.float32(u)) if u > 0 else 0.0
    j = int(np.searchsorted(c, u * c[-1], side="right"))
    j = min(j, int(np.flatnonzero(w)[-1]))
    near = np.abs(np.concatenate(([0.0], c)) / c[-1] - u)
    return int(ids[j]), w[j] / c[-1], near[near > 0].min(initial=1.0) if u else 1.0


# -------------------------------------------------------------- delta rule

def gates(gate, beta, rate=None, bias=None, sigmoid=False):
    g, b = gate.astype(np.float64), beta.astype(np.float64)
    if rate is not None:
        z = g + (0 if bias is None else bias.astype(np.float64))
        g = rate.astype(np.float64) * (np.maximum(z, 0) + np.log1p(np.exp(-np.abs(z))))
    if sigmoid:
        b = 1 / (1 + np.exp(-b))
    return g, b


def delta(q, k, v, g, b, state, qk_norm=False, eps=1e-6, scale=0.0):
    """One sequence: q, k [rows][k heads][kd], v [rows][v heads][vd], g, b [rows][v heads], state [v heads][vd][kd], all
    rows one by one.  Returns out, the state after it, and bounds of an fp32 kernel's error of both.

    The bounds.  With |b| <= 1 and normalised k (or shorter ones) the step S -> a (1 - b k k^T) S shrinks an error of a column of S, in the
    2-norm: errors add up, they do not grow.  A row adds to its u at most n roundings (n: the k_dim of the dot, the 16
    rows that may be solved together, three for each of them, and a few) of the magnitudes that it is made of, the 16 rows' among them (a triangular
    solve passes its rows' errors on, at most once more each through the magnitudes of the products between them), and to the
    state two roundings of its magnitude and the decay's relative error (4 roundings, and 8 of the decay's logarithm)."""
    q, k, v, S = (np.asarray(x, np.float64) for x in (q, k, v, state))
    rows, H, vd = v.shape
    kd, G = q.shape[2], H // q.shape[1]
    if qk_norm:
        q, k = (x / np.sqrt((x * x).sum(-1, keepdims=True) + np.float64(np.float32(eps))) for x in (q, k))
    q = q * (kd ** -0.5 if scale == 0 else scale)
    n = kd + 64
    out, tol = np.zeros((rows, H, vd)), np.zeros((rows, H, vd))
    S = S.copy()
    E = np.zeros((H, vd))  # of a column, in the 2-norm
    S_tol = np.zeros_like(S)
    for h in range(H):
        hist = []  # of the rows before in reach: |k|, |u| and its error
        for t in range(rows):
            kk, qq = k[t, h // G], q[t, h // G]
            a, bb = np.exp(g[t, h]), b[t, h]
            ea = U32 * (4 + 8 * abs(min(0.0, max(g[t, h], -200.0))))
            S[h] *= a
            ks = S[h] @ kk
            u = bb * (v[t, h] - ks)
            mags = np.abs(v[t, h]) + np.abs(S[h]) @ np.abs(kk)
            for ko, uo in hist[-16:]:
                mags = mags + (np.abs(kk) @ ko) * uo
            eu = U32 * n * abs(bb) * mags + abs(bb) * ea * np.abs(ks)
            S[h] += u[:, None] * kk
            nrm = np.linalg.norm(S[h], axis=1)
            E[h] = min(a, 1.0) * E[h] + np.linalg.norm(kk) * eu + (2 * U32 + ea) * (nrm + np.linalg.norm(kk) * np.abs(u)) + 6 * U32 * np.abs(u)
            out[t, h] = S[h] @ qq
            tol[t, h] = np.linalg.norm(qq) * E[h] + U32 * n * (np.abs(S[h]) @ np.abs(qq) + sum((np.abs(qq) @ ko) * uo for ko, uo in hist[-16:]))
            hist.append((np.abs(kk), np.abs(u)))
        S_tol[h] = E[h][:, None] + 4 * U32 * np.abs(S[h])
    return out, S, tol + 1e-37, S_tol + 1e-37
