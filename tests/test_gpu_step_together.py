"""The operators around the matmuls as a step of a model with linear and softmax attention layers uses them: norms and int8
rows, the delta rule, attention of new rows over the cache, sampling.  Stage by stage against 64 bits; prompts, proposed tokens
and single tokens in one call; captured and replayed; on several streams and threads at once; without workspace; far into large buffers."""
import ctypes
import os
import threading

import numpy as np
import pytest

import ggnpu_amd.lib as gl
from tests import attn_util as au
from tests import step_util as su
from tests.gpu_util import host, ptr
from tests.test_gpu_kv_chunk import row_of

pytestmark = pytest.mark.gpu
EPS, D, VOCAB = 1e-6, 256, 2048
KH, VH, KD, VD = 2, 4, 64, 32          # linear attention
NH, NKV, HD, PAGE = 4, 2, 64, 32       # softmax attention
WIDTH = 2 * KH * KD + 2 * VH * VD + 2 * VH  # q, k, v, z, gate, beta of a row


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


def q8_0(rng, n, k):
    """Random Q8_0 rows: blocks of a fp16 scale and 32 codes; and their values."""
    d = (rng.uniform(0.5, 1.5, (n, k // 32, 1)) / (64 * np.sqrt(k))).astype(np.float16)
    c = rng.integers(-127, 128, (n, k // 32, 32), dtype=np.int8)
    raw = np.concatenate([d.view(np.uint8).reshape(n, k // 32, 2), c.view(np.uint8)], -1)
    return t(raw.reshape(-1)), (d.astype(np.float64) * c).reshape(n, k)


class Step:
    """Two layers and the logits; every buffer is allocated once, so that calls can be captured.  Equal seeds, equal models."""

    def __init__(self, ctx, n_seq, per, rows, seed=0):
        import torch
        rng = np.random.default_rng(seed)
        self.ctx, self.n_seq, self.rows = ctx, n_seq, rows
        self.w = {n: q8_0(rng, *s) for n, s in dict(lin=(WIDTH, D), lin_out=(D, VH * VD), qkv=((NH + 2 * NKV) * HD, D), att_out=(D, NH * HD),
                                                    logits=(VOCAB, D)).items()}
        f = lambda *s: (1 + 0.1 * rng.standard_normal(s)).astype(np.float32)  # noqa: E731
        self.norm_w = {n: t(f(k)) for n, k in (("lin", D), ("heads", VD), ("att", D), ("logits", D))}
        self.rate, self.bias = t(-np.exp(rng.standard_normal(VH)).astype(np.float32)), t(f(VH))
        n_pages = n_seq * per + 1
        self.kv = (NKV, HD, 8, 4)
        size = gl.load_library().ggq_kv_page_bytes(ctypes.byref(gl.KvCache(None, 0, PAGE, *self.kv)))
        self.pool = torch.zeros((n_pages, size), dtype=torch.uint8, device="cuda")
        self.cache = gl.KvCache(self.pool.data_ptr(), n_pages, PAGE, *self.kv)
        self.table_np = rng.permutation(n_pages)[: n_seq * per].reshape(n_seq, per).astype(np.int32)
        self.slot_np = rng.permutation(n_seq + 2)[:n_seq].astype(np.int32)
        self.table, self.slot = t(self.table_np), t(self.slot_np)
        self.len, self.off = torch.zeros(n_seq, dtype=torch.int32, device="cuda"), torch.zeros(n_seq + 1, dtype=torch.int32, device="cuda")
        self.seqs = gl.KvSeqs(n_seq, per, per * PAGE, self.table.data_ptr(), self.len.data_ptr())
        self.state = t(rng.standard_normal((n_seq + 2, VH, VD, KD)).astype(np.float32))
        z = lambda *s, dt=torch.float32: torch.zeros(s, dtype=dt, device="cuda")  # noqa: E731
        self.b = dict(x=z(rows, D), p=z(rows, WIDTH), o=z(rows, VH * VD), y1=z(rows, D), s1=z(rows, D), qkv=z(rows, (NH + 2 * NKV) * HD),
                      att=z(rows, NH * HD), y2=z(rows, D), s2=z(rows, D), logits=z(rows, VOCAB), token=z(rows, dt=torch.int32), prob=z(rows))
        for n, k in (("c0", D), ("c1", VH * VD), ("c2", D), ("c3", NH * HD), ("c4", D)):
            self.b[n], self.b["s_" + n] = z(rows, k, dt=torch.int8), z(rows)
        self.temp, self.k, self.tp, self.mp, self.u = z(rows), z(rows, dt=torch.int32), z(rows), z(rows), z(rows)
        self.set_sampling(rng)

    def set_sampling(self, rng):
        n = self.rows
        self.temp.copy_(t(rng.choice([0, 0.7, 1, 1.5], n).astype(np.float32)))
        self.k.copy_(t(rng.choice([0, 1, 40], n).astype(np.int32)))
        self.tp.copy_(t(rng.choice([0.5, 0.95, 1], n).astype(np.float32)))
        self.mp.copy_(t(rng.choice([0, 0.05], n).astype(np.float32)))
        self.u.copy_(t(rng.random(n).astype(np.float32)))

    def matmul(self, w, codes, out, s):
        n, k = self.w[w][1].shape
        self.ctx.check(self.ctx.lib.ggq_mul_mat_q8_dev(self.ctx.h, ptr(self.w[w][0]), int(gl.GgmlType.Q8_0), n, k, ptr(self.b[codes]),
                                                       ptr(self.b["s_" + codes]), self.n, ptr(out), out.shape[1], s), "matmul")

    def norm(self, x, w, codes, s, add=None, sum=None, out=None, gate=None, norm_len=0):
        p = gl.NormParams(n_rows=self.n, n_cols=x.shape[1], x=x.data_ptr(), ldx=x.shape[1], norm_w=self.norm_w[w].data_ptr(), norm_len=norm_len,
                          eps=EPS, act_mode=gl.ActMode.Q8_ROW, codes=self.b[codes].data_ptr(), scales=self.b["s_" + codes].data_ptr())
        if add is not None:
            p.add, p.ld_add, p.sum, p.ld_sum = add.data_ptr(), add.shape[1], sum.data_ptr(), sum.shape[1]
        if gate is not None:
            p.gate, p.ld_gate = gate, WIDTH
        if out is not None:
            p.out, p.ldo = out.data_ptr(), out.shape[1]
        self.ctx.check(self.ctx.lib.ggq_norm_dev(self.ctx.h, p, s), "norm")

    def run(self, n, s):
        """The step on n rows (x, off, len set before)."""
        b, lib, h = self.b, self.ctx.lib, self.ctx.h
        self.n = n
        self.norm(b["x"], "lin", "c0", s)
        self.matmul("lin", "c0", b["p"], s)
        P, at = b["p"].data_ptr(), [4 * x for x in (0, KH * KD, 2 * KH * KD, 2 * KH * KD + VH * VD, 2 * KH * KD + 2 * VH * VD, WIDTH - VH)]
        p = gl.DeltaRuleParams(n_k_head=KH, n_v_head=VH, k_dim=KD, v_dim=VD, q=P, ldq=WIDTH, k=P + at[1], ldk=WIDTH, v=P + at[2], ldv=WIDTH,
                               gate=P + at[4], ld_gate=WIDTH, beta=P + at[5], ld_beta=WIDTH, gate_rate=self.rate.data_ptr(),
                               gate_bias=self.bias.data_ptr(), flags=gl.DELTA_BETA_SIGMOID | gl.DELTA_QK_NORM, eps=EPS, state=self.state.data_ptr(),
                               state_out=self.state.data_ptr(), n_slots=self.state.shape[0], slot=self.slot.data_ptr(), n_seq=self.n_seq,
                               n_rows=n, row_off=self.off.data_ptr(), out=b["o"].data_ptr(), ldo=VH * VD)
        self.ctx.check(lib.ggq_delta_rule_dev(h, p, s), "delta rule")
        self.norm(b["o"], "heads", "c1", s, gate=P + at[3], norm_len=VD)
        self.matmul("lin_out", "c1", b["y1"], s)
        self.norm(b["y1"], "att", "c2", s, add=b["x"], sum=b["s1"])
        self.matmul("qkv", "c2", b["qkv"], s)
        ld = (NH + 2 * NKV) * HD
        Q = b["qkv"].data_ptr()
        k, v = Q + 4 * NH * HD, Q + 4 * (NH + NKV) * HD
        self.ctx.check(lib.ggq_kv_store_dev(h, self.cache, self.seqs, ptr(self.off), n, k, ld, v, ld, 0, s), "store")
        self.ctx.check(lib.ggq_attention_kv_rows_dev(h, self.cache, self.seqs, ptr(self.off), n, Q, ld, NH, 0.0, 0, ptr(b["att"]), NH * HD, s), "attention")
        self.ctx.check(lib.ggq_quantize_act_dev(h, ptr(b["att"]), NH * HD, n, NH * HD, gl.ActMode.Q8_ROW, ptr(b["c3"]), ptr(b["s_c3"]), s), "quantize")
        self.matmul("att_out", "c3", b["y2"], s)
        self.norm(b["y2"], "logits", "c4", s, add=b["s1"], sum=b["s2"])
        self.matmul("logits", "c4", b["logits"], s)
        p = gl.SampleParams(n_rows=n, n_vocab=VOCAB, logits=b["logits"].data_ptr(), ld=VOCAB, temperature=self.temp.data_ptr(),
                            top_k=self.k.data_ptr(), top_p=self.tp.data_ptr(), min_p=self.mp.data_ptr(), u=self.u.data_ptr(),
                            token=b["token"].data_ptr(), prob=b["prob"].data_ptr())
        self.ctx.check(lib.ggq_sample_dev(h, p, s), "sample")

    def begin(self, x, rows, lens):
        """Rows of each sequence and the lengths with them."""
        n = sum(rows)
        self.b["x"][:n].copy_(x[:n])
        self.off.copy_(t(np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)))
        self.len.copy_(t(np.asarray(lens, np.int32)))
        return n

    def values(self):
        return {n: host(x) for n, x in self.b.items()}

    def same(self, other, n):
        a, b = self.values(), other.values()
        assert np.array_equal(host(self.state), host(other.state)) and np.array_equal(host(self.pool), host(other.pool))
        for x in ("o", "att", "logits", "token", "prob"):
            assert np.array_equal(a[x][:n], b[x][:n]), x


def stream():
    import torch
    return torch.cuda.current_stream().cuda_stream


def matmul_check(got, codes, scales, w):
    # int8 products of a block are exact, the blocks' sums in fp32: three roundings a block and what a split adds
    want = (codes.astype(np.float64) @ w.T) * scales[:, None]
    mag = (np.abs(codes).astype(np.float64) @ np.abs(w).T) * scales[:, None]
    au.check(got, want, su.U32 * (3 + w.shape[1] / 32 + 16) * mag)


def check_stages(st, n, rows, lens, state, x):
    """Every stage against 64 bits on the stage's own inputs."""
    b = {k: v[:n] for k, v in st.values().items()}
    off = np.concatenate([[0], np.cumsum(rows)])
    W = {k: host(v) for k, v in st.norm_w.items()}

    def norm_check(codes, y, out=None):
        q, sc = su.codes(y.astype(np.float32))
        # y rounded once may fall on the other side of a border only where 64 bits' sums differ: not at all but for the last bit
        au.check(b["s_" + codes], sc[:, 0], 2 * su.U32 * sc[:, 0])
        d = np.abs(b[codes].astype(int) - q)
        assert d.max() <= 1 and (d > 0).mean() < 1e-3
    norm_check("c0", su.norm(x, w=W["lin"], eps=EPS)[1])
    matmul_check(b["p"], b["c0"], b["s_c0"], st.w["lin"][1])
    p = b["p"]
    cut = np.cumsum([0, KH * KD, KH * KD, VH * VD, VH * VD, VH, VH])
    q, k, v, z, gate, beta = (p[:, a:e] for a, e in zip(cut[:-1], cut[1:]))
    g, be = su.gates(gate, beta, host(st.rate), host(st.bias), True)
    for s in range(st.n_seq):
        r = slice(off[s], off[s + 1])
        m = rows[s]
        out, S, tol, S_tol = su.delta(q[r].reshape(m, KH, KD), k[r].reshape(m, KH, KD), v[r].reshape(m, VH, VD), g[r], be[r],
                                      state[st.slot_np[s]], True, EPS)
        au.check(b["o"][r].reshape(m, VH, VD), out, tol)
        au.check(host(st.state)[st.slot_np[s]], S, S_tol)
    norm_check("c1", su.norm(b["o"], w=W["heads"], norm_len=VD, eps=EPS, gate=z)[1])
    matmul_check(b["y1"], b["c1"], b["s_c1"], st.w["lin_out"][1])
    s1, y = su.norm(b["y1"], add=x, w=W["att"], eps=EPS)
    assert np.array_equal(s1, b["s1"])
    norm_check("c2", y)
    matmul_check(b["qkv"], b["c2"], b["s_c2"], st.w["qkv"][1])
    Q, K, V = (b["qkv"][:, a:e].reshape(n, -1, HD) for a, e in ((0, NH * HD), (NH * HD, (NH + NKV) * HD), ((NH + NKV) * HD, None)))
    ck, cv = au.kv_unpack(host(st.pool), NKV, PAGE, HD, 8, 4)
    for s in range(st.n_seq):
        kk, vv = (c[st.table_np[s]].reshape(-1, NKV, HD) for c in (ck, cv))
        r = slice(off[s], off[s + 1])
        first = lens[s] - rows[s]
        if not rows[s]:
            continue
        assert np.array_equal(kk[first:lens[s]], au.kv_quantize(K[r], 8)[0]) and np.array_equal(vv[first:lens[s]], au.kv_quantize(V[r], 4)[0])
        for i in range(rows[s]):
            want, tol = row_of(Q[r][i:i + 1], kk[: first + i + 1], vv[: first + i + 1], None, True)
            au.check(b["att"][r][i:i + 1].reshape(1, NH, HD), want, tol)
    matmul_check(b["y2"], b["c3"], b["s_c3"], st.w["att_out"][1])
    s2, y = su.norm(b["y2"], add=b["s1"], w=W["logits"], eps=EPS)
    assert np.array_equal(s2, b["s2"])
    norm_check("c4", y)
    matmul_check(b["logits"], b["c4"], b["s_c4"], st.w["logits"][1])
    T, K_, TP, MP, U = (host(a) for a in (st.temp, st.k, st.tp, st.mp, st.u))
    for r in range(n):
        tok, prob, near = su.sample(b["logits"][r], T[r], K_[r], TP[r], MP[r], U[r])
        if near > su.BORDER:
            assert b["token"][r] == tok and abs(b["prob"][r] - prob) <= 2.0 ** -22 * prob + 1e-37, r


def draw(n, seed):
    return np.random.default_rng(seed).standard_normal((n, D)).astype(np.float32)


def test_prompts_proposals_and_tokens(ctx):
    """Prompts, then a prompt's next part with single tokens and proposed tokens in one call, then single tokens."""
    st = Step(ctx, 4, 6, 96)
    lens = [0] * 4
    for i, rows in enumerate(([50, 7, 17, 1], [33, 1, 5, 1], [1, 1, 1, 1], [0, 4, 0, 60], [1, 1, 1, 1])):
        lens = [a + b for a, b in zip(lens, rows)]
        x, state = draw(sum(rows), i), host(st.state).copy()
        n = st.begin(t(x), rows, lens)
        st.run(n, stream())
        check_stages(st, n, rows, lens, state, x)


def test_captured_steps(ctx):
    """Steps of single tokens and of proposed ones, captured once and replayed as the sequences grow; eager steps of an equal model
    between the replays give the same bits."""
    import torch
    a, b = Step(ctx, 3, 8, 16, seed=3), Step(ctx, 3, 8, 16, seed=3)
    lens = np.zeros(3, int)
    rows = [5, 9, 2]
    lens += rows
    x = t(draw(16, 1))
    for m in (a, b):
        m.run(m.begin(x, rows, lens), stream())
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    graphs = {}
    for n in (3, 12):
        graphs[n] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graphs[n], stream=s):
            a.run(n, s.cuda_stream)
    for i, rows in enumerate(([1, 1, 1], [4, 4, 4], [1, 1, 1], [10, 1, 1], [0, 2, 10], [1, 1, 1], [4, 4, 4])):
        lens = lens + rows
        x = t(draw(16, 10 + i))
        for m in (a, b):
            n = m.begin(x, rows, lens)
        torch.cuda.synchronize()
        graphs[n].replay()
        b.run(n, stream())
        torch.cuda.synchronize()
        a.same(b, n)


def test_two_graphs_and_eager_steps_in_flight_together(ctx):
    """Two captured steps and two eager ones, each on a stream of its own and all at once, one context."""
    import torch
    rows, lens = [70, 3, 20], [70, 3, 20]
    ref = [Step(ctx, 3, 8, 96, seed=20 + i) for i in range(4)]
    own = [Step(ctx, 3, 8, 96, seed=20 + i) for i in range(4)]
    xs = [t(draw(96, 30 + i)) for i in range(4)]
    for r, x in zip(ref, xs):
        r.run(r.begin(x, rows, lens), stream())
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for i, g in enumerate(graphs):
        n = own[i].begin(xs[i], rows, lens)
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=streams[i]):
            own[i].run(n, streams[i].cuda_stream)
    start = [r.state.clone() for r in (Step(ctx, 3, 8, 96, seed=20 + i) for i in range(4))]
    for _ in range(3):
        for m, x, z in zip(own, xs, start):
            m.state.copy_(z)
            m.begin(x, rows, lens)
        torch.cuda.synchronize()
        for i in range(4):
            if i < 2:
                with torch.cuda.stream(streams[i]):
                    graphs[i].replay()
            else:
                own[i].run(93, streams[i].cuda_stream)
        torch.cuda.synchronize()
        for m, r in zip(own, ref):
            m.same(r, 93)


def test_threads(ctx):
    """Steps by four threads on one context, each on its stream."""
    import torch
    rows, lens = [40, 1, 12], [40, 1, 12]
    ref, own = ([Step(ctx, 3, 4, 64, seed=40 + i) for i in range(4)] for _ in range(2))
    xs = [t(draw(64, 50 + i)) for i in range(4)]
    for r, x in zip(ref, xs):
        n = r.begin(x, rows, lens)
        r.run(n, stream())
        r.begin(x, [1, 1, 1], [41, 2, 13])
        r.run(3, stream())
    for m, x in zip(own, xs):
        m.begin(x, rows, lens)
    offs = [(t(np.array([0, 1, 2, 3], np.int32)), t(np.array([41, 2, 13], np.int32))) for _ in own]
    torch.cuda.synchronize()
    errors = []

    def work(m, o):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                m.run(53, s.cuda_stream)
                m.off.copy_(o[0])
                m.len.copy_(o[1])
                m.run(3, s.cuda_stream)
            s.synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)
    th = [threading.Thread(target=work, args=a) for a in zip(own, offs)]
    for x in th:
        x.start()
    for x in th:
        x.join()
    assert not errors
    for m, r in zip(own, ref):
        m.same(r, 3)


def test_capture_without_workspace():
    """Nothing set aside for captures: the delta rule goes row by row, attention in one part, and only sampling needs memory."""
    import torch
    c = gl.Context(0)
    try:
        st = Step(c, 1, 40, 700)
        rng = np.random.default_rng(4)
        q = t(rng.standard_normal((600, NH, HD)).astype(np.float32))
        k, v = (t(rng.standard_normal((1200, NKV, HD)).astype(np.float32)) for _ in range(2))
        st.begin(st.b["x"], [600], [1200])
        off, all_ = t(np.array([0, 600], np.int32)), t(np.array([0, 1200], np.int32))
        c.check(c.lib.ggq_kv_store_dev(c.h, st.cache, st.seqs, ptr(all_), 1200, ptr(k), NKV * HD, ptr(v), NKV * HD, 0, stream()), "store")
        out = torch.empty_like(q)
        torch.cuda.synchronize()
        s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            c.check(c.lib.ggq_attention_kv_rows_dev(c.h, st.cache, st.seqs, ptr(off), 600, ptr(q), NH * HD, NH, 0.0, 0, ptr(out), NH * HD,
                                                    s.cuda_stream), "attention")
        ck, cv = au.kv_unpack(host(st.pool), NKV, PAGE, HD, 8, 4)
        kk, vv = (x[st.table_np[0]].reshape(-1, NKV, HD) for x in (ck, cv))
        for _ in range(3):
            out.fill_(7.0)
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            O, Q = host(out), host(q)
            for i in (0, 1, 63, 64, 300, 599):
                au.check(O[i:i + 1], *row_of(Q[i:i + 1], kk[:601 + i], vv[:601 + i], None, True))
    finally:
        c.close()


def test_rows_and_states_beyond_four_gigabytes(ctx):
    """Rows with strides, and slots, whose byte offsets do not fit 32 bits."""
    import torch
    big = torch.empty(5 << 28, device="cuda")  # 5 GiB
    rng = np.random.default_rng(6)
    # the delta rule: slot 1 of a pool of 2^21 states of 2 KB less those before 4 GiB, rows 2^24 floats apart
    kd, vd, n_slots = 64, 16, (5 << 30) // (64 * 16 * 4)
    rows, ld = 20, 1 << 24
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    q, k, v, z = f(rows, 1, kd), f(rows, 1, kd), f(rows, 1, vd), f(1, vd, kd)
    slot = n_slots - 1
    big.view(n_slots, -1)[slot].copy_(t(z.reshape(-1)))
    g, b = t(np.full((rows, 1), -0.1, np.float32)), t(np.full((rows, 1), 0.5, np.float32))
    wide = big.as_strided((rows, kd), (ld, 1))
    wide.copy_(t(q.reshape(rows, kd)))
    kk, vv, sl = t(k), t(v), t(np.array([slot], np.int32))
    off = t(np.array([0, rows], np.int32))
    for parts in (0, 1):
        os.environ["GGQ_DELTA_PARTS"] = str(parts)
        try:
            out, so = torch.empty((rows, vd), device="cuda"), torch.empty_like(big)
            p = gl.DeltaRuleParams(n_k_head=1, n_v_head=1, k_dim=kd, v_dim=vd, q=big.data_ptr(), ldq=ld, k=kk.data_ptr(), ldk=kd, v=vv.data_ptr(),
                                   ldv=vd, gate=g.data_ptr(), ld_gate=1, beta=b.data_ptr(), ld_beta=1, flags=gl.DELTA_QK_NORM, eps=EPS,
                                   state=big.data_ptr(), state_out=so.data_ptr(), n_slots=n_slots, slot=sl.data_ptr(), n_seq=1, n_rows=rows,
                                   row_off=off.data_ptr(), out=out.data_ptr(), ldo=vd)
            ctx.check(ctx.lib.ggq_delta_rule_dev(ctx.h, p, stream()), "delta rule")
            O, S = host(out), host(so.view(n_slots, -1)[slot])
        finally:
            del os.environ["GGQ_DELTA_PARTS"]
        want, S_want, tol, S_tol = su.delta(q, k, v, host(g).astype(float), host(b).astype(float), z, True, EPS)
        au.check(O.reshape(rows, 1, vd), want, tol)
        au.check(S.reshape(1, vd, kd), S_want, S_tol)
        del so
    # logits and norm rows 2^24 floats apart
    n, V = 72, 1000
    x = f(n, V)
    big.as_strided((n, V), (ld, 1)).copy_(t(x))
    u, tok, temp = t(rng.random(n).astype(np.float32)), torch.zeros(n, dtype=torch.int32, device="cuda"), t(np.ones(n, np.float32))
    p = gl.SampleParams(n_rows=n, n_vocab=V, logits=big.data_ptr(), ld=ld, temperature=temp.data_ptr(), u=u.data_ptr(), token=tok.data_ptr())
    ctx.check(ctx.lib.ggq_sample_dev(ctx.h, p, stream()), "sample")
    for r, got in enumerate(host(tok)):
        want, _, near = su.sample(x[r], u=host(u)[r])
        assert got == want or near <= su.BORDER
    y = torch.empty((n, V), device="cuda")
    p = gl.NormParams(n_rows=n, n_cols=V, x=big.data_ptr(), ldx=ld, eps=EPS, out=y.data_ptr(), ldo=V)
    ctx.check(ctx.lib.ggq_norm_dev(ctx.h, p, stream()), "norm")
    want = su.norm(x, eps=EPS)[1]
    au.check(host(y), want, 2 * su.U32 * np.abs(want) + 1e-37)


@pytest.mark.parametrize("planes", ["0", "1"])
def test_captured_attention_of_prompts_in_flight_together(ctx, monkeypatch, planes):
    """Two captured calls of many rows that need workspace and an eager one, at once on three streams; lengths and offsets
    rewritten between replays; every replay equals the eager call bit for bit."""
    import torch
    monkeypatch.setenv("GGQ_KV_PLANES", planes)
    rng = np.random.default_rng(7)
    n_seq, per, rows = 3, 24, 400
    st = Step(ctx, n_seq, per, 8)
    total = n_seq * per * PAGE
    k, v = (t(rng.standard_normal((total, NKV, HD)).astype(np.float32)) for _ in range(2))
    full, all_ = t(np.full(n_seq, per * PAGE, np.int32)), t(np.arange(n_seq + 1, dtype=np.int32) * per * PAGE)
    seqs = gl.KvSeqs(n_seq, per, per * PAGE, st.table.data_ptr(), full.data_ptr())
    ctx.check(ctx.lib.ggq_kv_store_dev(ctx.h, st.cache, seqs, ptr(all_), total, ptr(k), NKV * HD, ptr(v), NKV * HD, 0, stream()), "store")
    qs = [t(rng.standard_normal((rows, NH, HD)).astype(np.float32)) for _ in range(3)]
    outs, refs = ([torch.zeros_like(q) for q in qs] for _ in range(2))
    lens, offs = [torch.zeros(n_seq, dtype=torch.int32, device="cuda") for _ in qs], [torch.zeros(n_seq + 1, dtype=torch.int32, device="cuda") for _ in qs]

    def call(i, out, s):
        own = gl.KvSeqs(n_seq, per, per * PAGE, st.table.data_ptr(), lens[i].data_ptr())
        ctx.check(ctx.lib.ggq_attention_kv_rows_dev(ctx.h, st.cache, own, ptr(offs[i]), rows, ptr(qs[i]), NH * HD, NH, 0.0, 0, ptr(out), NH * HD, s), "attention")

    call(0, outs[0], stream())  # sizes the workspace, and what captures take
    torch.cuda.synchronize()
    streams, graphs = [torch.cuda.Stream() for _ in range(3)], [torch.cuda.CUDAGraph() for _ in range(2)]
    for i, g in enumerate(graphs):
        with torch.cuda.graph(g, stream=streams[i]):
            call(i, outs[i], streams[i].cuda_stream)
    for turn in range(4):
        for i in range(3):
            cut = np.sort(rng.integers(0, rows + 1, 2))
            off = np.array([0, *cut, rows - turn], np.int32)
            off[1:3] = np.minimum(off[1:3], off[3])
            offs[i].copy_(t(off))
            lens[i].copy_(t(np.minimum(np.diff(off) + rng.integers(0, 300, n_seq), per * PAGE).astype(np.int32)))
            outs[i].fill_(7.0)
            refs[i].fill_(7.0)
        torch.cuda.synchronize()
        for i in range(3):
            if i < 2:
                with torch.cuda.stream(streams[i]):
                    graphs[i].replay()
            else:
                call(i, outs[i], streams[i].cuda_stream)
        torch.cuda.synchronize()
        for i in range(3):
            call(i, refs[i], stream())
        torch.cuda.synchronize()
        for o, r in zip(outs, refs):
            assert torch.equal(o, r), turn
