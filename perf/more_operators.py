"""Performance cases of the operators around a layer's matmuls in a server's step over new tokens: what mixes tokens
(the gated delta rule of linear attention layers, attention of new rows over a paged quantized cache), what stands
between the layers (residual, RMSNorm and the int8 rows that the next matmul reads) and what ends the step (sampling).

Four kinds of case, told apart by `kind`:

  norm    residual's addition, RMSNorm of rows or of their heads, a SiLU gate, int8 codes (`ggq_norm_dev`)
  sample  a token of each row of logits by temperature, top-k, top-p, min-p and a given random number (`ggq_sample_dev`)
  delta   gated delta rule of packed sequences with their states (`ggq_delta_rule_dev`)
  chunk   causal attention of the last rows of each sequence over its quantized cache (`ggq_attention_kv_rows_dev`)

With `own` false `run` computes the operators from elementary torch operations.
"""
import functools
import math

import torch

own = False

F32, Q8_ROW, Q8_BLOCK32 = 0, 1, 2  # activation treatments of a matmul's input
MXFP4, MXFP8 = 4, 8  # a cache's formats: 32 values share a power of two; e2m1 and e4m3 codes
TILE = 32  # positions of a record in a page


# ---------------------------------------------------------------- the cases

def _norm(name, rows, cols, add=True, head=0, gate=False, act=Q8_ROW):
    """`head`: values that are normalised together (0: the row); `act`: F32 returns the rows, the others their codes."""
    return dict(name=name, kind="norm", rows=rows, cols=cols, add=add, head=head, gate=gate, act=act)


def _sample(name, rows, vocab, top_k=0, top_p=1.0, min_p=0.0, spread=2.5, greedy=0):
    """`spread`: deviation of the logits; `greedy`: how many rows have temperature 0."""
    return dict(name=name, kind="sample", rows=rows, vocab=vocab, top_k=top_k, top_p=top_p, min_p=min_p, spread=spread,
                greedy=greedy)


def _delta(name, seqs, longest, k_heads, v_heads, k_dim, v_dim, raw=True):
    """`raw`: decay and step size come as a model's projections and are made from them, q and k are normalised."""
    return dict(name=name, kind="delta", seqs=seqs, longest=longest, k_heads=k_heads, v_heads=v_heads, k_dim=k_dim,
                v_dim=v_dim, raw=raw)


def _chunk(name, seqs, longest, before, heads, kv_heads, head_dim, k_type, v_type, page, window=0):
    """`seqs` sequences whose new rows go from `longest` down, each behind about `before` positions."""
    return dict(name=name, kind="chunk", seqs=seqs, longest=longest, before=before, heads=heads, kv_heads=kv_heads,
                head_dim=head_dim, k_type=k_type, v_type=v_type, page=page, window=window)


def listed():
    return [
        # one token of a 1B model between two matmuls of int8 rows: launch latency
        _norm("norm_token_q8", 1, 2048),
        # a prompt's rows of an 8B model
        _norm("norm_prompt_q8", 2047, 4096),
        # the heads of a linear attention layer, normalised one by one and gated, for an fp32 output projection
        _norm("norm_heads_gated", 513, 4096, add=False, head=128, gate=True, act=F32),
        # one sequence of a chat with the usual settings
        _sample("sample_token", 1, 128256, top_k=40, top_p=0.95, min_p=0.05),
        # a server's batch that samples by top-p alone, some of its rows greedy
        _sample("sample_batch_top_p", 33, 128256, top_p=0.9, greedy=3),
        # many rows of a small odd vocabulary, all of it kept
        _sample("sample_batch_whole", 200, 32003, spread=1.5),
        # one token of each sequence of a server's batch: the states' bytes
        _delta("delta_batch_tokens", 48, 1, 16, 32, 128, 128),
        # packed prompts of a small model, decays and step sizes already made
        _delta("delta_packed", 7, 413, 4, 8, 64, 64, raw=False),
        # a long prompt
        _delta("delta_long", 1, 8191, 16, 32, 128, 128),
        # five proposed tokens of one sequence to be checked: latency
        _chunk("chunk_check_one", 1, 5, 700, 12, 2, 128, MXFP4, MXFP4, 64),
        # the same of a server's batch behind long contexts: the cache's bytes
        _chunk("chunk_check_batch", 24, 4, 6000, 32, 8, 128, MXFP8, MXFP4, 64),
        # the next part of a long prompt: the matrix products
        _chunk("chunk_prompt", 1, 1023, 7000, 32, 8, 128, MXFP8, MXFP8, 256),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def _draw(rng):
    kind = rng.choice(["norm", "sample", "delta", "delta", "chunk", "chunk"])
    if kind == "norm":
        act = rng.choice([F32, Q8_ROW, Q8_ROW, Q8_BLOCK32])
        if rng.random() < 0.4:
            head = rng.choice([64, 128, 256])
            cols = head * _log(rng, 1, 64)
        else:
            head, cols = 0, 32 * _log(rng, 4, 512) if act == Q8_BLOCK32 else 4 * _log(rng, 32, 4096)
        rows = _log(rng, 1, 2048)
        c = _norm("", rows if rows * cols < 8 << 20 else max(1, (8 << 20) // cols), cols, rng.random() < 0.6, head,
                  head > 0 and rng.random() < 0.6, act)
    elif kind == "sample":
        rows = rng.choice([1, 1, _log(rng, 2, 128)])
        c = _sample("", rows, min(_log(rng, 1000, 200000), 4000000 // rows), rng.choice([0, 0, _log(rng, 1, 1000)]),
                    rng.choice([1.0, 0.95, rng.uniform(0.05, 0.99)]), rng.choice([0.0, 0.0, 0.05, rng.uniform(0.001, 0.5)]),
                    rng.uniform(0.5, 6.0), rng.choice([0, 0, rows // 3]))
    elif kind == "delta":
        k_heads, seqs = rng.choice([1, 2, 4, 8, 16]), rng.choice([1, 1, _log(rng, 2, 48)])
        c = _delta("", seqs, rng.choice([1, _log(rng, 2, 8191 // seqs), _log(rng, 2, 8191 // seqs)]), k_heads,
                   k_heads * rng.choice([1, 2, 2, 4]) if k_heads < 16 else rng.choice([16, 32]), rng.choice([64, 128, 128]),
                   rng.choice([64, 128, 128, 48]), rng.random() < 0.7)
    else:
        kv, seqs = rng.choice([1, 2, 4, 8]), rng.choice([1, 1, _log(rng, 2, 40)])
        c = _chunk("", seqs, rng.choice([_log(rng, 1, 16), _log(rng, 1, 1500 // seqs)]),
                   rng.choice([0, _log(rng, 1, min(20000, 150000 // seqs))]), kv * rng.choice([1, 2, 4, 5, 6, 8]), kv,
                   rng.choice([64, 128, 128, 256]), rng.choice([MXFP4, MXFP8]), rng.choice([MXFP4, MXFP4, MXFP8]),
                   TILE * _log(rng, 1, 16), rng.choice([0, 0, 0, _log(rng, 1, 4000)]))
    del c["name"]
    return c


@functools.lru_cache(maxsize=1)
def _most():
    most = {}
    for c in listed():
        for k, v in work(c).items():
            most[c["kind"], k] = max(most.get((c["kind"], k), 0), v)
    return most


def draw(rng):
    """One more case, of no more work than the largest listed one of its kind."""
    while True:
        c = _draw(rng)
        if all(v <= _most()[c["kind"], k] for k, v in work(c).items()):
            return c


# ------------------------------------------------------------------- shapes

def _lengths(case):
    """Rows of each sequence: from the longest down to a third of it, none alike the next."""
    n, longest = case["seqs"], case["longest"]
    return [max(1, longest - (longest * 2 * i) // (3 * n) - i % 2) for i in range(n)]


def _before(case):
    """Positions in front of each sequence's rows: no two sequences need have as many."""
    return [case["before"] - (case["before"] * i) // (2 * case["seqs"]) for i in range(case["seqs"])]


def _starts(counts):
    return [sum(counts[:i]) for i in range(len(counts) + 1)]


def _bits(case):
    """Bytes of one position of one kv head, K and V: the codes and a byte for each 32 values."""
    return case["head_dim"] * (case["k_type"] + case["v_type"]) // 8 + 2 * (case["head_dim"] // 32)


def work(case):
    kind = case["kind"]
    if kind == "norm":
        n = case["rows"] * case["cols"]
        scales = case["rows"] if case["act"] == Q8_ROW else n // 32 if case["act"] == Q8_BLOCK32 else 0
        return {"bytes": n * (4 + 8 * case["add"] + 4 * case["gate"] + (4 if case["act"] == F32 else 1)) + 4 * scales,
                "flops": n * 8}
    if kind == "sample":
        return {"bytes": case["rows"] * (4 * case["vocab"] + 28), "flops": case["rows"] * case["vocab"] * 4}
    lengths = _lengths(case)
    rows = sum(lengths)
    if kind == "delta":  # the recurrence's products
        state = case["v_heads"] * case["k_dim"] * case["v_dim"]
        return {"bytes": 4 * rows * (2 * case["k_heads"] * case["k_dim"] + 2 * case["v_heads"] * case["v_dim"] + 2 * case["v_heads"])
                + 8 * case["seqs"] * state, "flops": 6 * rows * state}
    seen = read = 0
    for n, b in zip(lengths, _before(case)):
        w = case["window"] or n + b
        full = max(0, min(n, w - b))  # rows that see all before them
        seen += full * (b + 1) + full * (full - 1) // 2 + (n - full) * w
        read += min(n + b, n + w - 1)
    return {"bytes": read * case["kv_heads"] * _bits(case) + rows * case["heads"] * case["head_dim"] * 8,
            "flops": 4 * seen * case["heads"] * case["head_dim"]}


# ------------------------------------------------------- formats of a cache

# e2m1: sign, two bits of exponent, one of mantissa
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]


@functools.lru_cache(maxsize=None)
def _table(bits, device):
    """The values of all codes of a format."""
    if bits == 4:
        return torch.tensor(E2M1, device=device)
    return torch.arange(256, device=device).to(torch.uint8).view(torch.float8_e4m3fn).float()


def _encode(x, bits):
    """Code and scale bytes of rows x [..., head_dim]: blocks of 32 under the power of two that brings their largest
    value below the largest code."""
    b = x.unflatten(-1, (-1, 32))
    e = torch.frexp(b.abs().amax(-1, keepdim=True) / (6.0 if bits == 4 else 448.0))[1].clamp(-60, 60)
    y = b * torch.exp2(-e.float())
    if bits == 8:
        codes = y.to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        mags = _table(4, x.device)[:8]
        codes = torch.bucketize(y.abs(), (mags[1:] + mags[:-1]) / 2).to(torch.uint8) + 8 * (y < 0).to(torch.uint8)
    return codes.flatten(-2), (e.squeeze(-1) + 127).to(torch.uint8)


def _pack(codes, bits, value):
    """Records' codes [n, 32, head_dim] as bytes: 64 lanes of 16-byte pieces.  K: lane 16 g + r has positions r and
    16 + r, the g-th quarter of the head; V (`value`): lane 16 g + r has positions 4 g .. 4 g + 3 and 16 further,
    the r-th sixteenth of the head."""
    n, _, hd = codes.shape
    c = (codes.view(n, 2, 4, 4, 16, hd // 16).permute(0, 2, 4, 1, 3, 5) if value
         else codes.view(n, 2, 16, 4, hd // 4).permute(0, 3, 2, 1, 4)).reshape(n, 64, hd // 2)
    if bits == 4:
        c = c[..., 0::2] | (c[..., 1::2] << 4)
    return c.reshape(n, 64, -1, 16).transpose(1, 2).reshape(n, -1)


def _pack_scales(s, value):
    """Records' scale bytes [n, 32, blocks] in the order of the lanes that use them."""
    n, _, b = s.shape
    return (s.view(n, 2, 4, 4, b).permute(0, 4, 2, 1, 3) if value else s.view(n, 2, 16, b).permute(0, 3, 2, 1)).reshape(n, -1)


def _record(case):
    """Byte offsets in a record of 32 positions of one kv head: K codes, V codes, K scales, V scales, end."""
    hd = case["head_dim"]
    k, v = TILE * hd * case["k_type"] // 8, TILE * hd * case["v_type"] // 8
    return 0, k, k + v, k + v + hd, k + v + 2 * hd


def _read(case, records):
    """fp32 K and V [..., 32, head_dim] of records."""
    hd, (a, b, c, d, e), lead = case["head_dim"], _record(case), records.shape[:-1]
    rec = records.reshape(-1, e)
    n = rec.shape[0]
    outs = []
    for at, end, sc, bits, value in ((a, b, c, case["k_type"], False), (b, c, d, case["v_type"], True)):
        x = rec[:, at:end].reshape(n, -1, 64, 16).transpose(1, 2).reshape(n, 64, -1)
        if bits == 4:
            x = torch.stack((x & 15, x >> 4), -1).flatten(-2)
        s = rec[:, sc:sc + hd]
        if value:
            x = x.view(n, 4, 16, 2, 4, hd // 16).permute(0, 3, 1, 4, 2, 5)
            s = s.reshape(n, hd // 32, 4, 2, 4).permute(0, 3, 2, 4, 1)
        else:
            x = x.view(n, 4, 16, 2, hd // 4).permute(0, 3, 2, 1, 4)
            s = s.reshape(n, hd // 32, 16, 2).permute(0, 3, 2, 1)
        x, s = _table(bits, rec.device)[x.reshape(n, 32, hd // 32, 32).int()], s.reshape(n, 32, hd // 32, 1)
        outs.append((x * torch.exp2(s.float() - 127.0)).view(*lead, 32, hd))
    return outs


# ------------------------------------------------------------------ inputs

def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, device="cuda", generator=g)

    s = {"case": case}
    if case["kind"] == "norm":
        rows, cols = case["rows"], case["cols"]
        # a residual stream: a few channels much larger than the others
        big = torch.where(torch.rand(cols, device="cuda", generator=g) < 0.01, 12.0, 1.0)
        s["x"], s["w"] = randn(rows, cols) * big, 1 + 0.2 * randn(case["head"] or cols)
        s["add"] = randn(rows, cols) * 0.3 if case["add"] else None
        s["gate"] = 2 * randn(rows, cols) if case["gate"] else None
        s["sum"] = torch.empty((rows, cols), device="cuda")
        s["out"] = torch.empty((rows, cols), device="cuda")
        s["codes"] = torch.empty((rows, cols), dtype=torch.int8, device="cuda")
        s["scales"] = torch.empty((rows, 1) if case["act"] == Q8_ROW else (rows, -(-cols // 32), 1), device="cuda")
        return s
    if case["kind"] == "sample":
        rows, n = case["rows"], case["vocab"]
        x = randn(rows, n) * case["spread"]
        # a handful of tokens that the model means, the best of them a different one from row to row
        at = torch.randint(0, n, (rows, 8), device="cuda", generator=g)
        s["x"] = x.scatter(1, at, x.amax(1, keepdim=True) + 2.5 * torch.rand((rows, 8), device="cuda", generator=g))
        t = 0.6 + 0.6 * torch.rand(rows, device="cuda", generator=g)
        t[: case["greedy"]] = 0.0
        s["t"], s["u"] = t, torch.rand(rows, device="cuda", generator=g)
        s["k"] = torch.full((rows,), case["top_k"], dtype=torch.int32, device="cuda")
        s["p"], s["m"] = torch.full((rows,), case["top_p"], device="cuda"), torch.full((rows,), case["min_p"], device="cuda")
        s["token"], s["prob"] = torch.empty(rows, dtype=torch.int32, device="cuda"), torch.empty(rows, device="cuda")
        return s
    lengths = _lengths(case)
    rows = sum(lengths)
    s["off"] = _i32(_starts(lengths))
    if case["kind"] == "delta":
        kh, vh, kd, vd, n = case["k_heads"], case["v_heads"], case["k_dim"], case["v_dim"], case["seqs"]
        s["q"], s["k"], s["v"] = randn(rows, kh, kd), randn(rows, kh, kd), randn(rows, vh, vd)
        if case["raw"]:  # a projection of the row, a learned rate (negative) and bias of each head
            s["gate"], s["beta"] = randn(rows, vh), 1.5 * randn(rows, vh)
            s["rate"], s["bias"] = -torch.exp(randn(vh) - 1.5), 0.5 * randn(vh) - 1.0
        else:
            s["gate"], s["beta"] = -torch.exp(1.2 * randn(rows, vh) - 3.0), torch.sigmoid(randn(rows, vh))
            s["rate"] = s["bias"] = None
            for x in ("q", "k"):
                s[x] = s[x] / s[x].norm(dim=-1, keepdim=True)
        s["state"], s["state_out"] = 0.3 * randn(n + 2, vh, vd, kd), torch.zeros((n + 2, vh, vd, kd), device="cuda")
        s["slot"] = torch.randperm(n + 2, device="cuda", generator=g)[:n].int().contiguous()
        s["out"] = torch.empty((rows, vh, vd), device="cuda")
        return s
    hd, kv = case["head_dim"], case["kv_heads"]
    lens = [n + b for n, b in zip(lengths, _before(case))]
    per = -(-max(lens) // case["page"])
    n_pages = case["seqs"] * per + 3
    s["lens"] = _i32(lens)
    s["table"] = torch.randperm(n_pages, device="cuda", generator=g)[: case["seqs"] * per].view(-1, per).int().contiguous()
    parts = []
    for bits, value in ((case["k_type"], False), (case["v_type"], True)):
        x = randn(n_pages * kv * (case["page"] // TILE), TILE, hd)
        x *= torch.where(torch.rand((1, 1, hd), device="cuda", generator=g) < 0.03, 10.0, 1.0)
        codes, scales = _encode(x, bits)
        parts.append((_pack(codes, bits, value), _pack_scales(scales, value)))
    s["pages"] = torch.cat([parts[0][0], parts[1][0], parts[0][1], parts[1][1]], 1).view(n_pages, -1).contiguous()
    s["q"], s["out"] = randn(rows, case["heads"], hd), torch.empty((rows, case["heads"], hd), device="cuda")
    return s


# ---------------------------------------------------- the framework's calls

@functools.lru_cache(maxsize=1)
def _ctx():
    import ggnpu_amd.lib as gl
    return gl.Context(torch.cuda.current_device())


def _ptr(t):
    return None if t is None else t.data_ptr()


def _own(s):
    import ggnpu_amd.lib as gl
    case, ctx, stream, kind = s["case"], _ctx(), torch.cuda.current_stream().cuda_stream, s["case"]["kind"]
    if kind == "norm":
        rows, cols, act = case["rows"], case["cols"], case["act"]
        p = gl.NormParams(n_rows=rows, n_cols=cols, x=_ptr(s["x"]), ldx=cols, add=_ptr(s["add"]), ld_add=cols,
                          sum=_ptr(s["sum"]) if case["add"] else None, ld_sum=cols, norm_w=_ptr(s["w"]),
                          norm_len=case["head"], eps=1e-6, gate=_ptr(s["gate"]), ld_gate=cols,
                          out=_ptr(s["out"]) if act == F32 else None, ldo=cols, act_mode=act,
                          codes=_ptr(s["codes"]) if act else None, scales=_ptr(s["scales"]) if act else None)
        ctx.check(ctx.lib.ggq_norm_dev(ctx.h, p, stream), "norm")
        if act == F32:
            y = s["out"]
        else:
            y = s["codes"] * s["scales"] if act == Q8_ROW else (s["codes"].view(rows, -1, 32) * s["scales"]).view(rows, cols)
        return (s["sum"], y) if case["add"] else (y,)
    if kind == "sample":
        p = gl.SampleParams(n_rows=case["rows"], n_vocab=case["vocab"], logits=_ptr(s["x"]), ld=case["vocab"],
                            temperature=_ptr(s["t"]), top_k=_ptr(s["k"]), top_p=_ptr(s["p"]), min_p=_ptr(s["m"]),
                            u=_ptr(s["u"]), token=_ptr(s["token"]), prob=_ptr(s["prob"]))
        ctx.check(ctx.lib.ggq_sample_dev(ctx.h, p, stream), "sample")
        return s["token"], s["prob"]
    if kind == "delta":
        kh, vh, kd, vd, n = case["k_heads"], case["v_heads"], case["k_dim"], case["v_dim"], case["seqs"]
        p = gl.DeltaRuleParams(n_k_head=kh, n_v_head=vh, k_dim=kd, v_dim=vd, q=_ptr(s["q"]), ldq=kh * kd, k=_ptr(s["k"]),
                               ldk=kh * kd, v=_ptr(s["v"]), ldv=vh * vd, gate=_ptr(s["gate"]), ld_gate=vh,
                               beta=_ptr(s["beta"]), ld_beta=vh, gate_rate=_ptr(s["rate"]), gate_bias=_ptr(s["bias"]),
                               flags=gl.DELTA_BETA_SIGMOID | gl.DELTA_QK_NORM if case["raw"] else 0, eps=1e-6,
                               state=_ptr(s["state"]), state_out=_ptr(s["state_out"]), n_slots=n + 2, slot=_ptr(s["slot"]),
                               n_seq=n, n_rows=s["q"].shape[0], row_off=_ptr(s["off"]), out=_ptr(s["out"]), ldo=vh * vd)
        ctx.check(ctx.lib.ggq_delta_rule_dev(ctx.h, p, stream), "delta rule")
        return s["out"], s["state_out"]
    hd = case["head_dim"]
    cache = gl.KvCache(_ptr(s["pages"]), s["pages"].shape[0], case["page"], case["kv_heads"], hd, case["k_type"], case["v_type"])
    seqs = gl.KvSeqs(case["seqs"], s["table"].shape[1], case["longest"] + case["before"], _ptr(s["table"]), _ptr(s["lens"]))
    ld = case["heads"] * hd
    ctx.check(ctx.lib.ggq_attention_kv_rows_dev(ctx.h, cache, seqs, _ptr(s["off"]), s["q"].shape[0], _ptr(s["q"]), ld,
                                                case["heads"], 0.0, case["window"], _ptr(s["out"]), ld, stream), "chunk attention")
    return s["out"]


# ------------------------------------------------------------ the plain form

def _quantize(y, act):
    """Rows as the values of their int8 codes: scale = the largest magnitude / 127, of a row or of 32 values."""
    b = y if act == Q8_ROW else y.unflatten(-1, (-1, 32))
    scale = b.abs().amax(-1, keepdim=True) / 127.0
    scale = torch.where(scale > 0, scale, 1.0)
    return (torch.round(b * (1.0 / scale)).clamp(-128, 127) * scale).view(y.shape)


def _plain_norm(case, s):
    x = s["x"] + s["add"] if case["add"] else s["x"]
    # in 64 bits, each value rounded once: a last bit of difference would move codes next to a border
    h = x.double().unflatten(-1, (-1, case["head"] or case["cols"]))
    y = (h * (1.0 / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-6)) * s["w"]).view(x.shape)
    if case["gate"]:
        z = s["gate"].double()
        y = y * (z / (1.0 + torch.exp(-z)))
    y = y.float()
    if case["act"]:
        y = _quantize(y, case["act"])
    return (x, y) if case["add"] else (y,)


def _plain_sample(case, s):
    # weights and their sums in 64 bits: a random number may fall next to the border between two tokens
    x, t = s["x"].double(), s["t"].double()[:, None]
    greedy = t <= 0
    top = x.amax(-1, keepdim=True)
    w = torch.where(greedy, (x == top).double(), torch.exp((x - top) / torch.where(greedy, 1.0, t)))
    v, order = torch.sort(w, dim=-1, descending=True, stable=True)
    at = torch.arange(w.shape[1], device=w.device)
    k = s["k"][:, None]
    keep = ((k <= 0) | (at < k)) & (~greedy | (at == 0))
    v = torch.where(keep, v, 0.0)
    ahead = v.cumsum(-1) - v  # of the larger ones
    p = s["p"].double()[:, None]
    keep &= (p >= 1) | (at == 0) | (ahead < p * v.sum(-1, keepdim=True))
    keep &= (at == 0) | (v >= s["m"].double()[:, None])
    kept = torch.zeros_like(w).scatter(1, order, torch.where(keep, v, 0.0))
    total = kept.sum(-1, keepdim=True)
    passed = kept.cumsum(-1) > s["u"].double()[:, None] * total
    token = passed.int().argmax(-1)
    return token.int(), (kept.gather(1, token[:, None]) / total)[:, 0].float()


def _padded(x, off, lengths, steps, fill=0.0):
    """Packed rows as [sequences, steps, ...]."""
    at = torch.arange(steps, device=x.device)
    there = at < lengths[:, None]
    rows = x[torch.where(there, off[:-1, None] + at, 0)]
    return torch.where(there.view(*there.shape, *([1] * (x.ndim - 1))), rows, fill)


def _plain_delta(case, s):
    """In blocks of up to 64 rows: within one the rows' values are solved for together, the state goes from block to block."""
    vh, kd, vd = case["v_heads"], case["k_dim"], case["v_dim"]
    q, k, v, g, b = s["q"], s["k"], s["v"], s["gate"], s["beta"]
    if case["raw"]:
        z = g + s["bias"]
        g = s["rate"] * torch.where(z > 20, z, torch.log1p(torch.exp(z.clamp(max=20))))
        b = 1.0 / (1.0 + torch.exp(-b))
        q, k = (x / torch.sqrt((x * x).sum(-1, keepdim=True) + 1e-6) for x in (q, k))
    off, lengths = s["off"].long(), (s["off"][1:] - s["off"][:-1]).long()
    n, longest = case["seqs"], case["longest"]
    c = min(64, longest)
    blocks = -(-longest // c)
    q, k, v, g, b = (_padded(x, off, lengths, blocks * c) for x in (q / math.sqrt(kd), k, v, g, b))
    # [block, sequence and head, row, value]
    q, k = (x.repeat_interleave(vh // case["k_heads"], 2).view(n, blocks, c, vh, kd).permute(1, 0, 3, 2, 4).reshape(blocks, -1, c, kd)
            for x in (q, k))
    v = v.view(n, blocks, c, vh, vd).permute(1, 0, 3, 2, 4).reshape(blocks, -1, c, vd)
    g, b = (x.view(n, blocks, c, vh).permute(1, 0, 3, 2).reshape(blocks, -1, c, 1) for x in (g, b))
    sums = g.double().cumsum(2)
    low = torch.ones((c, c), dtype=torch.bool, device=q.device).tril()
    decay = torch.where(low, torch.exp(torch.where(low, sums - sums.transpose(2, 3), 0.0)), 0.0).float()
    kt = k.transpose(2, 3).contiguous()
    # (1 + A)^-1 of the strictly lower triangular A as a product of its powers, in 64 bits
    a = -(torch.matmul(k, kt) * decay * b * ~torch.eye(c, dtype=torch.bool, device=q.device)).double()
    inv, power = torch.eye(c, dtype=torch.float64, device=q.device) + a, a
    for _ in range(max(0, (c - 1).bit_length() - 1)):
        power = torch.matmul(power, power)
        inv = inv + torch.matmul(inv, power)
    inv = inv.float()
    grown = torch.exp(sums).float()
    own_v, own_k = torch.matmul(inv, b * v), torch.matmul(inv, b * grown * k)
    scores = torch.matmul(q, kt) * decay
    q, kt = q * grown, (k * decay[:, :, -1:].transpose(2, 3)).transpose(2, 3).contiguous()
    state = s["state"][s["slot"].long()].view(-1, vd, kd).transpose(1, 2).contiguous()
    out = torch.empty_like(v)
    for i in range(blocks):
        u = own_v[i] - torch.matmul(own_k[i], state)
        out[i] = torch.matmul(q[i], state) + torch.matmul(scores[i], u)
        state = grown[i, :, -1:] * state + torch.matmul(kt[i], u)
    at = torch.arange(blocks * c, device=q.device) < lengths[:, None]
    out = out.view(blocks, n, vh, c, vd).permute(1, 0, 3, 2, 4).reshape(n, blocks * c, vh, vd)[at]
    states = torch.zeros_like(s["state"])
    states[s["slot"].long()] = state.transpose(1, 2).reshape(n, vh, vd, kd)
    return out, states


def _plain_chunk(case, s):
    hd, kv, heads, n = case["head_dim"], case["kv_heads"], case["heads"], case["seqs"]
    rec = s["pages"].view(s["pages"].shape[0], kv, case["page"] // TILE, -1)[s["table"].long()]
    k, v = (x.permute(0, 2, 1, 3, 4, 5).reshape(n * kv, -1, hd) for x in _read(case, rec))
    off, lengths = s["off"].long(), (s["off"][1:] - s["off"][:-1]).long()
    q = _padded(s["q"], off, lengths, case["longest"])
    q = q.view(n, -1, kv, heads // kv, hd).permute(0, 2, 3, 1, 4).reshape(n * kv, -1, hd)
    scores = torch.matmul(q, k.transpose(1, 2).contiguous()).view(n, kv, heads // kv, case["longest"], -1) / math.sqrt(hd)
    row = (s["lens"] - lengths)[:, None] + torch.arange(case["longest"], device=q.device)
    at = torch.arange(k.shape[1], device=q.device)
    sees = at <= row[..., None]
    if case["window"]:
        sees &= at > row[..., None] - case["window"]
    scores = torch.where(sees[:, None, None], scores, -torch.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(n * kv, -1, k.shape[1]), v).view(n, kv, heads // kv, case["longest"], hd)
    o = o.permute(0, 3, 1, 2, 4).reshape(n, case["longest"], heads, hd)
    return o[torch.arange(case["longest"], device=q.device) < lengths[:, None]]


def run(state):
    if own:
        return _own(state)
    case = state["case"]
    return {"norm": _plain_norm, "sample": _plain_sample, "delta": _plain_delta, "chunk": _plain_chunk}[case["kind"]](case, state)


# --------------------------------------------------------- in 64 bits, apart

def _exact_norm(case, s):
    x = s["x"].double()
    total = x + s["add"].double() if case["add"] else x
    # what is normalised is the residual stream as it is kept, rounded to 32 bits
    heads = total.float().double().view(case["rows"], -1, case["head"] or case["cols"])
    y = heads / torch.linalg.vector_norm(heads, dim=-1, keepdim=True).square().div(heads.shape[-1]).add(1e-6).sqrt()
    y = (y * s["w"].double()).view(total.shape)
    if case["gate"]:
        y = y * torch.nn.functional.silu(s["gate"].double())
    if case["act"]:
        # codes are defined on the fp32 rows: step, its reciprocal and the quotient are rounded to 32 bits
        b = y.float().view(case["rows"], -1, 32 if case["act"] == Q8_BLOCK32 else case["cols"])
        step = (b.abs().max(-1, keepdim=True)[0].double() / 127).float()
        quotient = (b.double() * (1 / step.double()).float().double()).float()
        y = (quotient.double().round() * step.double()).view(y.shape)
    return (total, y) if case["add"] else (y,)


def _exact_sample(case, s):
    import numpy as np
    x, t, u, k, p, m = (s[i].double().cpu().numpy() for i in ("x", "t", "u", "k", "p", "m"))
    tokens, probs = [], []
    for i in range(case["rows"]):
        if t[i] <= 0:
            tokens.append(int(np.argmax(x[i])))
            probs.append(1.0)
            continue
        order = np.argsort(-x[i], kind="stable")  # the lowest index first among equals
        w = np.exp((x[i][order] - x[i].max()) / t[i])
        n = int(k[i]) if 0 < k[i] < len(w) else len(w)
        if p[i] < 1:
            n = min(n, int(np.searchsorted(np.cumsum(w[:n]), p[i] * w[:n].sum())) + 1)
        n = max(1, min(n, int((w >= m[i]).sum())))
        ids = np.sort(order[:n])
        c = np.cumsum(np.exp((x[i][ids] - x[i].max()) / t[i]))
        j = min(int(np.searchsorted(c, u[i] * c[-1], side="right")), n - 1)
        tokens.append(int(ids[j]))
        probs.append((c[j] - (c[j - 1] if j else 0.0)) / c[-1])
    return torch.tensor(tokens, dtype=torch.int32), torch.tensor(probs, dtype=torch.float64)


def _exact_delta(case, s):
    """Row by row, for all heads of a sequence at once."""
    group, kd = case["v_heads"] // case["k_heads"], case["k_dim"]
    q, k, v, g, b = (s[x].double() for x in ("q", "k", "v", "gate", "beta"))
    if case["raw"]:
        g = s["rate"].double() * torch.nn.functional.softplus(g + s["bias"].double(), threshold=60)
        b = torch.sigmoid(b)
        q, k = (x * (x.square().sum(-1, keepdim=True) + 1e-6).rsqrt() for x in (q, k))
    alpha, q, out = torch.exp(g)[..., None, None], q * kd ** -0.5, torch.empty_like(v)
    states = torch.zeros(s["state"].shape, dtype=torch.float64, device="cuda")
    slots, ends = s["slot"].tolist(), s["off"].tolist()
    # one step for all sequences that have that many rows; [sequence, head, v, k]
    live = list(range(case["seqs"]))
    mem = s["state"].double()[s["slot"].long()]
    b = b[..., None]
    for i in range(max(ends[j + 1] - ends[j] for j in live)):
        stay = [a for a, j in enumerate(live) if ends[j + 1] - ends[j] > i]
        if len(stay) < len(live):
            for a, j in enumerate(live):
                if a not in stay:
                    states[slots[j]] = mem[a]
            mem, live = mem[stay], [live[a] for a in stay]
        at = torch.tensor([ends[j] + i for j in live], device="cuda") if len(live) > 1 else slice(ends[live[0]] + i, ends[live[0]] + i + 1)
        kk, qq = (x[at].repeat_interleave(group, 1)[..., None] for x in (k, q))
        mem = mem * alpha[at]
        miss = b[at] * (v[at] - (mem @ kk)[..., 0])
        mem = mem + miss[..., None] * kk[..., 0][..., None, :]
        out[at] = (mem @ qq)[..., 0]
    for a, j in enumerate(live):
        states[slots[j]] = mem[a]
    return out, states


def _exact_chunk(case, s):
    """Sequence by sequence; a value's byte is found by the format's definition."""
    hd, kv, page, (a, b, c, d, size) = case["head_dim"], case["kv_heads"], case["page"], _record(case)
    group, off = case["heads"] // kv, s["off"].tolist()
    p, e = torch.arange(TILE, device="cuda")[:, None], torch.arange(hd, device="cuda")

    def values(rec, at, scales_at, bits, value):
        g, r = ((p % 16) // 4, e // (hd // 16)) if value else (e // (hd // 4), p % 16)
        n = ((p // 16) * 4 + p % 4) * (hd // 16) + e % (hd // 16) if value else (p // 16) * (hd // 4) + e % (hd // 4)
        byte = n * bits // 8
        byte = byte // 16 * 1024 + (16 * g + r) * 16 + byte % 16
        code = rec[:, (at + byte).flatten()].view(-1, TILE, hd)
        if bits == 4:
            code = torch.where(n % 2 == 1, code >> 4, code & 15)
        blk = e // 32
        where = (blk * 4 + g) * 8 + (p // 16) * 4 + p % 4 if value else (blk * 16 + r) * 2 + p // 16
        sc = rec[:, (scales_at + where.expand(TILE, hd)).flatten()].view(-1, TILE, hd)
        return _table(bits, rec.device).double()[code.long()] * torch.exp2(sc.double() - 127)

    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for i, n in enumerate(s["lens"].tolist()):
        rec = s["pages"][s["table"][i].long()].view(-1, kv, page // TILE, size).transpose(0, 1).reshape(kv, -1, size)
        rows, first = off[i + 1] - off[i], n - (off[i + 1] - off[i])
        pos = first + torch.arange(rows, device="cuda")[:, None]
        j = torch.arange(n, device="cuda")
        hidden = (j > pos) | (j <= pos - case["window"]) if case["window"] else j > pos
        for h in range(kv):
            kk = values(rec[h], a, c, case["k_type"], False).view(-1, hd)[:n]
            vv = values(rec[h], b, d, case["v_type"], True).view(-1, hd)[:n]
            for x in range(h * group, (h + 1) * group):
                w = (s["q"][off[i]:off[i + 1], x].double() @ kk.T.contiguous()) * hd ** -0.5
                out[off[i]:off[i + 1], x] = torch.softmax(w.masked_fill(hidden, -torch.inf), -1) @ vv
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "sample": _exact_sample, "delta": _exact_delta, "chunk": _exact_chunk}[case["kind"]](case, s)
