"""Performance cases of the attention operators around the KV cache: what a GGUF inference program runs between the
q/k/v projections and the output projection of a layer.

Five kinds of case, told apart by `kind`:

  rope    rotary positions of q and k heads (`ggq_rope_dev`), optionally behind an RMSNorm of each head
  store   K and V rows quantized into the pages of a cache (`ggq_kv_store_dev`) and the same rows read back, since
          the values that the codes stand for are what can be compared
  load    positions of a quantized cache read back as rows (`ggq_kv_load_dev`)
  decode  attention of one token of each sequence over its quantized cache (`ggq_attention_kv_dev`)
  prompt  causal attention of whole prompts, packed one behind the other (`ggq_attention_prompt_dev`)

K and V rows are N(0, 1) with a few channels ten times larger, as keys have them; q rows N(0, 1).  With `own` false
`run` computes the operators from elementary torch operations.
"""
import functools
import math

import torch

own = False

HALF, INTERLEAVED = 0, 1
F32, F16 = 0, 1
MXFP4, MXFP8 = 4, 8  # a cache's formats: 32 values share a power of two; e2m1 and e4m3 codes
TORCH = {F32: torch.float32, F16: torch.float16}
TILE = 32  # positions of a record in a page


# ---------------------------------------------------------------- the cases

def _rope(name, tokens, heads, kv_heads, head_dim, rot, layout=HALF, base=10000.0, norm=False, factors=False, yarn=1.0,
          far=0, out=F32):
    return dict(name=name, kind="rope", tokens=tokens, heads=heads, kv_heads=kv_heads, head_dim=head_dim, rot=rot,
                layout=layout, base=base, norm=norm, factors=factors, yarn=yarn, far=far, out=out)


def _cache(name, kind, seqs, longest, kv_heads, head_dim, k_type, v_type, page, **more):
    """`seqs` sequences whose lengths go from `longest` down; `page` positions a page."""
    return dict(name=name, kind=kind, seqs=seqs, longest=longest, kv_heads=kv_heads, head_dim=head_dim, k_type=k_type,
                v_type=v_type, page=page, **more)


def _prompt(name, seqs, longest, before, heads, kv_heads, head_dim, type, window=0):
    """`seqs` prompts whose rows go from `longest` down, each behind `before` positions that are in K and V already."""
    return dict(name=name, kind="prompt", seqs=seqs, longest=longest, before=before, heads=heads, kv_heads=kv_heads,
                head_dim=head_dim, type=type, window=window)


def listed():
    return [
        # one token of a 1B model at a far position, with its checkpoint's frequency factors: launch latency
        _rope("rope_decode", 1, 32, 8, 64, 64, base=500000.0, factors=True, far=130000),
        # a prompt of a model that normalises q and k heads first
        _rope("rope_prompt_qknorm", 2049, 16, 8, 128, 128, base=1e6, norm=True),
        # a server's batch: every sequence writes its new token
        _cache("store_batch_fp4", "store", 33, 1, 8, 128, MXFP4, MXFP4, 64, before=900, type=F32),
        # three prompts written at once, keys in 8 bits and values in 4
        _cache("store_prompts_fp8_fp4", "store", 3, 2047, 8, 64, MXFP8, MXFP4, 128, before=37, type=F32),
        # the cache of one sequence read back, as a prompt's next chunk needs it
        _cache("load_one_fp4", "load", 1, 1500, 8, 64, MXFP4, MXFP4, 2048, type=F32),
        # the caches of a batch into half-precision slabs
        _cache("load_batch_fp8_f16", "load", 16, 4001, 2, 128, MXFP8, MXFP8, 64, type=F16),
        # one token of a 1.5B model early in its answer: six query heads share a kv head; launch latency
        _cache("decode_short_fp4", "decode", 1, 300, 2, 128, MXFP4, MXFP4, 512, heads=12, window=0),
        # one token of a 1B model behind a very long context: the split over positions
        _cache("decode_long_fp4", "decode", 1, 131001, 8, 64, MXFP4, MXFP4, 256, heads=32, window=0),
        # a server's batch of ragged sequences over 128-wide heads: the cache's bytes
        _cache("decode_batch_fp8_fp4", "decode", 64, 8191, 8, 128, MXFP8, MXFP4, 64, heads=32, window=0),
        # a short question to a model with 256-wide heads: launch latency
        _prompt("prompt_short_f32", 1, 19, 0, 16, 2, 256, F32),
        # packed prompts behind a shared start in a half-precision slab, six query heads to a kv head
        _prompt("prompt_packed_f16", 5, 513, 130, 12, 2, 128, F16),
        # a long document of an 8B model: the matrix products
        _prompt("prompt_long_f32", 1, 8191, 0, 32, 8, 128, F32),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def _draw(rng):
    kind = rng.choice(["rope", "store", "load", "decode", "decode", "prompt", "prompt"])
    kv = rng.choice([1, 2, 4, 8])
    if kind == "rope":
        hd = rng.choice([64, 80, 96, 128, 256])
        c = _rope("", _log(rng, 1, 4096), kv * rng.choice([1, 2, 4, 6, 8]), kv, hd,
                  rng.choice([hd, hd, 8 * rng.randint(1, hd // 8)]), rng.choice([HALF, INTERLEAVED]),
                  rng.choice([1e4, 5e5, 1e6]), rng.random() < 0.5, rng.random() < 0.3, rng.choice([1.0, 1.0, 4.0, 32.0]),
                  rng.choice([0, _log(rng, 100, 1000000)]), rng.choice([F32, F32, F16]))
    elif kind == "prompt":
        hd, seqs = rng.choice([64, 128, 128, 256]), rng.choice([1, 1, _log(rng, 2, 40)])
        before = rng.choice([0, 0, _log(rng, 1, 8000)])
        c = _prompt("", seqs, _log(rng, 1, 6000 // seqs), before if seqs * before < 20000 else 0,
                    kv * rng.choice([1, 2, 4, 5, 6, 8, 16]), kv, hd, rng.choice([F32, F16]),
                    rng.choice([0, 0, 0, _log(rng, 1, 2000)]))
    else:
        hd, types = rng.choice([64, 128, 128, 256]), [rng.choice([MXFP4, MXFP8]), rng.choice([MXFP4, MXFP4, MXFP8])]
        page, seqs = TILE * _log(rng, 1, 32), rng.choice([1, 1, _log(rng, 2, 100)])
        if kind == "decode":
            c = _cache("", kind, seqs, _log(rng, 1, 200000 // seqs), kv, hd, *types, page,
                       heads=kv * rng.choice([1, 2, 4, 5, 6, 8, 16]), window=rng.choice([0, 0, 0, _log(rng, 1, 4000)]))
        elif kind == "load":
            c = _cache("", kind, seqs, _log(rng, 1, 30000 // seqs), kv, hd, *types, page, type=rng.choice([F32, F16]))
        else:
            c = _cache("", kind, seqs, rng.choice([1, _log(rng, 1, 8000 // seqs)]), kv, hd, *types, page,
                       before=rng.choice([0, _log(rng, 1, 500)]), type=rng.choice([F32, F32, F16]))
    del c["name"]
    return c


@functools.lru_cache(maxsize=1)
def _most():
    w = [work(c) for c in listed()]
    return {k: max(v[k] for v in w) for k in ("bytes", "flops")}


def draw(rng):
    most = _most()
    while True:
        c = _draw(rng)
        w = work(c)
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"]:
            return c


# ------------------------------------------------------------------- shapes

def _lengths(case):
    """Rows of each sequence: from the longest down to a third of it, none alike the next."""
    n, longest = case["seqs"], case["longest"]
    return [max(1, longest - (longest * 2 * i) // (3 * n) - i % 2) for i in range(n)]


def _starts(counts):
    return [sum(counts[:i]) for i in range(len(counts) + 1)]


def _bits(case):
    """Bytes of one position of one kv head, K and V: the codes and a byte for each 32 values."""
    return case["head_dim"] * (case["k_type"] + case["v_type"]) // 8 + 2 * (case["head_dim"] // 32)


def _seen(case):
    """(row, position) pairs that a prompt's or a decode's rows see, over all sequences."""
    total = 0
    for n in _lengths(case):
        rows, first = (n, case["before"]) if case["kind"] == "prompt" else (1, n - 1)
        w = case["window"] or first + rows
        lo = first + 1  # positions that the first row sees without a window, one more for each further row
        full = max(0, min(rows, w - lo + 1))  # rows that see less than the window's length, or just it
        total += full * lo + full * (full - 1) // 2 + (rows - full) * w
    return total


def work(case):
    kind, hd, kv = case["kind"], case["head_dim"], case["kv_heads"]
    e = 2 if case.get("type") == F16 else 4
    if kind == "rope":
        n = case["tokens"] * (case["heads"] + kv) * hd
        return {"bytes": n * (4 + (2 if case["out"] == F16 else 4)) + 4 * case["tokens"], "flops": 3 * n}
    lengths = _lengths(case)
    rows = sum(lengths)
    if kind == "store":  # the rows, their codes twice, their values
        return {"bytes": rows * kv * (2 * hd * e + 2 * _bits(case) + 2 * hd * e), "flops": rows * kv * hd * 8}
    if kind == "load":
        return {"bytes": rows * kv * (_bits(case) + 2 * hd * e), "flops": rows * kv * hd * 2}
    qo = case["heads"] * hd * 8
    if kind == "decode":
        w = case["window"]
        read = sum(min(n, w) if w else n for n in lengths)
        return {"bytes": read * kv * _bits(case) + case["seqs"] * qo, "flops": 4 * _seen(case) * case["heads"] * hd}
    return {"bytes": (rows + case["seqs"] * case["before"]) * kv * 2 * hd * e + rows * qo,
            "flops": 4 * _seen(case) * case["heads"] * hd}


# ------------------------------------------------------- formats of a cache

# e2m1: sign, two bits of exponent, one of mantissa
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]


@functools.lru_cache(maxsize=None)
def _e2m1(device):
    return torch.tensor(E2M1, device=device)


def _quantize(x, bits):
    """Rows x [..., head_dim] in blocks of 32: codes' values [..., blocks, 32] and the exponent of each block's scale.
    The scale is the smallest power of two that rounds the block's largest magnitude to no more than the largest code;
    the rounding is to the nearest code, ties to the even mantissa.  In 64 bits: every step is exact but the rounding
    itself."""
    b = x.double().unflatten(-1, (-1, 32))
    mant, ex = torch.frexp(b.abs().amax(-1, keepdim=True) / (7.0 if bits == 4 else 464.0))
    e = torch.where(mant == 0.5, ex - 1, ex).clamp(-126, 127)
    e = torch.where(mant == 0, torch.full_like(e, -126), e)
    y = torch.ldexp(b, -e)
    low, most, frac = (0, 6.0, 1) if bits == 4 else (-6, 448.0, 3)
    step = (torch.frexp(y)[1] - 1).clamp(min=low)
    step = torch.where(y == 0, torch.full_like(step, low), step) - frac
    return torch.ldexp(torch.round(torch.ldexp(y, -step)), step).clamp(-most, most), e


def _codes(v, e, bits):
    """Code and scale bytes of what _quantize gives."""
    if bits == 4:
        codes = torch.bucketize(v.abs(), _e2m1(v.device)[:8].double()).to(torch.uint8) + 8 * (v < 0).to(torch.uint8)
    else:
        codes = v.float().to(torch.float8_e4m3fn).view(torch.uint8)
    return codes.flatten(-2), (e.squeeze(-1) + 127).to(torch.uint8)


def _values(codes, scales, bits):
    """fp32 values of codes [..., head_dim] with scale bytes [..., head_dim / 32]."""
    v = _e2m1(codes.device)[codes.long()] if bits == 4 else codes.view(torch.float8_e4m3fn).float()
    s = torch.bitwise_left_shift(scales.int(), 23).view(torch.float32)
    return (v.unflatten(-1, (-1, 32)) * s.unsqueeze(-1)).flatten(-2)


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


def _unpack(data, bits, value, hd):
    n = data.shape[0]
    c = data.reshape(n, -1, 64, 16).transpose(1, 2).reshape(n, 64, -1)
    if bits == 4:
        c = torch.stack((c & 15, c >> 4), -1).flatten(-2)
    return (c.view(n, 4, 16, 2, 4, hd // 16).permute(0, 3, 1, 4, 2, 5) if value
            else c.view(n, 4, 16, 2, hd // 4).permute(0, 3, 2, 1, 4)).reshape(n, 32, hd)


def _pack_scales(s, value):
    """Records' scale bytes [n, 32, blocks] in the order of the lanes that use them."""
    n, _, b = s.shape
    return (s.view(n, 2, 4, 4, b).permute(0, 4, 2, 1, 3) if value else s.view(n, 2, 16, b).permute(0, 3, 2, 1)).reshape(n, -1)


def _unpack_scales(data, value, b):
    n = data.shape[0]
    return (data.view(n, b, 4, 2, 4).permute(0, 3, 2, 4, 1) if value
            else data.view(n, b, 16, 2).permute(0, 3, 2, 1)).reshape(n, 32, b)


def _record(case):
    """Byte offsets in a record of 32 positions of one kv head: K codes, V codes, K scales, V scales, end."""
    hd = case["head_dim"]
    k, v = TILE * hd * case["k_type"] // 8, TILE * hd * case["v_type"] // 8
    return 0, k, k + v, k + v + hd, k + v + 2 * hd


def _read(case, pages, table):
    """fp32 K and V [seqs, positions, kv heads, head_dim] of the pages of a table."""
    hd, kv, (a, b, c, d, e) = case["head_dim"], case["kv_heads"], _record(case)
    rec = pages.view(pages.shape[0], kv, case["page"] // TILE, e)[table.long()].reshape(-1, e)
    shape = (table.shape[0], table.shape[1], kv, case["page"], hd)

    def rows(codes, scales, bits, value):
        v = _values(_unpack(codes, bits, value, hd), _unpack_scales(scales, value, hd // 32), bits)
        return v.view(shape).transpose(2, 3).reshape(shape[0], -1, kv, hd)

    return rows(rec[:, a:b], rec[:, c:d], case["k_type"], False), rows(rec[:, b:c], rec[:, d:e], case["v_type"], True)


# ------------------------------------------------------------------ inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _rows(g, n, heads, hd, type=F32, channels=True):
    x = torch.randn((n, heads, hd), device="cuda", generator=g)
    if channels:
        x *= torch.where(torch.rand((heads, hd), device="cuda", generator=g) < 0.03, 10.0, 1.0)
    return x.to(TORCH[type])


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g, hd, kv = _gen(seed), case["head_dim"], case["kv_heads"]
    s = {"case": case}
    if case["kind"] == "rope":
        n = case["tokens"]
        s["freq"], s["mag"] = _frequencies(case)
        s["q"], s["k"] = _rows(g, n, case["heads"], hd), _rows(g, n, kv, hd)
        s["pos"] = torch.arange(n, dtype=torch.int32, device="cuda") + (case["far"] + seed % 7)
        s["qw"] = 1 + 0.1 * torch.randn(hd, device="cuda", generator=g) if case["norm"] else None
        s["kw"] = 1 + 0.1 * torch.randn(hd, device="cuda", generator=g) if case["norm"] else None
        s["q_out"] = torch.empty((n, case["heads"], hd), dtype=TORCH[case["out"]], device="cuda")
        s["k_out"] = torch.empty((n, kv, hd), dtype=TORCH[case["out"]], device="cuda")
        return s
    lengths = _lengths(case)
    if case["kind"] == "prompt":
        keys = [n + case["before"] for n in lengths]
        rows, total = sum(lengths), sum(keys)
        s["q"] = _rows(g, rows, case["heads"], hd, channels=False)
        s["k"], s["v"] = _rows(g, total, kv, hd, case["type"]), _rows(g, total, kv, hd, case["type"])
        s["q_off"], s["kv_off"] = _i32(_starts(lengths)), _i32(_starts(keys))
        s["out"] = torch.empty((rows, case["heads"], hd), device="cuda")
        return s
    lens = [n + case.get("before", 0) for n in lengths]
    per = -(-max(lens) // case["page"])
    n_pages = case["seqs"] * per + 3
    s["lens"] = _i32(lens)
    s["table"] = torch.randperm(n_pages, device="cuda", generator=g)[: case["seqs"] * per].view(-1, per).int().contiguous()
    records = n_pages * kv * (case["page"] // TILE)
    size = _record(case)[-1]
    if case["kind"] == "store":
        s["pages"] = torch.zeros((n_pages, kv * (case["page"] // TILE) * size), dtype=torch.uint8, device="cuda")
        s["k"], s["v"] = (_rows(g, sum(lengths), kv, hd, case["type"]) for _ in range(2))
        s["k_out"], s["v_out"] = torch.empty_like(s["k"]), torch.empty_like(s["v"])
        s["off"] = _i32(_starts(lengths))
        return s
    parts = []
    for bits, value in ((case["k_type"], False), (case["v_type"], True)):
        x = _rows(g, records, TILE, hd, channels=False)
        x *= torch.where(torch.rand((1, 1, hd), device="cuda", generator=g) < 0.03, 10.0, 1.0)
        codes, scales = _codes(*_quantize(x, bits), bits)
        parts.append((_pack(codes, bits, value), _pack_scales(scales, value)))
    s["pages"] = torch.cat([parts[0][0], parts[1][0], parts[0][1], parts[1][1]], 1).view(n_pages, -1).contiguous()
    if case["kind"] == "load":
        s["off"] = _i32(_starts(lengths))
        s["k_out"], s["v_out"] = (torch.empty((sum(lengths), kv, hd), dtype=TORCH[case["type"]], device="cuda") for _ in range(2))
    else:
        s["q"] = _rows(g, case["seqs"], case["heads"], hd, channels=False)
        s["out"] = torch.empty((case["seqs"], case["heads"], hd), device="cuda")
    return s


# ---------------------------------------------------- the framework's calls

@functools.lru_cache(maxsize=1)
def _ctx():
    import ggnpu_amd.lib as gl
    return gl.Context(torch.cuda.current_device())


@functools.lru_cache(maxsize=None)
def _rope_handle(head_dim, rot, layout, base, factors, yarn):
    import ggnpu_amd.lib as gl
    f = _factors(rot).tolist() if factors else None
    return gl.Rope(_ctx(), head_dim, rot, layout, base, freq_factors=f, yarn_factor=yarn, yarn_ctx=4096)


def _own(s):
    import ggnpu_amd.lib as gl
    case, ctx, stream = s["case"], _ctx(), torch.cuda.current_stream().cuda_stream
    hd, kind = case["head_dim"], case["kind"]
    if kind == "rope":
        h = _rope_handle(hd, case["rot"], case["layout"], case["base"], case["factors"], case["yarn"])
        sets = (gl.RopeHeads * 2)()
        for d, x, w, o in ((sets[0], "q", "qw", "q_out"), (sets[1], "k", "kw", "k_out")):
            n = s[x].shape[1]
            d.x, d.ldx, d.n_head, d.out, d.ldo, d.out_type = s[x].data_ptr(), n * hd, n, s[o].data_ptr(), n * hd, case["out"]
            d.norm_w = s[w].data_ptr() if case["norm"] else None
        ctx.check(ctx.lib.ggq_rope_dev(ctx.h, h.h, sets, 2, s["pos"].data_ptr(), case["tokens"], 1e-6, stream), "rope")
        return s["q_out"], s["k_out"]
    if kind == "prompt":
        kv = case["kv_heads"]
        p = gl.AttnPromptParams(type=case["type"], n_head=case["heads"], n_kv_head=kv, head_dim=hd,
                                q=s["q"].data_ptr(), ldq=case["heads"] * hd, k=s["k"].data_ptr(), ldk=kv * hd,
                                v=s["v"].data_ptr(), ldv=kv * hd, out=s["out"].data_ptr(), ldo=case["heads"] * hd,
                                n_rows=s["q"].shape[0], n_kv_rows=s["k"].shape[0], n_seq=case["seqs"],
                                q_off=s["q_off"].data_ptr(), kv_off=s["kv_off"].data_ptr(), window=case["window"])
        ctx.check(ctx.lib.ggq_attention_prompt_dev(ctx.h, p, stream), "prompt attention")
        return s["out"]
    cache = gl.KvCache(s["pages"].data_ptr(), s["pages"].shape[0], case["page"], case["kv_heads"], hd, case["k_type"], case["v_type"])
    longest = case["longest"] + case.get("before", 0)
    seqs = gl.KvSeqs(case["seqs"], s["table"].shape[1], longest, s["table"].data_ptr(), s["lens"].data_ptr())
    if kind == "decode":
        ld = case["heads"] * hd
        ctx.check(ctx.lib.ggq_attention_kv_dev(ctx.h, cache, seqs, s["q"].data_ptr(), ld, case["heads"], 0.0, case["window"],
                                               s["out"].data_ptr(), ld, stream), "cache attention")
        return s["out"]
    ld, rows = case["kv_heads"] * hd, s["k_out"].shape[0]
    if kind == "store":
        ctx.check(ctx.lib.ggq_kv_store_dev(ctx.h, cache, seqs, s["off"].data_ptr(), rows, s["k"].data_ptr(), ld,
                                           s["v"].data_ptr(), ld, case["type"], stream), "store")
    ctx.check(ctx.lib.ggq_kv_load_dev(ctx.h, cache, seqs, s["off"].data_ptr(), rows, s["k_out"].data_ptr(), ld,
                                      s["v_out"].data_ptr(), ld, case["type"], stream), "load")
    return s["k_out"], s["v_out"]


# ------------------------------------------------------------ the plain form

def _factors(rot):
    """Divisors of the frequencies, as a checkpoint for long contexts carries them: 1 for the fast ones, 8 for the
    slow ones, in between a passage."""
    i = torch.arange(rot // 2, dtype=torch.float64)
    return (1 + 7 * ((i / max(1, rot // 2 - 1) - 0.4) / 0.3).clamp(0, 1)).float()


def _frequencies(case):
    """Radians a position of each pair, in 64 bits, and the magnitude of cosine and sine."""
    rot, yarn = case["rot"], case["yarn"]
    i = torch.arange(rot // 2, dtype=torch.float64)
    f = case["base"] ** (-2.0 * i / rot)
    if case["factors"]:
        f = f / _factors(rot).double()
    if yarn <= 1.0:
        return f.cuda(), 1.0
    at = [rot * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(case["base"])) for turns in (32.0, 1.0)]
    low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rot - 1)
    ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
    return (f / yarn * ramp + f * (1 - ramp)).cuda(), 1.0 + 0.1 * math.log(yarn)


def _rotate(x, w, cos, sin, case):
    """Heads x [tokens, heads, head_dim], normalised where w is given, their first rot values turned."""
    if w is not None:
        x = x * (1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6)) * w
    rot, half = case["rot"], case["rot"] // 2
    a, b = (x[..., :half], x[..., half:rot]) if case["layout"] == HALF else (x[..., 0:rot:2], x[..., 1:rot:2])
    turned = (a * cos - b * sin, a * sin + b * cos)
    turned = torch.cat(turned, -1) if case["layout"] == HALF else torch.stack(turned, -1).flatten(-2)
    return torch.cat((turned, x[..., rot:]), -1).to(TORCH[case["out"]])


def _sees(row_pos, key_pos, window):
    m = key_pos <= row_pos
    return m & (key_pos > row_pos - window) if window else m


def _softmax(scores, sees):
    """Weights of the seen positions; a row that sees none has none."""
    scores = torch.where(sees, scores, -torch.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.where(sees, torch.exp(scores - torch.where(torch.isfinite(top), top, 0.0)), 0.0)
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total > 0, total, 1.0)


def run(state):
    if own:
        return _own(state)
    s, case = state, state["case"]
    kind, hd, kv = case["kind"], case["head_dim"], case["kv_heads"]
    if kind == "rope":
        angle = s["pos"].double()[:, None, None] * s["freq"]
        cos, sin = (torch.cos(angle) * s["mag"]).float(), (torch.sin(angle) * s["mag"]).float()
        return _rotate(s["q"], s["qw"], cos, sin, case), _rotate(s["k"], s["kw"], cos, sin, case)
    if kind == "store":
        return tuple(torch.ldexp(*_quantize(s[x], case[x + "_type"])).flatten(-2).to(TORCH[case["type"]]) for x in ("k", "v"))
    if kind == "prompt":
        heads, rows, keys = case["heads"], s["q"].shape[0], s["k"].shape[0]
        at = torch.arange(rows, device="cuda")
        seq = torch.bucketize(at, s["q_off"][1:], right=True)
        ends = s["kv_off"].long()[1:][seq]
        row_pos = ends - (s["q_off"].long()[1:][seq] - at)
        sees = _sees(row_pos[:, None], torch.arange(keys, device="cuda"), case["window"])
        sees &= torch.arange(keys, device="cuda") >= s["kv_off"].long()[seq][:, None]
        q = s["q"].view(rows, kv, heads // kv, hd).permute(1, 2, 0, 3).reshape(kv, -1, hd)
        k, v = (s[x].float().transpose(0, 1).contiguous() for x in ("k", "v"))
        scores = torch.matmul(q, k.transpose(1, 2).contiguous()).view(kv, heads // kv, rows, keys) / math.sqrt(hd)
        p = _softmax(scores, sees)
        o = torch.matmul(p.view(kv, -1, keys), v).view(kv, heads // kv, rows, hd)
        return o.permute(2, 0, 1, 3).reshape(rows, heads, hd)
    k, v = _read(case, s["pages"], s["table"])
    at = torch.arange(k.shape[1], device="cuda")
    if kind == "load":
        there = at < s["lens"][:, None]
        return k[there].to(TORCH[case["type"]]), v[there].to(TORCH[case["type"]])
    heads, n = case["heads"], case["seqs"]
    sees = _sees(s["lens"][:, None].long() - 1, at, case["window"])[:, None, None]
    q = s["q"].view(n, kv, heads // kv, hd)
    k, v = k.permute(0, 2, 3, 1).contiguous(), v.transpose(1, 2).contiguous()
    p = _softmax(torch.matmul(q, k) / math.sqrt(hd), sees)
    return torch.matmul(p, v).reshape(n, heads, hd)


# --------------------------------------------------------- in 64 bits, apart

def _exact_rope(case, s):
    rot, base = case["rot"], case["base"]
    freq = [base ** (-2.0 * i / rot) for i in range(rot // 2)]
    mag = 1.0
    if case["factors"]:
        freq = [f / d for f, d in zip(freq, _factors(rot).tolist())]
    if case["yarn"] > 1.0:
        # the pairs that turn 32 times and once over the 4096 positions trained on: kept as they are, or slowed down
        edge = [(rot / 2) * math.log(4096 / (2 * math.pi * t), base) for t in (32, 1)]
        lo, hi = max(0, math.floor(edge[0])), min(rot - 1, math.ceil(edge[1]))
        for i in range(rot // 2):
            keep = 1.0 - min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
            freq[i] *= keep + (1.0 - keep) / case["yarn"]
        mag += 0.1 * math.log(case["yarn"])
    turn = s["pos"].double()[:, None] * torch.tensor(freq, dtype=torch.float64, device="cuda")
    z = torch.polar(torch.full_like(turn, mag), turn)[:, None]
    outs = []
    for x, w in ((s["q"], s["qw"]), (s["k"], s["kw"])):
        x = x.double()
        if w is not None:
            x = x / (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
        y = x.clone()
        first, second = ((slice(0, rot // 2), slice(rot // 2, rot)) if case["layout"] == HALF
                         else (slice(0, rot, 2), slice(1, rot, 2)))
        c = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * z
        y[..., first], y[..., second] = c.real, c.imag
        outs.append(y)
    return tuple(outs)


def _exact_store(x, bits):
    """The nearest of all magnitudes that the format has, found in their sorted list; the even one of two as near."""
    if bits == 4:
        mags = torch.tensor(E2M1[:8], dtype=torch.float64, device="cuda")
        edge = 7.0
    else:
        mags = torch.arange(127, device="cuda").to(torch.uint8).view(torch.float8_e4m3fn).double()
        edge = 464.0
    b = x.double().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    scale = torch.full_like(top, 2.0 ** -126)
    for e in range(-126, 127):
        scale = torch.where(top > edge * 2.0 ** e, 2.0 ** (e + 1), scale)
    y = b.abs() / scale
    mid = (mags[1:] + mags[:-1]) / 2
    up = torch.bucketize(y, mid)  # a middle goes down here
    tie = (y == torch.cat((mid, mid.new_full((1,), torch.inf)))[up]) & (up % 2 == 1)
    return (mags[(up + tie.long()).clamp(max=len(mags) - 1)] * scale * b.sign()).flatten(-2)


def _exact_attention(q, k, v, first, window):
    """q [rows, heads, hd], k and v [positions, kv heads, hd]; row i sits at position first + i."""
    rows, heads, hd = q.shape
    out = torch.zeros((rows, heads, hd), dtype=torch.float64, device="cuda")
    group = heads // k.shape[1]
    i = first + torch.arange(rows, device="cuda")[:, None]
    j = torch.arange(k.shape[0], device="cuda")
    hidden = (j > i) | (j <= i - window if window else torch.zeros_like(j > i))
    for h in range(heads):
        x = (q[:, h].double() @ k[:, h // group].double().T.contiguous()) * hd ** -0.5
        out[:, h] = torch.softmax(x.masked_fill(hidden, -torch.inf), -1) @ v[:, h // group].double()
    return out


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "rope":
        return _exact_rope(case, s)
    if kind == "store":
        return _exact_store(s["k"], case["k_type"]), _exact_store(s["v"], case["v_type"])
    lengths = _lengths(case)
    if kind == "prompt":
        a, b = _starts(lengths), s["kv_off"].tolist()
        return torch.cat([_exact_attention(s["q"][a[i]:a[i + 1]], s["k"][b[i]:b[i + 1]], s["v"][b[i]:b[i + 1]],
                                           case["before"], case["window"]) for i in range(case["seqs"])])
    # record by record and position by position: the byte that holds a value, by the format's definition
    hd, kv, page, (a, b, c, d, size) = case["head_dim"], case["kv_heads"], case["page"], _record(case)
    p, e = torch.arange(TILE, device="cuda")[:, None], torch.arange(hd, device="cuda")

    def values(rec, at, scales_at, bits, value):
        g, r = ((p % 16) // 4, e // (hd // 16)) if value else (e // (hd // 4), p % 16)
        n = ((p // 16) * 4 + p % 4) * (hd // 16) + e % (hd // 16) if value else (p // 16) * (hd // 4) + e % (hd // 4)
        byte = n * bits // 8
        byte = byte // 16 * 1024 + (16 * g + r) * 16 + byte % 16
        code = rec[:, (at + byte).flatten()].view(-1, TILE, hd)
        if bits == 4:
            code = torch.where(n % 2 == 1, code >> 4, code & 15)
            v = torch.tensor(E2M1, dtype=torch.float64, device="cuda")[code.long()]
        else:
            v = code.view(torch.float8_e4m3fn).double()
        blk = e // 32
        where = (blk * 4 + g) * 8 + (p // 16) * 4 + p % 4 if value else (blk * 16 + r) * 2 + p // 16
        sc = rec[:, (scales_at + where.expand(TILE, hd)).flatten()].view(-1, TILE, hd)
        return v * torch.exp2(sc.double() - 127)

    outs = []
    for i, n in enumerate(lengths):
        rec = s["pages"][s["table"][i].long()].view(-1, kv, page // TILE, size)
        kk, vv = (values(rec.reshape(-1, size), *w).view(-1, kv, page, hd).transpose(1, 2).reshape(-1, kv, hd)[:n]
                  for w in ((a, c, case["k_type"], False), (b, d, case["v_type"], True)))
        outs.append((kk, vv) if kind == "load"
                    else _exact_attention(s["q"][i:i + 1], kk, vv, n - 1, case["window"]))
    return tuple(torch.cat(x) for x in zip(*outs)) if kind == "load" else torch.cat(outs)
