"""The attention operators without a GPU: page sizes, refusals of a null context, and the plain forms that the GPU tests
compare with."""
import ctypes

import numpy as np
import pytest

import ggnpu_amd.lib as gl
from tests import attn_util as au


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("kt,vt", [(4, 4), (8, 4), (4, 8), (8, 8)])
def test_page_bytes(hd, kt, vt):
    """4.25 and 8.25 bits a value."""
    lib = gl.load_library()
    c = gl.KvCache(None, 0, 96, 3, hd, kt, vt)
    want = 3 * 96 * hd * ((kt + 0.25) + (vt + 0.25)) / 8
    assert lib.ggq_kv_page_bytes(ctypes.byref(c)) == want == 3 * 3 * au.kv_record(hd, kt, vt)[-1]


@pytest.mark.parametrize("kw", [dict(page_len=0), dict(page_len=-32), dict(page_len=33), dict(n_kv_head=0), dict(n_kv_head=40000),
                                dict(head_dim=80), dict(head_dim=0), dict(k_type=0), dict(v_type=16)])
def test_page_bytes_of_what_is_not_supported(kw):
    d = dict(page_len=64, n_kv_head=2, head_dim=64, k_type=4, v_type=8)
    d.update(kw)
    assert gl.load_library().ggq_kv_page_bytes(ctypes.byref(gl.KvCache(**d))) == 0
    assert gl.load_library().ggq_kv_page_bytes(None) == 0


def test_null_context():
    lib, bad, out = gl.load_library(), gl.Status.INVALID_PARAM, ctypes.c_void_p()
    assert lib.ggq_rope_create(None, ctypes.byref(gl.RopeParams(head_dim=64)), ctypes.byref(out)) == bad
    assert lib.ggq_rope_free(None, None) == bad
    assert lib.ggq_rope_dev(None, None, None, 1, None, 1, 1e-6, None) == bad
    c, q = gl.KvCache(), gl.KvSeqs()
    assert lib.ggq_kv_store_dev(None, c, q, None, 1, None, 64, None, 64, 0, None) == bad
    assert lib.ggq_kv_load_dev(None, c, q, None, 1, None, 64, None, 64, 0, None) == bad
    assert lib.ggq_attention_kv_dev(None, c, q, None, 64, 1, 0.0, 0, None, 64, None) == bad
    assert lib.ggq_attention_prompt_dev(None, gl.AttnPromptParams(), None) == bad


@pytest.mark.parametrize("bits", [4, 8])
def test_plain_quantizer_takes_the_nearest_code(bits):
    """Against a search over all codes at the scale it chose, and over all smaller scales: none is allowed."""
    rng = np.random.default_rng(bits)
    mags, edge = (au.E2M1, 7.0) if bits == 4 else (au.E4M3, 464.0)
    x = (rng.standard_normal((64, 64)) * np.exp2(rng.integers(-100, 90, (64, 2))).repeat(32, -1)).astype(np.float32).astype(np.float64)
    v, codes, scales = au.kv_quantize(x, bits)
    s = np.exp2(scales.astype(float) - 127).repeat(32, -1)
    best = np.abs(np.abs(x)[..., None] / s[..., None] - mags).min(-1)
    assert np.array_equal(np.abs(np.abs(x) / s - np.abs(v) / s), best)
    top = np.abs(x).reshape(64, 2, 32).max(-1)
    least = np.exp2(scales.astype(float) - 127)
    assert (top <= edge * least).all() and (top > edge * least / 2).all()
    assert np.array_equal(au.kv_values(codes, scales, bits), v)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("kt,vt", [(4, 8), (8, 4)])
def test_plain_layout_holds_every_value_once(hd, kt, vt):
    rng = np.random.default_rng(hd)
    k, v = rng.standard_normal((3, 64, 2, hd)), rng.standard_normal((3, 64, 2, hd))
    pages = au.kv_pack(k, v, 2, 64, kt, vt)
    for got, x, bits in zip(au.kv_unpack(pages, 2, 64, hd, kt, vt), (k, v), (kt, vt)):
        assert np.array_equal(got, au.kv_quantize(x, bits)[0])
    for bits, value in ((kt, False), (vt, True)):
        byte, half, scale = au.kv_places(hd, bits, value)
        assert len(set(zip(byte.ravel().tolist(), (half * (bits == 4)).ravel().tolist()))) == 32 * hd
        assert byte.max() == 32 * hd * bits // 8 - 1 and sorted(scale.ravel().tolist()) == list(range(hd))


def test_plain_attention_of_one_and_of_none():
    q, k, v = np.ones((2, 2, 64)), np.ones((1, 1, 64)), np.arange(64.0).reshape(1, 1, 64)
    out, tol = au.attention(q, k, v, -1)  # the first row sees nothing, the second one key
    assert (out[0] == 0).all() and np.allclose(out[1], np.arange(64.0)) and (tol >= 0).all()
