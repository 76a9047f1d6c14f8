"""The operators around a layer's matmuls without a GPU: refusals of a null context, and the plain forms that the GPU tests
compare with."""
import ctypes

import numpy as np
import pytest

import ggnpu_amd.lib as gl
from tests import step_util as su


def test_null_context():
    lib, bad = gl.load_library(), gl.Status.INVALID_PARAM
    assert lib.ggq_attention_kv_rows_dev(None, gl.KvCache(), gl.KvSeqs(), None, 1, None, 64, 1, 0.0, 0, None, 64, None) == bad
    assert lib.ggq_delta_rule_dev(None, gl.DeltaRuleParams(), None) == bad
    assert lib.ggq_norm_dev(None, gl.NormParams(), None) == bad
    assert lib.ggq_sample_dev(None, gl.SampleParams(), None) == bad


def test_struct_sizes():
    """The layouts that a C compiler gives the structs of include/ggq.h (checked by their sizes)."""
    assert ctypes.sizeof(gl.DeltaRuleParams) == 192
    assert ctypes.sizeof(gl.NormParams) == 128
    assert ctypes.sizeof(gl.SampleParams) == 80


def test_plain_delta_rule_is_a_projection_when_nothing_decays():
    """b = 1 and unit keys: after a row the state gives the row's value for its key, whatever it held."""
    rng = np.random.default_rng(1)
    k = rng.standard_normal((5, 1, 64))
    k /= np.linalg.norm(k, axis=-1, keepdims=True)
    v = rng.standard_normal((5, 2, 16))
    S0 = rng.standard_normal((2, 16, 64))
    for n in (1, 5):
        out, S, _, _ = su.delta(k[:n], k[:n], v[:n], np.zeros((n, 2)), np.ones((n, 2)), S0, scale=1.0)
        assert np.allclose(np.einsum("hvk,k->hv", S, k[n - 1, 0]), v[n - 1]) and np.allclose(out[n - 1], v[n - 1])


def test_plain_delta_rule_against_differences():
    """out's derivative by b of a row, from the recurrence by hand, against a difference quotient."""
    rng = np.random.default_rng(2)
    k, q = (rng.standard_normal((1, 1, 64)) / 8 for _ in range(2))
    v, S0, g, b = rng.standard_normal((1, 1, 16)), rng.standard_normal((1, 16, 64)), np.full((1, 1), -0.3), np.full((1, 1), 0.7)
    d = 1e-6
    f = lambda bb: su.delta(q, k, v, g, bb, S0, scale=1.0)[0][0, 0]  # noqa: E731
    by_hand = (v[0, 0] - np.exp(-0.3) * S0[0] @ k[0, 0]) * (k[0, 0] @ q[0, 0])
    assert np.allclose((f(b + d) - f(b - d)) / (2 * d), by_hand, rtol=1e-6, atol=1e-8)


@pytest.mark.parametrize("kw,kept", [(dict(), 6), (dict(top_k=2), 2), (dict(top_p=0.5), 2), (dict(top_p=0.3), 1), (dict(top_p=0.0), 1), (dict(min_p=1.0), 2),
                                     (dict(min_p=2.0), 2), (dict(top_k=1), 1), (dict(top_k=99), 6)])
def test_plain_sampling_keeps(kw, kept):
    x = np.array([1.0, -np.inf, 3.0, 0.5, 3.0, np.nan, -1.0, 2.0], np.float32)
    seen = {su.sample(x, 1.0, u=u, **kw)[0] for u in np.linspace(0, 0.999999, 4001)}
    assert len(seen) == kept and (1 not in seen) and (5 not in seen) and 2 in seen


def test_plain_sampling_of_nothing_and_greedy():
    assert su.sample(np.full(4, -np.inf, np.float32))[:2] == (0, 0.0)
    assert su.sample(np.array([0, 7, 7], np.float32), 0.0, u=0.9)[:2] == (1, 1.0)
    assert su.sample(np.array([0, np.inf, 7, np.inf], np.float32), 1.0, u=0.6)[:2] == (3, 0.5)


def test_plain_codes():
    y = np.array([[0, 0, 0, 0], [1, -2, 0.5, 2]], np.float32)
    q, sc = su.codes(y)
    assert (q[0] == 0).all() and sc[0, 0] == 1 and sc[1, 0] == np.float32(2) / np.float32(127) and q[1].tolist() == [64, -127, 32, 127]
