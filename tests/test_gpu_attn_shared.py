"""The attention operators where calls could meet: captured and eager calls that need workspace in flight together."""
import numpy as np
import pytest

import ggnpu_amd.lib as gl
from tests import attn_util as au
from tests.gpu_util import host
from tests.test_gpu_attn_prompt import t
from tests.test_gpu_attn_together import Layer, _buffers, stream

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import torch
    assert torch.cuda.is_available()
    c = gl.Context(0)
    yield c
    c.close()


def _generator(seed):
    import torch
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


def _prompt_of(lay, rows, gen):
    """Buffers of a prompt whose offsets split it in two."""
    import torch
    q, k, v = (torch.randn((rows, h, lay.hd), device="cuda", generator=gen) for h in (lay.n_head, lay.n_kv, lay.n_kv))
    return q, k, v, torch.empty_like(q), t(np.array([0, rows // 3, rows], np.int32))


@pytest.mark.parametrize("hd", [64, 256])
def test_graphs_and_streams_with_planes_and_parts(ctx, monkeypatch, hd):
    """Two captured and two eager pairs of calls, each on a stream of its own and all in flight together; every prompt
    goes through planes and every cache call through parts, so that a shared buffer would show."""
    import torch
    monkeypatch.setenv("GGQ_PROMPT_MFMA", "1")
    monkeypatch.setenv("GGQ_KV_SPLITS", "9")
    gen = _generator(50)
    lays = [Layer(ctx, 1, 1, 4096, 8, 2, hd, 4, 8, seed=i) for i in range(4)]
    bufs = [_buffers(x, 1, 60 + i) for i, x in enumerate(lays)]
    prompts = [_prompt_of(x, 400 + 90 * i, gen) for i, x in enumerate(lays)]
    for x in lays:
        k, v = (torch.randn((4000, 2, hd), device="cuda", generator=gen) for _ in range(2))
        x.len.fill_(4000)
        x.store(k, v, t(np.array([0, 4000], np.int32)), stream())

    def work(i, s):
        q, k, v, out, off = prompts[i]
        lays[i].prompt(q, k, v, out, off, off, s)
        lays[i].decode(bufs[i]["q"], bufs[i]["out"], s)
        lays[i].prompt(q, k, v, out, off, off, s)
    want = []
    for i in range(4):
        work(i, stream())
        torch.cuda.synchronize()
        want.append((bufs[i]["out"].clone(), prompts[i][3].clone()))
    q, k, v, _, _ = prompts[3]
    n = q.shape[0]
    for r in (0, n // 3 - 1):
        w, tol = au.attention(host(q)[r:r + 1], host(k), host(v), r)
        au.check(host(want[3][1])[r:r + 1], w, tol)
    streams = [torch.cuda.Stream() for _ in range(4)]
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for i in range(2):
        with torch.cuda.graph(graphs[i], stream=streams[i]):
            work(i, streams[i].cuda_stream)
    for _ in range(6):
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
