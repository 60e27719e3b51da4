"""Captured attention over the 8-bit key/value cache: every route, compared bit for bit with the eager call."""
import numpy as np
import pytest

from test_gpu_kv import Batch, dev, starts_of

pytestmark = pytest.mark.gpu

CASES = [
    # lens, rows per sequence, heads, kv heads, D
    ([700], [640], 16, 16, 64),       # a prompt whose tiles fill the SMs: no key splits, no scratch
    ([900, 70], [40, 9], 4, 2, 128),  # key splits, joined by a second kernel
    ([300, 33], [5, 3], 8, 2, 80),    # 17 to 32 pairs: split keys, two tiles
    ([2000], [1], 28, 4, 128),        # a single token
]


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_captured_attention(pxq, case, weights):
    import torch

    lens, ns, heads, H, D = CASES[case]
    rng = np.random.default_rng(case)
    b = Batch(pxq, rng, lens, H, D)
    starts, n = starts_of(ns), sum(ns)
    qs = [dev(rng.standard_normal((n, heads * D)).astype(np.float32)) for _ in range(3)]
    q, out = torch.zeros_like(qs[0]), torch.zeros_like(qs[0])
    w = torch.zeros((len(lens), H, b.cap), device="cuda") if weights else None

    def call():
        pxq.kv_attention(q, b.cache, heads, starts=starts, max_rows=max(ns), out=out, weights_out=w)

    want = []
    for x in qs:
        q.copy_(x)
        call()
        want.append((out.clone(), w.clone() if weights else None))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for x, (o, wt) in zip(qs, want):
        q.copy_(x)
        out.fill_(-1)
        graph.replay()
        pxq.synchronize()
        assert torch.equal(out, o)
        if weights:
            assert torch.equal(w, wt)
    del graph


def test_captured_eviction(pxq):
    """With the places of the kept tokens in scratch of the call's own."""
    import torch

    rng = np.random.default_rng(9)
    b = Batch(pxq, rng, [300, 90], 2, 64)
    spare, other = pxq.KVCache(2, 100, 2, 64), pxq.KVCache(2, 100, 2, 64)
    w = dev(rng.uniform(0, 1, (2, 2, b.cap)).astype(np.float32))
    pxq.kv_evict(b.cache, other, w, recent=10)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pxq.kv_evict(b.cache, spare, w, recent=10)
    for _ in range(2):
        spare.truncate()
        graph.replay()
        pxq.synchronize()
        for got, want in zip(spare.read(), other.read()):
            assert torch.equal(got, want)
    del graph
