"""Host threads that share a stream: calls of several kernels over scratch of the stream's (decode attention and its join,
eviction, the matvec's quantize step and product) keep together, so each thread gets what it would get alone."""
import threading

import numpy as np
import pytest

from pixelina_b200 import synth
from test_gpu_kv import dev, rows_of

pytestmark = pytest.mark.gpu


def together(workers, rounds=200):
    """Runs work(i) of every worker, i < rounds, each in a thread of its own, all at once."""
    failed, gate = [], threading.Barrier(len(workers))

    def run(work):
        try:
            gate.wait()
            for i in range(rounds):
                work(i)
        except BaseException as e:  # noqa: BLE001 (handed to the test's own thread)
            failed.append(e)

    threads = [threading.Thread(target=run, args=(w,)) for w in workers]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    if failed:
        raise failed[0]


class Chat:
    """A cache, queries and outputs of a thread's own; step i answers rows of its i-th query."""

    KEEP = 8  # outputs kept, in turn

    def __init__(self, pxq, seed, lens, heads, H, D, n, weights, stream=None):
        import torch

        rng = np.random.default_rng(seed)
        self.pxq, self.heads, self.stream = pxq, heads, stream
        S = len(lens)
        self.cache = pxq.KVCache(S, max(lens), H, D)
        starts = dev(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32))
        x = rows_of(rng, sum(lens), H, D).reshape(sum(lens), -1)
        self.cache.append(dev(x), dev(x[::-1].copy()), starts=starts)
        self.spare = pxq.KVCache(S, max(lens), H, D)
        self.q = dev(rng.standard_normal((self.KEEP, S * n, heads * D)).astype(np.float32))
        self.out = torch.zeros_like(self.q)
        self.w = torch.zeros((self.KEEP, S, H, max(lens)), device="cuda") if weights else None
        self.moved = torch.zeros_like(self.w) if weights else None
        self.keep = max(1, min(lens) // 2)

    def step(self, i):
        j = i % self.KEEP
        self.pxq.kv_attention(self.q[j], self.cache, self.heads, out=self.out[j], weights_out=None if self.w is None else self.w[j], stream=self.stream)
        if self.w is not None:
            self.pxq.kv_evict(self.cache, self.spare, self.w[j], keep=self.keep, weights_out=self.moved[j], stream=self.stream)

    def clear(self):
        for x in (self.out, self.w, self.moved):
            if x is not None:
                x.zero_()

    def results(self):
        return [x.clone() for x in (self.out, self.w, self.moved) if x is not None]


def chats(pxq, streams=(None, None, None)):
    return [Chat(pxq, 1, [900, 700], 28, 4, 128, 1, False, streams[0]), Chat(pxq, 2, [1500, 40], 8, 8, 64, 1, True, streams[1]),
            Chat(pxq, 3, [400], 4, 1, 80, 30, True, streams[2])]


def test_threads_on_one_stream(pxq):
    import torch

    mine = chats(pxq)
    for c in mine:
        for i in range(Chat.KEEP):
            c.step(i)
    pxq.synchronize()
    want = [c.results() for c in mine]
    for c in mine:
        c.clear()
    torch.cuda.synchronize()
    together([c.step for c in mine])
    pxq.synchronize()
    for c, w in zip(mine, want):
        assert all(torch.equal(got, x) for got, x in zip(c.results(), w))


def test_the_per_thread_stream(pxq):
    """cudaStreamPerThread is one handle for as many streams as there are threads, so its calls have scratch of their own; here
    from one thread, the results those of the default stream."""
    import torch

    per_thread = torch.cuda.ExternalStream(2)
    results = []
    for stream in (None, per_thread):
        mine = chats(pxq, (stream,) * 3)
        torch.cuda.synchronize()
        for c in mine:
            for i in range(Chat.KEEP):
                c.step(i)
        torch.cuda.synchronize()
        results.append([x for c in mine for x in c.results()])
    assert all(torch.equal(a, b) for a, b in zip(*results))
    W = pxq.Weight(synth.random_q5_K(200, 2048, np.random.default_rng(1)), 13, 2048, 200)
    x = dev(synth.activations(8, 2048, seed=6))
    torch.cuda.synchronize()
    with torch.cuda.stream(per_thread):
        got = [pxq.matmul(W, x) for _ in range(4)]
        per_thread.synchronize()
    want = pxq.matmul(W, x)
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    W.release()


def test_threads_share_a_stream_with_older_calls(pxq):
    """fp32 attention with split keys and matvecs (with and without a quantize step) beside the cache's attention."""
    import torch

    rng = np.random.default_rng(5)
    heads, H, D, t = 28, 4, 128, 2000
    q, k, v = (dev(rng.standard_normal(s).astype(np.float32)) for s in ((2, heads * D), (t, H * D), (t, H * D)))
    weights = [pxq.Weight(synth.random_q5_K(200, inner, np.random.default_rng(inner)), 13, inner, 200) for inner in (18944, 2048)]
    x = [dev(synth.activations(cols, w.inner, seed=6)) for w, cols in zip(weights, (1, 8))]
    chat = chats(pxq)[0]
    outs = [torch.zeros((2, heads * D), device="cuda")] + [None, None]

    def attention(i):
        outs[0] = pxq.attention(q, k, v, heads, H)

    def matvec(at):
        def f(i):
            outs[1 + at] = pxq.matmul(weights[at], x[at])
        return f

    work = [attention, matvec(0), matvec(1), chat.step]
    for f in work:
        for i in range(Chat.KEEP):
            f(i)
    pxq.synchronize()
    want = [o.clone() for o in outs] + [chat.out.clone()]
    chat.clear()
    torch.cuda.synchronize()
    together(work, rounds=400)
    pxq.synchronize()
    for got, w in zip(outs + [chat.out], want):
        assert torch.equal(got, w)
    for w in weights:
        w.release()
