"""The 8-bit key/value cache over the sizes that its interface promises: up to 1024 sequences, capacities far above the
lengths, prompts beside single tokens, long evictions.  References and tolerances as in test_gpu_kv.py."""
import numpy as np
import pytest

import kv_reference as ref
from conftest import max_abs_rel
from test_gpu_kv import ATT_TOL, Batch, dev, i32, rows_of, starts_of

pytestmark = pytest.mark.gpu


def check_attention(pxq, b, ns, heads, causal, rng, max_rows=None):
    """Outputs and weights of one call against 64 bits, sequence by sequence; entries that are nobody's stay."""
    import torch

    S, D = len(b.k), b.D
    q = (1.5 * rng.standard_normal((sum(ns) + 1, heads, D))).astype(np.float32)
    w0 = rng.uniform(0, 2, (S, b.H, b.cap)).astype(np.float32)
    w = torch.full(w0.shape, -3.0, device="cuda")
    out = torch.full((len(q), heads * D), 9.0, device="cuda")
    pxq.kv_attention(dev(q.reshape(len(q), -1)), b.cache, heads, starts=starts_of(ns), max_rows=max_rows, causal=causal, out=out,
                     weights=dev(w0), weights_out=w)
    plain = torch.full_like(out, 9.0)
    pxq.kv_attention(dev(q.reshape(len(q), -1)), b.cache, heads, starts=starts_of(ns), max_rows=max_rows, causal=causal, out=plain)
    pxq.synchronize()
    assert torch.equal(out, plain) and bool((out[-1] == 9).all())
    got, w, at = out.cpu().numpy().reshape(-1, heads, D), w.cpu().numpy(), 0
    for s, n in enumerate(ns):
        t = len(b.k[s])
        want, wt = ref.attention(q[at:at + n], ref.values(b.k[s]), ref.values(b.v[s]), heads, causal)
        if n:
            assert max_abs_rel(got[at:at + n], want) <= ATT_TOL, s
        if t:
            assert max_abs_rel(w[s, :, :t], wt + w0[s, :, :t]) <= ATT_TOL, s
        assert (w[s, :, t:] == -3).all(), s
        at += n


def many(rng, S, longest):
    """Lengths of S sequences: every fifth empty, a few long ones."""
    lens = rng.integers(1, 100, S)
    lens[::5] = 0
    lens[rng.choice(S, 3, replace=False)] = longest
    return [int(x) for x in lens]


@pytest.mark.parametrize("S", [33, 200, 1024])
@pytest.mark.parametrize("kind", ["decode", "decode G", "rows", "chunks"])
def test_many_sequences(pxq, S, kind):
    """Empty sequences and sequences without rows among them; with so many the single tokens' blocks are divided as one list,
    several (sequence, head)s to a CTA."""
    rng = np.random.default_rng(S)
    lens = many(rng, S, 700)
    b = Batch(pxq, rng, lens, 2, 64)
    b.check()
    ns = {"decode": rng.integers(0, 2, S), "decode G": rng.integers(0, 2, S), "rows": rng.integers(0, 4, S), "chunks": rng.integers(0, 30, S)}[kind]
    ns = [int(x) for x in ns]
    check_attention(pxq, b, ns, 14 if kind == "decode G" else 4, kind != "chunks", rng, max_rows=max(ns))


@pytest.mark.parametrize("S", [33, 1024])
def test_many_sequences_appended_to_and_shortened(pxq, S):
    rng = np.random.default_rng(S + 1)
    H, D = 1, 80
    b = Batch(pxq, rng, many(rng, S, 300), H, D, cap=340)
    ns = rng.integers(0, 3, S)
    ns[7] = 40
    new = [rows_of(rng, int(n), H, D) for n in ns]
    x = dev(np.concatenate(new).reshape(-1, H * D))
    b.cache.append(x, x, starts=starts_of(ns))
    b.k, b.v = ([np.concatenate([y, n]) for y, n in zip(z, new)] for z in (b.k, b.v))
    b.check()
    # within each open block, where nothing is lost
    to = [len(y) if len(y) % 32 == 0 else len(y) - int(rng.integers(0, len(y) % 32)) for y in b.k]
    b.cache.truncate(i32(to))
    b.k, b.v = ([y[:n] for y, n in zip(z, to)] for z in (b.k, b.v))
    b.check()
    pxq.synchronize()


def test_many_sequences_evicted(pxq):
    rng = np.random.default_rng(3)
    S, H, D, keep = 200, 2, 64, 40
    lens = many(rng, S, 200)
    b = Batch(pxq, rng, lens, H, D)
    w = (rng.integers(0, 30, (S, H, b.cap)) / 8).astype(np.float32)
    dst = pxq.KVCache(S, keep, H, D)
    pxq.kv_evict(b.cache, dst, dev(w), keep=keep, recent=8)
    pxq.synchronize()
    assert dst.lengths().cpu().tolist() == [min(t, keep) for t in lens]
    k, v = (x.cpu().numpy().reshape(S, keep, H, D) for x in dst.read())
    for s, t in enumerate(lens):
        kv, vv, c = ref.values(b.k[s]), ref.values(b.v[s]), min(t, keep)
        for h in range(H):
            at = ref.kept(w[s, h, :t], keep, 8)
            assert np.array_equal(k[s, :c, h:h + 1], ref.values(kv[at, h:h + 1])) and np.array_equal(v[s, :c, h:h + 1], ref.values(vv[at, h:h + 1]))


@pytest.mark.parametrize("G", [1, 7])
def test_prompts_beside_single_tokens(pxq, G):
    """Single tokens over long caches, a prompt, a short chunk and a sequence without rows in one call."""
    rng = np.random.default_rng(G)
    b = Batch(pxq, rng, [9000, 300, 40, 4000, 65], 2, 128)
    check_attention(pxq, b, [1, 200, 0, 1, 17], 2 * G, True, rng, max_rows=200)


@pytest.mark.parametrize("ns,G", [([1, 1], 4), ([2, 1], 12), ([40, 3], 1)])
def test_a_capacity_far_above_the_lengths(pxq, ns, G):
    """The routes and grids go by the capacity; what is done goes by the lengths."""
    rng = np.random.default_rng(12)
    b = Batch(pxq, rng, [90, 33], 2, 64, cap=150_000)
    check_attention(pxq, b, ns, 2 * G, True, rng, max_rows=max(ns))


def test_starts_without_max_rows(pxq):
    """A decode step whose most rows per sequence are not told: planned as if one sequence had them all."""
    rng = np.random.default_rng(13)
    b = Batch(pxq, rng, [500, 31, 1, 0, 64, 90, 700, 2], 2, 128)
    check_attention(pxq, b, [1] * 8, 14, True, rng)


@pytest.mark.parametrize("rows,group", [(2, 1), (5, 1), (8, 1), (3, 4), (4, 4), (5, 4), (8, 4), (40, 1)])
def test_rows_that_do_not_see_a_block_that_is_not_finite(pxq, rows, group):
    """The last token alone opens a block and is not finite, in K or in V or in both: the last row is NaN, the others are
    what they are without it; and so are the weights once it is taken back."""
    import torch

    H, D, t = 3, 64, 32 * 9 + 1
    rng = np.random.default_rng(rows)
    for bad_k, bad_v in ((np.nan, None), (None, np.inf), (-np.inf, np.nan)):
        k, v = rows_of(rng, t, H, D), rows_of(rng, t, H, D)
        kv, vv = ref.values(k[:-1]), ref.values(v[:-1])
        if bad_k is not None:
            k[-1, :, 5] = bad_k
        if bad_v is not None:
            v[-1, :, 6] = bad_v
        cache = pxq.KVCache(1, t + 70, H, D)
        cache.memory[256 + 12 + 244:].fill_(255)  # everything but the zeroed head: scales NaN, codes 127
        cache.append(dev(k.reshape(t, -1)), dev(v.reshape(t, -1)))
        q = rng.standard_normal((rows, H * group, D)).astype(np.float32)
        got = pxq.kv_attention(dev(q.reshape(rows, -1)), cache, H * group).cpu().numpy().reshape(rows, H * group, D)
        assert np.isnan(got[-1]).all()
        for i in range(rows - 1):
            lim = t - rows + i + 1
            want, _ = ref.attention(q[i:i + 1], kv[:lim], vv[:lim], H * group, False)
            assert max_abs_rel(got[i:i + 1], want) <= ATT_TOL, i
        cache.truncate(i32([t - 1]))
        w = torch.zeros((1, H, t + 70), device="cuda")
        got = pxq.kv_attention(dev(q[:-1].reshape(rows - 1, -1)), cache, H * group, weights_out=w).cpu().numpy()
        want, wt = ref.attention(q[:-1], kv, vv, H * group, True)
        assert max_abs_rel(got.reshape(want.shape), want) <= ATT_TOL
        assert max_abs_rel(w[0, :, :t - 1].cpu().numpy(), wt) <= ATT_TOL and not w[0, :, t - 1:].any()
    pxq.synchronize()


@pytest.mark.parametrize("keep,recent", [(30_000, 5), (55_000, 0), (4, 4), (52_000, 52_000)])
def test_evict_from_more_tokens_than_shared_memory_holds(pxq, keep, recent):
    """60000 tokens, the weights' order kept in shared memory for the first 51200; ties on both sides of that border."""
    import torch

    rng = np.random.default_rng(keep)
    H, D, t = 2, 64, 60_000
    b = Batch(pxq, rng, [t], H, D)
    w = (rng.integers(0, 40, (1, H, t)) / 16).astype(np.float32)
    w[0, 0, rng.choice(t, 50, replace=False)] = np.nan
    dst = pxq.KVCache(1, keep, H, D)
    kept = torch.full((1, H, keep), -1, dtype=torch.int32, device="cuda")
    wo = torch.zeros((1, H, keep), device="cuda")
    pxq.kv_evict(b.cache, dst, dev(w), keep=keep, recent=recent, kept=kept, weights_out=wo)
    pxq.synchronize()
    k, v = (x.cpu().numpy().reshape(keep, H, D) for x in dst.read())
    sk, sv = (x.cpu().numpy().reshape(t, H, D) for x in b.cache.read())
    for h in range(H):
        at = ref.kept(w[0, h], keep, recent)
        assert np.array_equal(kept[0, h].cpu().numpy(), at)
        assert np.array_equal(wo[0, h].cpu().numpy(), w[0, h, at], equal_nan=True)
        assert np.array_equal(k[:, h:h + 1], ref.values(sk[at, h:h + 1])) and np.array_equal(v[:, h:h + 1], ref.values(sv[at, h:h + 1]))


@pytest.mark.parametrize("causal", [False, True])
def test_weights_whose_partial_sums_take_several_passes(pxq, causal):
    """A capacity of 2^19 tokens and 8 heads: 16 MB of partial sums per tile of 128 rows, 256 MB at a time; the border
    between two passes falls into the second sequence."""
    import torch

    rng = np.random.default_rng(21)
    lens, ns, H, D, cap = [300, 500], [1200, 1000], 8, 64, 1 << 19
    b = Batch(pxq, rng, lens, H, D, cap=cap)
    q = rng.standard_normal((sum(ns), H, D)).astype(np.float32)
    w0 = rng.uniform(0, 2, (2, H, 600)).astype(np.float32)
    w = torch.zeros((2, H, cap), device="cuda")
    w[:, :, :600] = dev(w0)
    out = pxq.kv_attention(dev(q.reshape(len(q), -1)), b.cache, H, starts=starts_of(ns), max_rows=max(ns), causal=causal, weights=w, weights_out=w)
    pxq.synchronize()
    got, at = out.cpu().numpy().reshape(-1, H, D), 0
    for s, (t, n) in enumerate(zip(lens, ns)):
        want, wt = ref.attention(q[at:at + n], ref.values(b.k[s]), ref.values(b.v[s]), H, causal)
        assert max_abs_rel(got[at:at + n], want) <= ATT_TOL
        assert max_abs_rel(w[s, :, :t].cpu().numpy(), wt + w0[s, :, :t]) <= ATT_TOL
        assert np.array_equal(w[s, :, t:600].cpu().numpy(), w0[s, :, t:])
        at += n


def test_a_token_taken_back_and_appended_again(pxq):
    """Leaves lengths, scales and codes as they were, at a block's border too."""
    H, D = 2, 128
    for t in (31, 32, 33, 64, 65, 97):
        b = Batch(pxq, np.random.default_rng(t), [t], H, D)
        nb = -(-t // 32)
        codes, scales = H * nb * 64 * D, H * nb * 8
        before = b.cache.memory.clone()
        b.cache.truncate(i32([t - 1]))
        b.cache.append(dev(b.k[0][-1:].reshape(1, -1)), dev(b.v[0][-1:].reshape(1, -1)))
        after = b.cache.memory
        assert bool((before[:512 + scales] == after[:512 + scales]).all()) and bool((before[-codes:] == after[-codes:]).all())
    pxq.synchronize()


def test_drafts_taken_back_with_their_weights(pxq):
    """A rejected draft: the cache shortened and the dropped tokens' running totals set to zero, as the interface asks; later
    steps then add up to what they would without the draft."""
    import torch

    rng = np.random.default_rng(31)
    H, D, heads, t, cap = 2, 64, 8, 50, 80
    x = [dev(rows_of(rng, n, H, D).reshape(n, -1)) for n in (t, 5, 3)]
    qs = [dev(rng.standard_normal((n, heads * D)).astype(np.float32)) for n in (1, 5, 3)]
    totals = []
    for draft in (False, True):
        cache, w = pxq.KVCache(1, cap, H, D), torch.zeros((1, H, cap), device="cuda")
        cache.append(x[0], x[0])
        pxq.kv_attention(qs[0], cache, heads, weights=w, weights_out=w)
        if draft:
            seen = w.clone()
            cache.append(x[1], x[1])
            pxq.kv_attention(qs[1], cache, heads, weights=w, weights_out=w)
            assert bool((w[:, :, t:t + 5] > 0).all())
            cache.truncate(i32([t]))
            w.copy_(seen)  # what the draft gave to the tokens before it goes too
            w[:, :, t:] = 0
        cache.append(x[2], x[2])
        pxq.kv_attention(qs[2], cache, heads, weights=w, weights_out=w)
        totals.append(w)
    pxq.synchronize()
    assert torch.equal(*totals)
