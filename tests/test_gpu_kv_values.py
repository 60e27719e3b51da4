"""Attention over the 8-bit key/value cache where its blocks' values differ much in scale.

A row's output is the weighted mean of the values that it sees, so what it may not see, or gives next to no weight, may
not cost it accuracy, however large those values are.  Outputs are compared row by row, relative to the row's own
largest output.

Tolerance, as in test_gpu_kv.py: scores of the tokens that matter stay below 2^5 (their own fp32 steps 2^-19), p dv and q
reach the products to 2^-22, sums are fp32: 2e-5 leaves a factor of about 5."""
import numpy as np
import pytest

import kv_reference as ref
from test_gpu_kv import ATT_TOL, Batch, dev, i32, rows_of, starts_of

pytestmark = pytest.mark.gpu


def assert_rows_close(got, want):
    """Each row and head against its own largest output."""
    assert np.isfinite(got).all()
    got, want = got.astype(np.float64).reshape(-1, got.shape[-1]), want.reshape(-1, want.shape[-1])
    off = np.abs(got - want).max(1) / np.maximum(np.abs(want).max(1), 1e-300)
    assert off.max() <= ATT_TOL, (int(off.argmax()), float(off.max()))


def filled(pxq, k, v, H, D):
    t = len(k)
    cache = pxq.KVCache(1, t, H, D)
    cache.append(dev(k.reshape(t, -1)), dev(v.reshape(t, -1)))
    return cache


# rows, heads of a group: 1 pair, 4 (hi and lo in one fragment), 12 (two fragments), 20 (two tiles), 160 (prompt)
ROWS = [(1, 1), (1, 4), (3, 4), (5, 4), (40, 4)]


def kv_heads(rows):
    """As many that a warp of the split kernel takes several blocks of one head in turn."""
    return 40 if rows < 40 else 2


@pytest.mark.parametrize("rows,group", ROWS)
@pytest.mark.parametrize("ratio", [20, 30, 60, 90, 120])
def test_blocks_of_little_weight_with_large_values(pxq, rows, group, ratio):
    """Every third block, the first among them, holds values 2^ratio as large, with scores so low that they are 2^-25 of the
    output or less."""
    D, t, H = 64, 1536, kv_heads(rows)
    rng = np.random.default_rng(ratio)
    loud = (np.arange(t) // 32 % 3 == 0)
    k, v = rows_of(rng, t, H, D, 0.0) * np.float32(0.3), rows_of(rng, t, H, D, 0.0)
    u = np.full(D, 1 / np.sqrt(D))
    k[loud] = (-16 * u + 0.01 * rng.standard_normal((loud.sum(), H, D))).astype(np.float32)
    scale = 2.0 ** (-ratio // 2)
    v = (v * np.where(loud, 2.0 ** ratio, 1.0)[:, None, None] * scale).astype(np.float32)
    g = (ratio + 40) * np.log(2) * np.sqrt(D) / 16  # scores 2^-(ratio + 40) of the others'
    q = (g * u + 0.5 * rng.standard_normal((rows, H * group, D))).astype(np.float32)
    got = pxq.kv_attention(dev(q.reshape(rows, -1)), filled(pxq, k, v, H, D), H * group, causal=False)
    pxq.synchronize()
    want, w = ref.attention(q, ref.values(k), ref.values(v), H * group, False)
    assert w[:, loud].max() < 2.0 ** -(ratio + 25) * rows * group  # (what the test is about)
    assert_rows_close(got.cpu().numpy().reshape(rows, H * group, D), want)


@pytest.mark.parametrize("rows,group", ROWS[2:] + [(8, 1), (2, 7)])
@pytest.mark.parametrize("ratio", [30, 110, 140])
def test_large_values_that_the_mask_hides(pxq, rows, group, ratio):
    """The last token opens a block and its values are 2^ratio as large: the last row sees it, the others do not."""
    D, t, H = 128, 32 * 42 + 1, kv_heads(rows)
    rng = np.random.default_rng(ratio + rows)
    k, v = rows_of(rng, t, H, D, 0.0), rows_of(rng, t, H, D, 0.0) * np.float32(2.0 ** (-ratio // 2))
    v[-1] = (v[-1].astype(np.float64) * 2.0 ** ratio).astype(np.float32)  # (2^140 is no fp32 number)
    q = rng.standard_normal((rows, H * group, D)).astype(np.float32)
    got = pxq.kv_attention(dev(q.reshape(rows, -1)), filled(pxq, k, v, H, D), H * group)
    pxq.synchronize()
    want, _ = ref.attention(q, ref.values(k), ref.values(v), H * group, True)
    assert_rows_close(got.cpu().numpy().reshape(rows, H * group, D), want)


@pytest.mark.parametrize("rows,group", ROWS)
def test_the_smallest_values(pxq, rows, group):
    """Values around 2^-115, little above those that the cache holds as zeros."""
    D, t, H = 80, 700, kv_heads(rows)
    rng = np.random.default_rng(rows)
    k, v = rows_of(rng, t, H, D), (rows_of(rng, t, H, D, 0.0) * 2.0 ** -115).astype(np.float32)
    q = rng.standard_normal((rows, H * group, D)).astype(np.float32)
    got = pxq.kv_attention(dev(q.reshape(rows, -1)), filled(pxq, k, v, H, D), H * group, causal=False)
    pxq.synchronize()
    want, _ = ref.attention(q, ref.values(k), ref.values(v), H * group, False)
    assert_rows_close(got.cpu().numpy().reshape(rows, H * group, D), want)


@pytest.mark.parametrize("rows", [1, 3, 40])
def test_scales_that_rise_and_fall(pxq, rows):
    """Scores that rise from block to block while the values' scale wanders over 2^80, and the other way round: the unit of
    the sums moves with every block."""
    D, t, H = 64, 1600, kv_heads(rows)
    rng = np.random.default_rng(rows)
    u = np.full(D, 1 / np.sqrt(D))
    for falling in (False, True):
        at = np.arange(t) // 32
        rise = (at[::-1] if falling else at) * 0.25
        k = (0.2 * rng.standard_normal((t, H, D)) + (rise[:, None] * u)[:, None]).astype(np.float32)
        v = (rng.standard_normal((t, H, D)) * 2.0 ** (40 * np.sin(at * 0.7))[:, None, None]).astype(np.float32)
        q = (8 * u + 0.2 * rng.standard_normal((rows, 4 * H, D))).astype(np.float32)
        got = pxq.kv_attention(dev(q.reshape(rows, -1)), filled(pxq, k, v, H, D), 4 * H, causal=False)
        pxq.synchronize()
        want, _ = ref.attention(q, ref.values(k), ref.values(v), 4 * H, False)
        assert_rows_close(got.cpu().numpy().reshape(rows, 4 * H, D), want)


def test_large_values_over_a_long_cache(pxq):
    """As the first test over 400000 tokens, where a warp's sums are put aside several times: large blocks of no weight at the
    beginning of each stretch."""
    D, t, ratio = 64, 400_000, 40
    rng = np.random.default_rng(40)
    loud = (np.arange(t) // 32 % 9 < 4)
    u = np.full(D, 1 / np.sqrt(D))
    k, v = rng.standard_normal((t, 1, D)).astype(np.float32) * np.float32(0.3), rng.standard_normal((t, 1, D)).astype(np.float32)
    k[loud] = (-16 * u + 0.01 * rng.standard_normal((loud.sum(), 1, D))).astype(np.float32)
    v[loud] *= np.float32(2.0 ** ratio)
    g = (ratio + 40) * np.log(2) * np.sqrt(D) / 16
    q = (g * u + 0.5 * rng.standard_normal((1, 2, D))).astype(np.float32)
    cache = filled(pxq, k, v, 1, D)
    got = pxq.kv_attention(dev(q.reshape(1, -1)), cache, 2, causal=False)
    kv, vv = (x.cpu().numpy().reshape(t, 1, D) for x in cache.read())  # (compared with 64-bit arithmetic elsewhere)
    pxq.synchronize()
    want, _ = ref.attention(q, kv, vv, 2, False)
    assert_rows_close(got.cpu().numpy().reshape(1, 2, D), want)


def test_a_hidden_block_in_a_ragged_batch(pxq):
    """Sequences of which one alone holds large values, and not in rows' sight: every sequence has its units."""
    rng = np.random.default_rng(77)
    lens, ns, heads, H, D = [33, 200, 65], [2, 2, 2], 4, 2, 80
    b = Batch(pxq, rng, [0, 0, 0], H, D, cap=200)
    b.k, b.v = [rows_of(rng, t, H, D) for t in lens], [rows_of(rng, t, H, D) for t in lens]
    b.v[0][-1] *= np.float32(2.0 ** 70)
    b.v[2][-1, 1] *= np.float32(2.0 ** 70)
    b.cache.append(dev(np.concatenate(b.k).reshape(-1, H * D)), dev(np.concatenate(b.v).reshape(-1, H * D)), starts=starts_of(lens))
    q = rng.standard_normal((sum(ns), heads, D)).astype(np.float32)
    got = pxq.kv_attention(dev(q.reshape(len(q), -1)), b.cache, heads, starts=i32([0, 2, 4, 6]), max_rows=2).cpu().numpy().reshape(-1, heads, D)
    pxq.synchronize()
    for s in range(3):
        want, _ = ref.attention(q[2 * s:2 * s + 2], ref.values(b.k[s]), ref.values(b.v[s]), heads, True)
        assert_rows_close(got[2 * s:2 * s + 2], want)


@pytest.mark.parametrize("rows,group", ROWS)
@pytest.mark.parametrize("up", [18, 24, 40])
def test_scores_beyond_what_a_softmax_can_tell_apart(pxq, rows, group, up):
    """Scores of 2^up and more, the blocks' values of very different scale: every row takes the value of its best token (the
    next one is 2^(up - 8) below it or more; a tenth of the rows, with a nearer one, is left out)."""
    D, t, H = 64, 1536, kv_heads(rows)
    rng = np.random.default_rng(up)
    k = rows_of(rng, t, H, D, 0.0)
    v = (rng.standard_normal((t, H, D)) * 2.0 ** (30 * np.sin(np.arange(t) // 32))[:, None, None]).astype(np.float32)
    q = (2.0 ** up * rng.standard_normal((rows, H * group, D))).astype(np.float32)
    w = dev(np.zeros((1, H, t), np.float32))
    got = pxq.kv_attention(dev(q.reshape(rows, -1)), filled(pxq, k, v, H, D), H * group, causal=False, weights_out=w).cpu().numpy().reshape(rows, H * group, D)
    pxq.synchronize()
    kv, vv, w = ref.values(k).astype(np.float64), ref.values(v), w[0].cpu().numpy()
    for h in range(H):
        left, count = 0, np.zeros(t)
        for i in range(rows):
            for g in range(h * group, (h + 1) * group):
                z = kv[:, h] @ q[i, g].astype(np.float64) / np.sqrt(D)
                second, best = np.partition(z, -2)[-2:]
                if best - second < 2.0 ** (up - 8):
                    left += 1
                    continue
                count[z.argmax()] += 1
                assert_rows_close(got[i, g], vv[z.argmax(), h].astype(np.float64))
        assert left <= 2 + 0.1 * rows * group
        assert np.abs(w[h] - count).sum() <= left * 1.01 + ATT_TOL * rows * group
