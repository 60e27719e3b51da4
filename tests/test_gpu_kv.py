"""The 8-bit key/value cache (pxq_kv_*) against its plain 64-bit forms.

What the cache holds is compared bit for bit: codes and scales have one right
value.  Attention is compared to ATT_TOL of the largest output: q and p reach
the products as two fp16 numbers (2^-22 of the value each), the codes exactly,
sums and exponentials are fp32, so a score z (|z| up to about 2^5 here, sums of
2 D terms) is off by a few 2^-24 * 2^5 and p and the output by as much: some
2^-18 = 4e-6 at the worst elements.  2e-5 is the tolerance that pxq_attention,
the same computation in fp32, is held to."""
import numpy as np
import pytest

import kv_reference as ref
from conftest import max_abs_rel

pytestmark = pytest.mark.gpu
ATT_TOL = 2e-5


def dev(x, dtype=None):
    import torch

    t = torch.as_tensor(np.ascontiguousarray(x)).cuda()
    return t if dtype is None else t.to(dtype)


def i32(x):
    return dev(np.asarray(x, np.int32))


def starts_of(ns):
    return i32(np.concatenate([[0], np.cumsum(ns)]))


def rows_of(rng, t, H, D, spread=0.5):
    return (rng.standard_normal((t, H, D)) * np.exp(spread * rng.standard_normal((t, 1, 1)))).astype(np.float32)


class Batch:
    """A cache and the rows that were appended to each sequence."""

    def __init__(self, pxq, rng, lens, H, D, cap=None, spread=0.5):
        self.pxq, self.H, self.D, self.rng = pxq, H, D, rng
        self.cap = cap or max(max(lens), 1)
        self.cache = pxq.KVCache(len(lens), self.cap, H, D)
        self.k = [rows_of(rng, t, H, D, spread) for t in lens]
        self.v = [rows_of(rng, t, H, D, spread) for t in lens]
        if sum(lens):
            self.cache.append(dev(np.concatenate(self.k).reshape(-1, H * D)), dev(np.concatenate(self.v).reshape(-1, H * D)),
                              starts=starts_of(lens))

    def check(self, lens=None):
        lens = [len(x) for x in self.k] if lens is None else lens
        assert self.cache.lengths().cpu().tolist() == lens
        k, v = (x.cpu().numpy().reshape(len(lens), self.cap, self.H, self.D) for x in self.cache.read())
        for s, t in enumerate(lens):
            assert np.array_equal(k[s, :t], ref.values(self.k[s]), equal_nan=True), s
            assert np.array_equal(v[s, :t], ref.values(self.v[s]), equal_nan=True), s
            assert not k[s, t:].any() and not v[s, t:].any()


# ------------------------------------------------------------------ append ---

@pytest.mark.parametrize("D", [64, 80, 128])
@pytest.mark.parametrize("lens", [[1], [31, 32, 33], [100, 0, 257, 64]])
def test_append_is_exact(pxq, D, lens):
    Batch(pxq, np.random.default_rng(D + len(lens)), lens, 3, D).check()
    pxq.synchronize()


@pytest.mark.parametrize("D", [64, 80, 128])
@pytest.mark.parametrize("cut", [[1] * 70, [33, 37], [5, 27, 32, 6], [31, 1, 1, 37], [64, 6]])
def test_append_does_not_depend_on_the_cuts(pxq, D, cut):
    b = Batch(pxq, np.random.default_rng(1), [0, 0], 2, D, cap=90)
    for n in cut:
        new = [rows_of(b.rng, n, 2, D), rows_of(b.rng, n // 2, 2, D)]
        vnew = [rows_of(b.rng, n, 2, D), rows_of(b.rng, n // 2, 2, D)]
        b.cache.append(dev(np.concatenate(new).reshape(-1, 2 * D)), dev(np.concatenate(vnew).reshape(-1, 2 * D)),
                       starts=i32([0, n, n + n // 2]))
        for s in range(2):
            b.k[s] = np.concatenate([b.k[s], new[s]])
            b.v[s] = np.concatenate([b.v[s], vnew[s]])
    b.check()
    pxq.synchronize()


@pytest.mark.parametrize("D", [64, 80, 128])
def test_append_strided_and_unaligned_rows(pxq, D):
    """k and v as column slices of one wider buffer, starting off 16 bytes."""
    rng = np.random.default_rng(2)
    H, t = 2, 77
    for pad in (1, 4):
        wide = rng.standard_normal((t, 2 * H * D + 3 * pad)).astype(np.float32)
        w = dev(wide)
        c = pxq.KVCache(1, t, H, D)
        c.append(w[:, pad:pad + H * D], w[:, 2 * pad + H * D:2 * pad + 2 * H * D])
        k, v = (x.cpu().numpy().reshape(t, H, D) for x in c.read())
        assert np.array_equal(k, ref.values(wide[:, pad:pad + H * D].reshape(t, H, D)))
        assert np.array_equal(v, ref.values(wide[:, 2 * pad + H * D:2 * pad + 2 * H * D].reshape(t, H, D)))
    pxq.synchronize()


def test_append_special_values(pxq):
    """Blocks of zeros, of magnitudes below the smallest scale and just above, of halves (ties), of the largest numbers,
    and with values that are not finite, which make their own block NaN and no other."""
    H, D = 1, 64
    rng = np.random.default_rng(3)
    blocks = [np.zeros((32, H, D)), np.full((32, H, D), 2.0 ** -119), np.full((32, H, D), 2.0 ** -118) * rng.uniform(-1, 1, (32, H, D))]
    ties = rng.integers(-127, 127, (32, H, D)) + 0.5
    ties[0, 0, 0] = 127.0  # scale 1: every other value lies half way between two codes
    near = np.nextafter(np.float32(ties), np.float32(0))
    near[0, 0, 0] = 127.0
    big = 3.4e38 * rng.uniform(-1, 1, (32, H, D))
    blocks += [ties, near, big]
    blocks[2][0, 0, 0] = 2.0 ** -118
    for bad in (np.nan, np.inf, -np.inf):
        x = rng.standard_normal((32, H, D))
        x[7, 0, 9] = bad
        blocks += [x, rng.standard_normal((32, H, D))]
    b = Batch(pxq, rng, [0], H, D, cap=32 * len(blocks))
    b.k = [np.concatenate(blocks).astype(np.float32)]
    b.v = [b.k[0][::-1].copy()]
    b.cache.append(dev(b.k[0].reshape(-1, D)), dev(b.v[0].reshape(-1, D)))
    b.check()
    pxq.synchronize()


def test_append_beyond_capacity_and_bad_bounds(pxq):
    """What only the device sees: the sequence that would overflow keeps what it had, bounds outside the rows drop the
    call, and pxq_synchronize says so once."""
    H, D = 2, 64
    b = Batch(pxq, np.random.default_rng(4), [60, 10], H, D, cap=64)
    new = [rows_of(b.rng, 5, H, D), rows_of(b.rng, 5, H, D)]
    x = dev(np.concatenate(new).reshape(-1, H * D))
    b.cache.append(x, x)
    with pytest.raises(pxq.PxqError) as err:
        pxq.synchronize()
    assert err.value.code == pxq.ERR_DEVICE_STATUS and "capacity" in str(err.value)
    b.k[1], b.v[1] = np.concatenate([b.k[1], new[1]]), np.concatenate([b.v[1], new[1]])
    b.check()
    for bad in ([0, 6, 11], [-1, 2, 4], [3, 2, 10], [0, 9, 8]):
        b.cache.append(x, x, starts=i32(bad))
        with pytest.raises(pxq.PxqError) as err:
            pxq.synchronize()
        assert err.value.code == pxq.ERR_DEVICE_STATUS and "bounds" in str(err.value)
        b.check()
    b.cache.append(x, x, starts=i32([2, 2, 6]))  # rows before the first and behind the last are nobody's
    b.k[1], b.v[1] = (np.concatenate([y, x.cpu().numpy()[2:6].reshape(-1, H, D)]) for y in (b.k[1], b.v[1]))
    b.check()
    pxq.synchronize()


# ---------------------------------------------------------------- truncate ---

@pytest.mark.parametrize("D", [64, 80, 128])
def test_truncate(pxq, D):
    H = 2
    b = Batch(pxq, np.random.default_rng(5), [100, 96, 70, 33], H, D, cap=130)
    # within the last block, at a block's border, as it is (too long, negative)
    b.cache.truncate(i32([97, 64, 200, -1]))
    b.k, b.v = ([x[0][:97], x[1][:64], x[2], x[3]] for x in (b.k, b.v))
    b.check()
    # into a closed block: it is opened from the values it stands for (sequence 1: the border left no rows at hand)
    b.cache.truncate(i32([40, 63, 70, 32]))
    for x in (b.k, b.v):
        x[0] = np.concatenate([x[0][:32], ref.values(x[0][:64])[32:40]])
        x[1] = np.concatenate([x[1][:32], ref.values(x[1])[32:63]])
        x[3] = x[3][:32]
    b.check()
    new = [rows_of(b.rng, 30, H, D) for _ in range(4)]
    b.cache.append(dev(np.concatenate(new).reshape(-1, H * D)), dev(np.concatenate(new).reshape(-1, H * D)))
    b.k, b.v = ([np.concatenate([y, n]) for y, n in zip(x, new)] for x in (b.k, b.v))
    b.check()
    b.cache.truncate()
    b.k = b.v = [np.zeros((0, H, D), np.float32)] * 4
    b.check()
    pxq.synchronize()


def test_truncate_then_append_gives_the_same_cache(pxq):
    """A token taken back and appended again (at a border and within a block) leaves the cache as it was."""
    H, D = 2, 128
    for t in (31, 32, 33, 64, 65):
        b = Batch(pxq, np.random.default_rng(t), [t], H, D)
        before = b.cache.memory.clone()
        b.cache.truncate(i32([t - 1]))
        b.cache.append(dev(b.k[0][-1:].reshape(1, -1)), dev(b.v[0][-1:].reshape(1, -1)))
        b.check()
        tail = 256 + 12  # ticket and the per-sequence words
        assert bool((before[:tail] == b.cache.memory[:tail]).all()) or (t % 32 == 1)
    pxq.synchronize()


def test_read_of_a_part(pxq):
    import torch

    H, D = 2, 80
    b = Batch(pxq, np.random.default_rng(6), [50, 130, 7], H, D)
    first = [33, 64, 9]
    k = torch.full((3, 41, H * D), 7.0, device="cuda")
    v = torch.full((3, 41, H * D), 7.0, device="cuda")
    b.cache.read(i32(first), 41, k=k, v=v)
    for got, rows in ((k, b.k), (v, b.v)):
        got = got.cpu().numpy().reshape(3, 41, H, D)
        for s in range(3):
            want = ref.values(rows[s])[first[s]:first[s] + 41]
            assert np.array_equal(got[s, :len(want)], want)
            assert (got[s, len(want):] == 7).all()
    pxq.synchronize()


# --------------------------------------------------------------- attention ---

CASES = [
    # lens, rows per sequence, heads, kv heads, D, causal
    ([1], [1], 4, 4, 64, True),                          # one token
    ([33], [1], 7, 1, 128, True),                        # one block and a token
    ([1000], [1], 28, 4, 128, True),                     # decode, a run shared by several CTAs
    ([5000, 31, 777], [1, 1, 1], 8, 2, 80, True),        # ragged decode: parts, whole segments, short ones
    ([300, 4000], [1, 2], 4, 4, 64, False),              # few rows, non-causal
    ([4096], [8], 28, 4, 128, True),                     # 56 pairs
    ([70], [70], 4, 2, 64, True),                        # a prompt against itself
    ([200, 150, 129], [130, 20, 1], 6, 3, 80, True),     # ragged chunks
    ([150], [40], 28, 2, 128, False),                    # 14 heads a group
    ([40, 0, 65], [3, 2, 0], 2, 2, 128, True),           # an empty sequence with rows, one without rows
    ([3, 10], [7, 10], 4, 1, 64, True),                  # more rows than tokens: the first see nothing
    ([513], [257], 2, 1, 128, True),
    ([1300, 1290], [300, 5], 16, 16, 80, False),         # several key tiles and pair tiles
    ([260], [260], 3, 3, 128, True),
    ([700, 33], [4, 3], 28, 4, 128, True),               # 17 to 32 pairs: two tiles of 16 side by side
    ([50, 900, 0], [17, 25, 4], 2, 2, 80, False),
    ([500], [32], 1, 1, 64, True),
    ([300, 40000], [2, 3], 8, 1, 64, True),              # the same over a cache too long for that
]


def run_attention(pxq, b, ns, heads, causal, q, **kw):
    H = b.H
    out = pxq.kv_attention(q, b.cache, heads, starts=starts_of(ns), max_rows=max(ns), causal=causal, **kw)
    return out


@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention(pxq, case):
    import torch

    lens, ns, heads, H, D, causal = CASES[case]
    rng = np.random.default_rng(50 + case)
    b = Batch(pxq, rng, lens, H, D)
    q = (1.5 * rng.standard_normal((sum(ns), heads, D))).astype(np.float32)
    w0 = rng.uniform(0, 2, (len(lens), H, b.cap)).astype(np.float32)
    w_out = torch.full(w0.shape, -3.0, device="cuda")
    qd = dev(q.reshape(len(q), -1))
    out = run_attention(pxq, b, ns, heads, causal, qd)
    again = run_attention(pxq, b, ns, heads, causal, qd, weights=dev(w0), weights_out=w_out)
    pxq.synchronize()
    assert torch.equal(out, again)  # the weights change nothing, and nothing depends on the order of execution
    got, w_got, at = out.cpu().numpy().reshape(-1, heads, D), w_out.cpu().numpy(), 0
    for s, (t, n) in enumerate(zip(lens, ns)):
        want, w = ref.attention(q[at:at + n], ref.values(b.k[s]), ref.values(b.v[s]), heads, causal)
        if n:
            assert max_abs_rel(got[at:at + n], want) <= ATT_TOL, s
            if causal and n > t:
                assert not got[at:at + n - t].any()
        assert max_abs_rel(w_got[s, :, :t], w + w0[s, :, :t]) <= ATT_TOL if t else True
        assert (w_got[s, :, t:] == -3).all()
        at += n


def test_attention_uniform_rows_strides_and_rows_behind(pxq):
    """No starts: rows / sequences each; q and out with a row stride, out starting off 16 bytes; rows behind the last
    sequence, and the columns between, are left as they were; weights in place."""
    import torch

    rng = np.random.default_rng(7)
    heads, H, D, lens = 4, 2, 128, [90, 40]
    b = Batch(pxq, rng, lens, H, D)
    for n in (1, 3, 40):
        q = rng.standard_normal((2 * n + 2, heads, D)).astype(np.float32)
        wide = torch.zeros((2 * n + 2, heads * D + 5), device="cuda")
        wide[:, 3:3 + heads * D] = dev(q.reshape(len(q), -1))
        qd = wide[:, 3:3 + heads * D]
        buf = torch.full((2 * n + 2, heads * D + 6), 9.0, device="cuda")
        w = torch.zeros((2, H, b.cap), device="cuda")
        pxq.kv_attention(qd, b.cache, heads, starts=starts_of([n, n]), max_rows=n, causal=True, out=buf[:, 1:1 + heads * D], weights=w, weights_out=w)
        same = pxq.kv_attention(qd[:2 * n], b.cache, heads, causal=True)
        pxq.synchronize()
        assert torch.equal(buf[:2 * n, 1:1 + heads * D], same)
        assert (buf[2 * n:] == 9).all() and (buf[:, 0] == 9).all() and (buf[:, 1 + heads * D:] == 9).all()
        for s in range(2):
            want, wt = ref.attention(q[s * n:(s + 1) * n], ref.values(b.k[s]), ref.values(b.v[s]), heads, True)
            assert max_abs_rel(same[s * n:(s + 1) * n].cpu().numpy().reshape(n, heads, D), want) <= ATT_TOL
            assert max_abs_rel(w[s, :, :lens[s]].cpu().numpy(), wt) <= ATT_TOL


@pytest.mark.parametrize("n", [1, 2, 40])
def test_attention_ignores_what_is_masked(pxq, n):
    """A block that is not finite changes the rows that see it (to NaN) and no other; an unused cache's memory may hold
    anything."""
    import torch

    rng = np.random.default_rng(8)
    heads, H, D, t = 2, 1, 128, 96
    b = Batch(pxq, rng, [0], H, D, cap=200)
    b.cache.memory[256 + 12 + 244:].fill_(255)  # everything but the zeroed head: scales NaN, codes 127
    k, v = rows_of(rng, t + n, H, D), rows_of(rng, t + n, H, D)
    k[t + n - 1, 0, 5] = np.inf if n == 2 else np.nan  # the last token
    v[t + n - 1, 0, 6] = np.nan
    b.cache.append(dev(k.reshape(-1, D)), dev(v.reshape(-1, D)))
    q = rng.standard_normal((n, heads, D)).astype(np.float32)
    got = pxq.kv_attention(dev(q.reshape(n, -1)), b.cache, heads).cpu().numpy().reshape(n, heads, D)
    pxq.synchronize()
    first_bad = (t + n - 1) // 32 * 32  # the NaN block's first token
    sees = [t + i >= first_bad for i in range(n)]
    kv, vv = ref.values(k), ref.values(v)
    for i in range(n):
        if sees[i]:
            assert np.isnan(got[i]).all()
        else:
            want, _ = ref.attention(q[i:i + 1], kv[:t + i + 1], vv[:t + i + 1], heads, True)
            assert max_abs_rel(got[i:i + 1], want) <= ATT_TOL
    w = torch.zeros((1, H, 200), device="cuda")
    b.cache.truncate(i32([first_bad]))
    out = pxq.kv_attention(dev(q.reshape(n, -1)), b.cache, heads, causal=False, weights_out=w)
    assert torch.isfinite(out).all() and torch.isfinite(w).all()
    pxq.synchronize()


@pytest.mark.parametrize("rows", [1, 50])
def test_attention_over_blocks_of_very_different_scale(pxq, rows):
    """V's magnitude ranges over 2^40 between blocks, K's over 2^8, q's rows over 2^60."""
    rng = np.random.default_rng(9)
    heads, H, D, t = 4, 2, 64, 640
    b = Batch(pxq, rng, [0], H, D, cap=t)
    grow = 2.0 ** rng.integers(-20, 21, (t // 32, 1, 1, 1))
    k = (rng.standard_normal((t // 32, 32, H, D)) * 2.0 ** rng.integers(-6, 3, (t // 32, 1, 1, 1))).astype(np.float32)
    v = (rng.standard_normal((t // 32, 32, H, D)) * grow).astype(np.float32)
    b.k, b.v = [k.reshape(t, H, D)], [v.reshape(t, H, D)]
    b.cache.append(dev(k.reshape(t, -1)), dev(v.reshape(t, -1)))
    q = (rng.standard_normal((rows, heads, D)) * 2.0 ** rng.integers(-60, 1, (rows, 1, 1))).astype(np.float32)
    got = pxq.kv_attention(dev(q.reshape(rows, -1)), b.cache, heads, causal=False).cpu().numpy().reshape(rows, heads, D)
    pxq.synchronize()
    want, _ = ref.attention(q, ref.values(b.k[0]), ref.values(b.v[0]), heads, False)
    for i in range(rows):
        assert max_abs_rel(got[i], want[i]) <= ATT_TOL


@pytest.mark.parametrize("rows", [1, 9, 300])
def test_attention_with_the_largest_numbers(pxq, rows):
    """V up to fp32's largest numbers (sums of p V before the division would not fit), q up to 2^127 with K down at 2^-117."""
    rng = np.random.default_rng(14)
    heads, H, D, t = 2, 1, 64, 700
    k = (2.0 ** -117 * rng.uniform(-1, 1, (t, H, D))).astype(np.float32)
    v = (3.4e38 * rng.uniform(-1, 1, (t, H, D))).astype(np.float32)
    q = (2.0 ** 118 * rng.uniform(-1, 1, (rows, heads, D))).astype(np.float32)
    q[0] = 2.0 ** 127 * 1.9 * np.sign(q[0])
    cache = pxq.KVCache(1, t, H, D)
    cache.append(dev(k.reshape(t, -1)), dev(v.reshape(t, -1)))
    got = pxq.kv_attention(dev(q.reshape(rows, -1)), cache, heads, causal=False).cpu().numpy().reshape(rows, heads, D)
    pxq.synchronize()
    want, _ = ref.attention(q, ref.values(k), ref.values(v), heads, False)
    for i in range(1, rows):
        assert max_abs_rel(got[i], want[i]) <= ATT_TOL
    # row 0's scores go up to 2^17, where one step of fp32 is 2^-6: what is left to ask is that no number overflowed
    assert np.isfinite(got[0]).all() and float(np.abs(got[0]).max()) <= 3.5e38


def test_attention_bad_bounds(pxq):
    """A sequence with more rows than announced, or bounds outside q, is left alone and reported; the others are right."""
    import torch

    rng = np.random.default_rng(10)
    heads, H, D = 2, 2, 64
    b = Batch(pxq, rng, [50, 50], H, D)
    q = dev(rng.standard_normal((6, heads * D)).astype(np.float32))
    good = pxq.kv_attention(q, b.cache, heads, starts=i32([0, 2, 4]))
    pxq.synchronize()
    for starts, most, fine in (([0, 2, 6], 2, (0, 2)), ([0, 2, 7], 4, (0, 2)), ([3, 2, 4], 4, (2, 4))):
        out = torch.full_like(q, 5.0)
        pxq.kv_attention(q, b.cache, heads, starts=i32(starts), max_rows=most, out=out)
        with pytest.raises(pxq.PxqError) as err:
            pxq.synchronize()
        assert err.value.code == pxq.ERR_DEVICE_STATUS
        assert torch.equal(out[fine[0]:fine[1]], good[fine[0]:fine[1]])
        assert (out[:fine[0]] == 5).all() and (out[fine[1]:] == 5).all()


# ------------------------------------------------------------------- evict ---

@pytest.mark.parametrize("D", [64, 80, 128])
@pytest.mark.parametrize("keep,recent", [(1, 0), (32, 32), (100, 7), (63, 0), (5000, 10)])
def test_evict(pxq, D, keep, recent):
    import torch

    rng = np.random.default_rng(keep + D)
    H, lens = 2, [300, 90, 0, 4500]
    b = Batch(pxq, rng, lens, H, D)
    w = rng.uniform(0, 1, (4, H, b.cap)).astype(np.float32) ** 4
    w[w < 0.05] = 0.0  # ties, some of them negative zeros
    w[0, 0, 5:9] = [np.nan, np.inf, -np.inf, -0.0]
    w[3, 1, :40] = -1.5
    cap = min(keep, 5000) + 40
    dst = pxq.KVCache(4, cap, H, D)
    w_out = torch.full((4, H, cap), -7.0, device="cuda")
    kept = torch.full((4, H, keep), -1, dtype=torch.int32, device="cuda")
    pxq.kv_evict(b.cache, dst, dev(w), keep=keep, recent=recent, weights_out=w_out, kept=kept)
    other = pxq.KVCache(4, cap, H, D)
    pxq.kv_evict(b.cache, other, dev(w), keep=keep, recent=recent)
    pxq.synchronize()
    k, v = (x.cpu().numpy().reshape(4, cap, H, D) for x in dst.read())
    for got, want in zip(other.read(), dst.read()):
        assert torch.equal(got, want)
    w_got, kept = w_out.cpu().numpy(), kept.cpu().numpy()
    assert dst.lengths().cpu().tolist() == [min(t, keep) for t in lens]
    for s, t in enumerate(lens):
        c = min(t, keep)
        kv, vv = ref.values(b.k[s]), ref.values(b.v[s])
        for h in range(H):
            at = ref.kept(w[s, h, :t], keep, recent)
            assert np.array_equal(kept[s, h, :c], at), (s, h)
            assert (kept[s, h, c:] == -1).all() and (w_got[s, h, c:] == -7).all()
            assert np.array_equal(w_got[s, h, :c], w[s, h, at], equal_nan=True)
            assert np.array_equal(k[s, :c, h:h + 1], ref.values(kv[at, h:h + 1]))
            assert np.array_equal(v[s, :c, h:h + 1], ref.values(vv[at, h:h + 1]))
    # the destination goes on like any cache
    new = rows_of(rng, 4, H, D)
    before = [x.cpu().numpy().reshape(4, cap, H, D) for x in dst.read()]
    dst.append(dev(new.reshape(4, -1)), dev(new.reshape(4, -1)))
    after = [x.cpu().numpy().reshape(4, cap, H, D) for x in dst.read()]
    for s, t in enumerate(lens):
        c = min(t, keep)
        for x0, x1 in zip(before, after):
            # the open block's rows are the fp32 values that were moved
            assert np.array_equal(x1[s, :c // 32 * 32], x0[s, :c // 32 * 32])
    kv0, at = ref.values(b.k[0]), [ref.kept(w[0, h, :lens[0]], keep, recent) for h in range(H)]
    c = min(lens[0], keep)
    for h in range(H):
        rows = np.concatenate([kv0[at[h], h:h + 1], new[0:1, h:h + 1]])
        assert np.array_equal(after[0][0, :c + 1, h:h + 1], ref.values(rows))
    pxq.synchronize()


# ---------------------------------------------------------------- together ---

def test_a_chat_with_eviction(pxq):
    """A prompt, decode steps that gather weights, an eviction, and more steps, as a decode loop runs them."""
    import torch

    rng = np.random.default_rng(11)
    heads, H, D, S, cap = 6, 2, 128, 2, 128
    lens = [90, 61]
    b = Batch(pxq, rng, lens, H, D, cap=cap)
    spare = pxq.KVCache(S, cap, H, D)
    w, spare_w = torch.zeros((S, H, cap), device="cuda"), torch.zeros((S, H, cap), device="cuda")
    K = [[ref.values(b.k[s])[:, h] for h in range(H)] for s in range(S)]  # what each head holds, as appended rows
    rows_k = [[b.k[s][:, h] for h in range(H)] for s in range(S)]
    rows_v = [[b.v[s][:, h] for h in range(H)] for s in range(S)]
    W = [[np.zeros(len(K[s][h])) for h in range(H)] for s in range(S)]
    cache = b.cache
    for step in range(12):
        n = [1, 3][step % 2]
        k, v = rows_of(rng, S * n, H, D), rows_of(rng, S * n, H, D)
        q = rng.standard_normal((S * n, heads, D)).astype(np.float32)
        cache.append(dev(k.reshape(S * n, -1)), dev(v.reshape(S * n, -1)))
        out = pxq.kv_attention(dev(q.reshape(S * n, -1)), cache, heads, weights=w, weights_out=w)
        got = out.cpu().numpy().reshape(S, n, heads, D)
        for s in range(S):
            for h in range(H):
                rows_k[s][h] = np.concatenate([rows_k[s][h], k[s * n:(s + 1) * n, h]])
                rows_v[s][h] = np.concatenate([rows_v[s][h], v[s * n:(s + 1) * n, h]])
                G = heads // H
                want, wt = ref.attention(q[s * n:(s + 1) * n, h * G:(h + 1) * G], ref.values(rows_k[s][h][:, None]),
                                         ref.values(rows_v[s][h][:, None]), G, True)
                assert max_abs_rel(got[s][:, h * G:(h + 1) * G], want) <= ATT_TOL, (step, s, h)
                W[s][h] = np.concatenate([W[s][h], np.zeros(n)]) + wt[0]
                assert max_abs_rel(w[s, h, :len(W[s][h])].cpu().numpy(), W[s][h]) <= ATT_TOL
        if step == 5:
            pxq.kv_evict(cache, spare, w, keep=50, recent=10, weights_out=spare_w)
            for s in range(S):
                for h in range(H):
                    at = ref.kept(w[s, h, :len(W[s][h])].cpu().numpy(), 50, 10)
                    rows_k[s][h] = ref.values(rows_k[s][h][:, None])[at, 0]
                    rows_v[s][h] = ref.values(rows_v[s][h][:, None])[at, 0]
                    W[s][h] = w[s, h].cpu().numpy()[at].astype(np.float64)
            cache, spare, w, spare_w = spare, cache, spare_w, w
            w[:, :, 50:] = 0
    pxq.synchronize()


def test_captured_step_advances_on_every_replay(pxq):
    """A decode step (append, attention with weights, lengths) captured once and replayed equals eager steps; two graphs
    captured on one stream and replayed on two at once do not share scratch."""
    import torch

    rng = np.random.default_rng(12)
    heads, H, D, S, steps = 8, 2, 128, 3, 40
    k, v = (dev(rows_of(rng, S * steps, H, D).reshape(steps, S, H * D)) for _ in range(2))
    q = dev(rng.standard_normal((steps, S, heads * D)).astype(np.float32))

    class Step:
        def __init__(self):
            self.cache = pxq.KVCache(S, 64, H, D)
            self.k, self.v, self.q = (torch.zeros_like(x[0]) for x in (k, v, q))
            self.w = torch.zeros((S, H, 64), device="cuda")
            self.out = torch.zeros((S, heads * D), device="cuda")

        def load(self, i):
            self.k.copy_(k[i]), self.v.copy_(v[i]), self.q.copy_(q[i])

        def __call__(self):
            self.cache.append(self.k, self.v)
            pxq.kv_attention(self.q, self.cache, heads, weights=self.w, weights_out=self.w, out=self.out)

    eager = Step()
    want = []
    for i in range(steps):
        eager.load(i)
        eager()
        want.append(eager.out.clone())
    two = [Step(), Step()]
    graphs = []
    for st in two:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            st()
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for i in range(steps):
        for j, st in enumerate(two):
            with torch.cuda.stream(streams[j]):
                st.load(i)
                graphs[j].replay()
                got[j].append(st.out.clone())
    torch.cuda.synchronize()
    for j in range(2):
        for i in range(steps):
            assert torch.equal(got[j][i], want[i]), (j, i)
        assert torch.equal(two[j].w, eager.w)
        assert two[j].cache.lengths().cpu().tolist() == [steps] * S
    pxq.synchronize()
    del graphs


def test_other_stream(pxq):
    """Every call on a side stream, whose work is ordered by that stream alone."""
    import torch

    rng = np.random.default_rng(13)
    heads, H, D = 4, 2, 64
    x = dev(rows_of(rng, 500, H, D).reshape(500, -1))
    q = dev(rng.standard_normal((500, heads * D)).astype(np.float32))
    cache = pxq.KVCache(1, 500, H, D)
    cache.append(x, x)
    want = pxq.kv_attention(q, cache, heads)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
    other = pxq.KVCache(1, 500, H, D, stream=side)
    other.append(x.t().contiguous().t(), x, stream=side)  # not row-major: copied on the call's stream
    got = pxq.kv_attention(q, other, heads, stream=side)
    k, _ = other.read(stream=side)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(k, cache.read()[0])
    pxq.synchronize(side)


def test_offsets_beyond_32_bits(pxq):
    """A cache of more than 2^31 bytes: its last blocks are written, read and attended to at their right places."""
    import torch

    H, D, t = 8, 128, 1_200_000
    cache = pxq.KVCache(1, t, H, D)
    assert cache.memory.numel() > 2 ** 31
    g = torch.Generator(device="cuda").manual_seed(3)
    chunk = torch.randn((150_000, H * D), generator=g, device="cuda")
    for i in range(8):
        cache.append(chunk * (1.0 if i < 7 else 2.0), chunk)
    out = torch.zeros((1, 64, H * D), device="cuda")
    cache.read(i32([t - 64]), 64, k=out, v=torch.empty_like(out))
    want = ref.values((2 * chunk[-64:]).cpu().numpy().reshape(64, H, D))
    assert np.array_equal(out.cpu().numpy().reshape(64, H, D), want)
    q = torch.randn((1, H * D), generator=g, device="cuda")
    w = torch.zeros((1, H, t), device="cuda")
    got = pxq.kv_attention(q, cache, H, weights_out=w).view(H, D)
    pxq.synchronize()
    k, v = cache.read()
    for h in (0, H - 1):
        z = (k[0, :, h * D:(h + 1) * D].double() @ q[0, h * D:(h + 1) * D].double()) / np.sqrt(D)
        p = torch.softmax(z, 0)
        assert max_abs_rel(got[h].cpu().numpy(), (p @ v[0, :, h * D:(h + 1) * D].double()).cpu().numpy()) <= ATT_TOL
        assert max_abs_rel(w[0, h].cpu().numpy(), p.cpu().numpy()) <= ATT_TOL


# ---------------------------------------------------------------- refusals ---

def test_refusals(pxq):
    import torch

    H, D = 2, 64
    c = pxq.KVCache(2, 40, H, D)
    x = torch.zeros((4, H * D), device="cuda")
    q = torch.zeros((4, 4 * D), device="cuda")
    for bad in (lambda: c.append(x[:3], x[:3]), lambda: c.append(x[:0], x[:0]),
                lambda: pxq.kv_attention(torch.zeros((4, 3 * D), device="cuda"), c, 3),
                lambda: pxq.kv_attention(q[:3], c, 4), lambda: pxq.kv_attention(q, c, 4, starts=i32([0, 2, 4]), max_rows=5),
                lambda: pxq.kv_attention(q, c, 4, weights=torch.zeros((2, H, 40), device="cuda")),
                lambda: c.read(count=0),
                lambda: pxq.kv_evict(c, c, torch.zeros((2, H, 40), device="cuda")),
                lambda: pxq.kv_evict(c, pxq.KVCache(2, 40, H, 80), torch.zeros((2, H, 40), device="cuda")),
                lambda: pxq.kv_evict(c, pxq.KVCache(2, 20, H, D), torch.zeros((2, H, 40), device="cuda"), keep=21),
                lambda: pxq.kv_evict(c, pxq.KVCache(2, 20, H, D), torch.zeros((2, H, 40), device="cuda"), recent=21)):
        with pytest.raises(pxq.PxqError) as err:
            bad()
        assert err.value.code == pxq.ERR_INVALID
    for bad in (lambda: c.append(x.half(), x), lambda: c.append(x, x[:2]), lambda: c.append(x[:, :-1], x),
                lambda: c.append(x.cpu(), x), lambda: c.append(x, x, starts=torch.zeros(2, dtype=torch.int32, device="cuda")),
                lambda: c.truncate(torch.zeros(2, dtype=torch.int64, device="cuda")),
                lambda: pxq.kv_attention(q, c, 4, out=torch.zeros((4, 5 * D), device="cuda")),
                lambda: pxq.kv_attention(q, c, 4, weights_out=torch.zeros((2, H, 41), device="cuda")),
                lambda: pxq.kv_evict(c, pxq.KVCache(2, 20, H, D), None)):
        with pytest.raises(ValueError):
            bad()
    c.release()
    with pytest.raises(ValueError):
        c.lengths()
    torch.cuda.synchronize()
    pxq.synchronize()


def test_memory_that_is_not_the_devices_is_refused(pxq):
    """Plain and pinned host memory: refused before anything is written to it."""
    import ctypes as C

    import torch

    lib = pxq.load()
    n = lib.pxq_kv_cache_bytes(1, 32, 1, 64)
    h = C.c_void_p()
    for pinned in (False, True):
        memory = torch.full((n + 256,), 7, dtype=torch.uint8, pin_memory=pinned)
        at = -(-memory.data_ptr() // 256) * 256
        assert lib.pxq_kv_cache_create(at, 1, 32, 1, 64, C.byref(h), None) == pxq.ERR_INVALID
        assert not h.value and bool((memory == 7).all())
    torch.cuda.synchronize()


@pytest.mark.parametrize("rows", [1, 40])
def test_output_that_is_q_is_refused(pxq, rows):
    import torch

    c = pxq.KVCache(1, 64, 2, 64)
    x = torch.zeros((rows, 2 * 64), device="cuda")
    c.append(x, x)
    with pytest.raises(pxq.PxqError) as err:
        pxq.kv_attention(x, c, 2, out=x)
    assert err.value.code == pxq.ERR_INVALID
    pxq.synchronize()
