"""Errors of the key/value cache that only the device sees, beside other callers and beside a kernel that gave up waiting."""
import ctypes as C

import numpy as np
import pytest

from conftest import TOL, max_abs_rel
from pixelina_b200 import synth
from test_gpu_kv import dev, i32

pytestmark = pytest.mark.gpu


def overflowing(pxq):
    """A cache of 8 tokens after an append of 9 rows, which was dropped."""
    import torch

    c = pxq.KVCache(1, 8, 1, 64)
    x = torch.ones((9, 64), device="cuda")
    c.append(x, x)
    return c


def test_a_dropped_append_keeps_nobody_waiting(pxq):
    """The error is reported without waiting for what other streams have under way (a timeout has to, to reset the
    scratch; an append beyond the capacity leaves nothing to reset)."""
    import torch

    side, done = torch.cuda.Stream(), torch.cuda.Event()
    overflowing(pxq)  # (kernels are loaded by now, which may wait for the device)
    with pytest.raises(pxq.PxqError):
        pxq.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(1000)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(1_000_000_000)  # half a second
        done.record()
    overflowing(pxq)
    with pytest.raises(pxq.PxqError) as err:
        pxq.synchronize()
    assert err.value.code == pxq.ERR_DEVICE_STATUS and "capacity" in str(err.value)
    assert not done.query()
    done.synchronize()
    pxq.synchronize()


def test_both_errors_are_reported(pxq):
    """Bad bounds and an overflow before one synchronize: neither hides the other."""
    c = overflowing(pxq)
    x = dev(np.ones((2, 64), np.float32))
    c.append(x, x, starts=i32([0, 3]))
    with pytest.raises(pxq.PxqError) as err:
        pxq.synchronize()
    assert "capacity" in str(err.value) and "bounds" in str(err.value)
    pxq.synchronize()
    assert c.lengths().cpu().tolist() == [0]


def test_a_timeout_is_not_hidden_by_a_dropped_append(pxq):
    """A matvec that gives up its bounded waits behind a dropped append (pxq_debug_matvec_stall): the timeout is reported first,
    its scratch is reset, and the append's error is not lost."""
    import torch

    lib = pxq.load()
    rows, inner = 200, 18944
    W = pxq.Weight(synth.random_q5_K(rows, inner, np.random.default_rng(5)), 13, inner, rows)
    x = dev(synth.activations(1, inner, seed=6))
    want = pxq.matmul(W, x)
    pxq.synchronize()
    overflowing(pxq)
    junk = torch.empty((1, rows), device="cuda")
    sp = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert lib.pxq_debug_matvec_stall(W.handle, x.data_ptr(), 1, junk.data_ptr(), 0, sp) == 0, pxq.last_error()
    for what in ("gave up", "capacity"):
        with pytest.raises(pxq.PxqError) as err:
            pxq.synchronize()
        assert err.value.code == pxq.ERR_DEVICE_STATUS and what in str(err.value)
    for _ in range(2):
        got = pxq.matmul(W, x)
        pxq.synchronize()
        assert max_abs_rel(got.cpu().numpy(), want.cpu().numpy()) <= TOL
    W.release()


def test_a_host_product_does_not_take_the_caches_error(pxq):
    """pxq_matmul_host waits for its own stream and reports what concerns the product; the cache's error stays for
    pxq_synchronize."""
    rows, inner = 64, 2048
    W = pxq.Weight(synth.random_q5_K(rows, inner, np.random.default_rng(7)), 13, inner, rows)
    x = synth.activations(2, inner, seed=8)
    want = pxq.matmul(W, dev(x)).cpu().numpy()
    overflowing(pxq)
    got = np.zeros((2, rows), np.float32)
    assert pxq.load().pxq_matmul_host(W.handle, 0, rows, x.ctypes.data, 2, got.ctypes.data, rows) == 0, pxq.last_error()
    assert max_abs_rel(got, want) <= TOL
    with pytest.raises(pxq.PxqError) as err:
        pxq.synchronize()
    assert "capacity" in str(err.value)
    pxq.synchronize()
    W.release()


@pytest.mark.parametrize("rows", [1, 40])
def test_max_rows_of_zero_is_refused(pxq, rows):
    import torch

    c = pxq.KVCache(1, 64, 2, 64)
    x = torch.zeros((rows, 2 * 64), device="cuda")
    with pytest.raises(pxq.PxqError) as err:
        pxq.kv_attention(x, c, 2, starts=i32([0, rows]), max_rows=0)
    assert err.value.code == pxq.ERR_INVALID
