"""CPU: the key/value cache's size rules and its refusals that need no device."""
import ctypes as C

import pytest

from pixelina_b200 import pxq


def test_cache_bytes():
    """Per (sequence, head, 32 tokens) 64 * D bytes of codes and 8 of scales; two fp32 blocks of K and V per (sequence,
    head); 12 bytes per sequence and the head, each part rounded up to 256 bytes."""
    lib = pxq.load()
    up = lambda n: -(-n // 256) * 256  # noqa: E731
    for S, cap, H, D in ((1, 1, 1, 64), (3, 33, 2, 80), (8, 4096, 4, 128), (1024, 31, 5, 128), (1, 1 << 30, 2, 64)):
        nb = -(-cap // 32)
        want = up(256 + 12 * S) + up(S * H * nb * 8) + up(S * H * 512 * D) + up(S * H * nb * 64 * D)
        assert lib.pxq_kv_cache_bytes(S, cap, H, D) == want, (S, cap, H, D)


@pytest.mark.parametrize("sizes", [(0, 1, 1, 64), (1, 0, 1, 64), (1, 1, 0, 64), (1, 1, 1, 0), (1, 1, 1, 96), (1025, 1, 1, 64),
                                   (1, 1, 4097, 64), (1, (1 << 30) + 1, 1, 64), (1024, 1 << 20, 4096, 64)])
def test_sizes_that_are_refused(sizes):
    lib = pxq.load()
    assert lib.pxq_kv_cache_bytes(*sizes) == 0
    assert pxq.last_error()
    h = C.c_void_p()
    assert lib.pxq_kv_cache_create(C.c_void_p(256), *sizes, C.byref(h), None) in (pxq.ERR_INVALID, pxq.ERR_UNSUPPORTED)
    with pytest.raises(pxq.PxqError):
        pxq.KVCache(*sizes)


def test_null_and_misaligned_arguments():
    lib = pxq.load()
    h, p = C.c_void_p(), C.c_void_p(4096)
    assert lib.pxq_kv_cache_create(None, 1, 1, 1, 64, C.byref(h), None) == pxq.ERR_INVALID
    assert lib.pxq_kv_cache_create(p, 1, 1, 1, 64, None, None) == pxq.ERR_INVALID
    assert lib.pxq_kv_cache_create(C.c_void_p(4096 + 16), 1, 1, 1, 64, C.byref(h), None) == pxq.ERR_INVALID
    assert "aligned" in pxq.last_error()
    assert lib.pxq_kv_cache_release(None) == pxq.ERR_INVALID
    assert lib.pxq_kv_cache_lengths(None, p, None) == pxq.ERR_INVALID
    assert lib.pxq_kv_append(None, p, 64, p, 64, 1, None, None) == pxq.ERR_INVALID
    assert lib.pxq_kv_truncate(None, None, None) == pxq.ERR_INVALID
    assert lib.pxq_kv_read(None, None, 1, p, p, None) == pxq.ERR_INVALID
    assert lib.pxq_kv_attention(None, p, 64, 1, None, 1, 1, 1, p, 64, None, None, None) == pxq.ERR_INVALID
    assert lib.pxq_kv_evict(None, None, p, 1, 0, None, None, None) == pxq.ERR_INVALID
