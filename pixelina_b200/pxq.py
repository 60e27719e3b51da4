"""Python host mirror of the pxq C ABI (include/pxq.h).

The operator surface follows Pixelina's matmul boundary (paths within the
Pixelina source tree):

* ``quant_matmul``   -- cpu_quant_matmul (src/kernels_quant.cpp:369-412):
  host buffers in, host buffer out, ``(handled, output)`` like its bool.
* ``Weight``         -- a device-resident GGUF tensor, the Vulkan backend's
  weight cache entry (src/backend_vulkan.cpp:742-758).
* ``matmul``         -- cpu_matmul / vulkan_matmul (src/backend_cpu.cpp:103,
  src/backend_vulkan.cpp:1083) on device tensors, with the row-range view of
  tensor_linear_rows (src/tensor.cpp:529-544) and the bias of tensor_linear
  (src/tensor.cpp:156-172).
* ``quantize_q8_0`` / ``quantize_q8_K`` / ``decode`` -- the reference's
  quantizers and cpu_decode on device buffers.

torch is used only for device memory and streams.  Everything computes in
libpxq.so; importing this module on a machine without the built library or
without a B200 raises instead of falling back to any CPU path.
"""
from __future__ import annotations

import contextlib
import ctypes as C
import os
from typing import Optional

import numpy as np

LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "libpxq.so")

OK = 0
ERR_INVALID = 1
ERR_UNSUPPORTED = 2
ERR_CUDA = 3
ERR_NO_MEMORY = 4
ERR_NO_DEVICE = 5
ERR_DEVICE_STATUS = 6
ERR_IO = 7
ERR_FORMAT = 8
ERR_TIMEOUT = 9

TYPE_Q8_0 = 8
TYPE_Q5_K = 13
TYPE_Q6_K = 14
BLOCK_ELEMS = {TYPE_Q8_0: 32, TYPE_Q5_K: 256, TYPE_Q6_K: 256}
BLOCK_BYTES = {TYPE_Q8_0: 34, TYPE_Q5_K: 176, TYPE_Q6_K: 210}
Q8_0_BYTES = 34
Q8_K_BYTES = 292

# name -> (restype, argtypes); must list exactly the functions of include/pxq.h
_vp, _sz, _u32, _u64, _i = C.c_void_p, C.c_size_t, C.c_uint32, C.c_uint64, C.c_int
SIGNATURES = {
    "pxq_version": (_i, []),
    "pxq_last_error": (C.c_char_p, []),
    "pxq_init": (_i, [_i]),
    "pxq_weight_bytes": (_u64, [_u64, _u64, _u32]),
    "pxq_quantize_q8_0": (_i, [_vp, _vp, _sz, _sz, _vp]),
    "pxq_quantize_q8_K": (_i, [_vp, _vp, _sz, _sz, _vp]),
    "pxq_quantize_q8_K_matvec": (_i, [_vp, _vp, _sz, _sz, _vp]),
    "pxq_decode": (_i, [_vp, _u32, _sz, _vp, _vp]),
    "pxq_weight_upload": (_i, [_vp, _i, _u32, _sz, _sz, C.c_char_p, C.POINTER(_vp)]),
    "pxq_weight_upload_gated": (_i, [_vp, _vp, _i, _u32, _sz, _sz, C.c_char_p, C.POINTER(_vp)]),
    "pxq_matmul_gated": (_i, [_vp, _vp, _sz, _vp, _sz, _vp]),
    "pxq_weight_release": (_i, [_vp]),
    "pxq_weight_cache_clear": (_i, []),
    "pxq_weight_cache_limit": (_i, [_u64]),
    "pxq_weight_cache_usage": (_i, [C.POINTER(_u64), C.POINTER(_u64), C.POINTER(_u64)]),
    "pxq_matmul": (_i, [_vp, _sz, _sz, _vp, _sz, _vp, _sz, _vp, _vp]),
    "pxq_matvec": (_i, [_vp, _sz, _sz, _vp, _sz, _vp, _sz, _vp, _vp]),
    "pxq_gemm": (_i, [_vp, _sz, _sz, _vp, _sz, _vp, _sz, _vp, _vp]),
    "pxq_quant_matmul": (_i, [_vp, _u32, _vp, _vp, _sz, _sz, _sz]),
    "pxq_matmul_host": (_i, [_vp, _sz, _sz, _vp, _sz, _vp, _sz]),
    "pxq_synchronize": (_i, [_vp]),
    "pxq_gather_shards": (_i, [_vp, _sz, _sz, _sz, _vp, _sz, _vp]),
    "pxq_matmul_scatter": (_i, [_vp, _sz, _sz, _vp, _sz, _vp, _sz, _sz, _sz, _vp]),
    "pxq_ipc_alloc": (_i, [_sz, _vp, _vp]),
    "pxq_ipc_free": (_i, [_vp]),
    "pxq_ipc_open": (_i, [_vp, _vp]),
    "pxq_ipc_close": (_i, [_vp]),
    "pxq_gemm_block_dots": (_i, [_vp, _sz, _sz, _vp, _sz, _vp, _vp]),
    "pxq_activation_quantize": (_i, [_u32, _vp, _sz, _sz, C.POINTER(_vp), _vp]),
    "pxq_matmul_quantized": (_i, [_vp, _sz, _sz, _vp, _vp, _sz, _vp, _vp]),
    "pxq_activation_release": (_i, [_vp, _vp]),
    "pxq_kernel_launches": (_u64, []),
    "pxq_matvec_noalloc": (_i, [_vp, _sz, _sz, _vp, _sz, _vp, _sz, _vp, _vp]),
    "pxq_debug_matvec_stall": (_i, [_vp, _vp, _sz, _vp, _i, _vp]),
    "pxq_comm_unique_id": (_i, [_vp]),
    "pxq_comm_init": (_i, [_vp, _i, _i, _i, C.POINTER(_vp)]),
    "pxq_comm_size": (_i, [_vp, C.POINTER(_i), C.POINTER(_i)]),
    "pxq_comm_barrier": (_i, [_vp]),
    "pxq_comm_synchronize": (_i, [_vp, _vp]),
    "pxq_comm_destroy": (_i, [_vp]),
    "pxq_sharded_output_create": (_i, [_vp, _sz, _sz, C.POINTER(_vp), C.POINTER(_vp)]),
    "pxq_sharded_output_destroy": (_i, [_vp]),
    "pxq_sharded_matmul": (_i, [_vp, _vp, _sz, _vp, _sz, _vp, _vp, _sz, _vp]),
    "pxq_sharded_matmul_host": (_i, [_vp, _vp, _sz, _vp, _sz, _sz, _vp]),
    "pxq_attention": (_i, [_vp, _sz, _vp, _vp, _sz, _sz, _sz, _sz, _vp, _sz, _sz, _vp, _vp]),
    "pxq_kv_cache_bytes": (_u64, [_sz, _sz, _sz, _sz]),
    "pxq_kv_cache_create": (_i, [_vp, _sz, _sz, _sz, _sz, C.POINTER(_vp), _vp]),
    "pxq_kv_cache_release": (_i, [_vp]),
    "pxq_kv_cache_lengths": (_i, [_vp, _vp, _vp]),
    "pxq_kv_append": (_i, [_vp, _vp, _sz, _vp, _sz, _sz, _vp, _vp]),
    "pxq_kv_truncate": (_i, [_vp, _vp, _vp]),
    "pxq_kv_read": (_i, [_vp, _vp, _sz, _vp, _vp, _vp]),
    "pxq_kv_attention": (_i, [_vp, _vp, _sz, _sz, _vp, _sz, _sz, _i, _vp, _sz, _vp, _vp, _vp]),
    "pxq_kv_evict": (_i, [_vp, _vp, _vp, _sz, _sz, _vp, _vp, _vp]),
    "pxq_gguf_open": (_i, [C.c_char_p, C.POINTER(_vp)]),
    "pxq_gguf_close": (_i, [_vp]),
    "pxq_gguf_tensor_count": (_sz, [_vp]),
    "pxq_gguf_metadata_count": (_sz, [_vp]),
    "pxq_gguf_data": (_vp, [_vp]),
    "pxq_gguf_tensor_at": (_i, [_vp, _sz, _vp]),
    "pxq_gguf_find": (_i, [_vp, C.c_char_p, _vp]),
    "pxq_gguf_upload": (_i, [_vp, C.c_char_p, _sz, _sz, C.POINTER(_vp)]),
    "pxq_gguf_upload_gated": (_i, [_vp, C.c_char_p, _sz, C.c_char_p, _sz, _sz, C.POINTER(_vp)]),
}


class GGUFTensor(C.Structure):
    """pxq_gguf_tensor (include/pxq.h)."""

    _fields_ = [("name", C.c_char_p), ("type", C.c_uint32), ("rank", C.c_uint32), ("shape", C.c_uint64 * 5),
                ("offset", C.c_uint64), ("bytes", C.c_uint64)]

    def as_dict(self) -> dict:
        return {"name": self.name.decode(), "type": int(self.type), "shape": [int(v) for v in self.shape[:self.rank]],
                "offset": int(self.offset), "bytes": int(self.bytes)}


class PxqError(RuntimeError):
    def __init__(self, code: int, msg: str):
        super().__init__(f"pxq error {code}: {msg}")
        self.code = code


_lib = None


def load(path: str = LIB_PATH):
    """Load libpxq.so (raises if it has not been built)."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(path):
        raise ImportError(f"{path} is missing: build it with `python -c 'import __graft_entry__ as g; g.build()'`")
    lib = C.CDLL(path)
    for name, (res, args) in SIGNATURES.items():
        f = getattr(lib, name)
        f.restype = res
        f.argtypes = args
    _lib = lib
    return lib


def _check(rc: int) -> None:
    if rc != OK:
        raise PxqError(rc, load().pxq_last_error().decode(errors="replace"))


def last_error() -> str:
    return load().pxq_last_error().decode(errors="replace")


def weight_bytes(inner: int, rows: int, wtype: int) -> int:
    return int(load().pxq_weight_bytes(inner, rows, wtype))


# ------------------------------------------------------------ device side ---

_torch_module = None


def _torch():
    global _torch_module
    if _torch_module is None:
        import torch  # noqa: WPS433 (device memory and streams only)

        _torch_module = torch
    return _torch_module


def _stream_ptr(stream=None):
    if stream is not None:
        return C.c_void_p(stream.cuda_stream)
    torch = _torch()
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # the current stream without a Stream object around it
    if raw is not None:
        return C.c_void_p(raw(torch.cuda.current_device()))
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _ptr(t) -> C.c_void_p:
    return C.c_void_p(t.data_ptr()) if t is not None else C.c_void_p(0)


def init(device: int = 0) -> None:
    torch = _torch()
    torch.cuda.set_device(device)
    _check(load().pxq_init(device))


def quantize_q8_0(x, stream=None):
    """fp32 [rows, inner] cuda tensor -> uint8 [rows, inner/32*34] GGUF Q8_0 blocks."""
    torch = _torch()
    x = x.contiguous()
    rows, inner = x.shape
    out = torch.empty((rows, inner // 32 * Q8_0_BYTES), dtype=torch.uint8, device=x.device)
    _check(load().pxq_quantize_q8_0(_ptr(x), _ptr(out), rows, inner, _stream_ptr(stream)))
    return out


def quantize_q8_K(x, stream=None):
    """fp32 [rows, inner] cuda tensor -> uint8 [rows, inner/256*292] Q8_K blocks."""
    torch = _torch()
    x = x.contiguous()
    rows, inner = x.shape
    out = torch.empty((rows, inner // 256 * Q8_K_BYTES), dtype=torch.uint8, device=x.device)
    _check(load().pxq_quantize_q8_K(_ptr(x), _ptr(out), rows, inner, _stream_ptr(stream)))
    return out


Q8K_MATVEC_BYTES = 288


def quantize_q8_K_matvec(x, stream=None):
    """fp32 [rows <= 8, inner] cuda tensor -> uint8 [rows, inner/256*288] matvec
    records (the Q8_K quants, permuted, plus 32-element sums and d)."""
    torch = _torch()
    x = x.contiguous()
    rows, inner = x.shape
    out = torch.empty((rows, inner // 256 * Q8K_MATVEC_BYTES), dtype=torch.uint8, device=x.device)
    _check(load().pxq_quantize_q8_K_matvec(_ptr(x), _ptr(out), rows, inner, _stream_ptr(stream)))
    return out


def decode(data, wtype: int, count: int, stream=None):
    torch = _torch()
    out = torch.empty(count, dtype=torch.float32, device=data.device)
    _check(load().pxq_decode(_ptr(data), wtype, count, _ptr(out), _stream_ptr(stream)))
    return out


class Weight:
    """A GGUF weight tensor resident on the current device."""

    def __init__(self, data, wtype: int, inner: int, rows: int, key: Optional[str] = None):
        lib = load()
        self.wtype, self.inner, self.rows = wtype, inner, rows
        handle = C.c_void_p()
        if hasattr(data, "data_ptr"):  # torch tensor (host or device)
            on_dev = 1 if data.is_cuda else 0
            ptr = C.c_void_p(data.data_ptr())
            self._keep = data
        else:
            arr = np.ascontiguousarray(data, dtype=np.uint8)
            on_dev, ptr = 0, arr.ctypes.data_as(C.c_void_p)
            self._keep = arr
        kb = key.encode() if key else None
        _check(lib.pxq_weight_upload(ptr, on_dev, wtype, inner, rows, kb, C.byref(handle)))
        self.handle = handle
        self._keep = None

    def release(self) -> None:
        if self.handle:
            _check(load().pxq_weight_release(self.handle))
            self.handle = C.c_void_p()


class GatedWeight:
    """The gate and up projections of a gated feed-forward, resident on the
    current device as one weight (pxq_weight_upload_gated)."""

    def __init__(self, gate, up, wtype: int, inner: int, rows: int, key: Optional[str] = None):
        lib = load()
        self.wtype, self.inner, self.rows = wtype, inner, rows
        keep, ptrs, on_dev = [], [], 0
        for data in (gate, up):
            if hasattr(data, "data_ptr"):
                on_dev = 1 if data.is_cuda else 0
                ptrs.append(C.c_void_p(data.data_ptr()))
                keep.append(data)
            else:
                arr = np.ascontiguousarray(data, dtype=np.uint8)
                ptrs.append(arr.ctypes.data_as(C.c_void_p))
                keep.append(arr)
        handle = C.c_void_p()
        kb = key.encode() if key else None
        _check(lib.pxq_weight_upload_gated(ptrs[0], ptrs[1], on_dev, wtype, inner, rows, kb, C.byref(handle)))
        self.handle = handle

    def release(self) -> None:
        if self.handle:
            _check(load().pxq_weight_release(self.handle))
            self.handle = C.c_void_p()


class AttentionRange(C.Structure):
    """pxq_attention_range (include/pxq.h)."""

    _fields_ = [("query_begin", C.c_size_t), ("query_end", C.c_size_t), ("key_end", C.c_size_t), ("causal", C.c_int)]


def attention(q, k, v, heads: int, kv_heads: int, ranges=None, query_offset: int = 0, causal: bool = False, out=None,
              stream=None):
    """tensor_attention on device fp32 tensors q [rows][heads*d], k, v [keys][kv_heads*d].
    ranges: [(query_begin, query_end, key_end, causal)] (the second overload);
    None: one range over all rows and keys with `causal` (the first overload)."""
    torch = _torch()
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    rows, keys = q.shape[0], k.shape[0]
    d = q.shape[1] // heads
    if ranges is None:
        ranges = [(0, rows, keys, causal)]
    arr = (AttentionRange * len(ranges))(*[AttentionRange(b, e, ke, 1 if c else 0) for b, e, ke, c in ranges])
    if out is None:
        out = torch.empty_like(q)
    _check(load().pxq_attention(_ptr(q), rows, _ptr(k), _ptr(v), keys, heads, kv_heads, d, C.cast(arr, C.c_void_p), len(ranges),
                                query_offset, _ptr(out), _stream_ptr(stream)))
    return out


def _on(stream):
    """Tensors made within belong to the stream that the call runs on."""
    return contextlib.nullcontext() if stream is None else _torch().cuda.stream(stream)


def _kv_stream(stream, device):
    """Address of the stream, or of the device's current one."""
    if stream is not None:
        return stream.cuda_stream
    raw = getattr(_torch()._C, "_cuda_getCurrentRawStream", None)
    return raw(device.index) if raw is not None else _torch().cuda.current_stream(device).cuda_stream


def _rows(x, width: int, what: str, device, stream=None):
    """An fp32 matrix of `width` columns on `device` whose rows may be strided,
    and its row stride (of one row: its width, whatever torch says).  A copy,
    where one is needed, is made on the stream that the call runs on."""
    shape = x.shape
    if x.dtype is not _torch().float32 or len(shape) != 2 or shape[1] != width or x.device != device:
        raise ValueError(f"{what} must be fp32 [rows, {width}] on {device}")
    if x.is_contiguous():
        return x, width
    ld, step = x.stride()
    if step != 1 or ld < width:
        with _on(stream):
            return x.contiguous(), width
    return x, ld if shape[0] > 1 else width


def _whole(x, shape, dtype, what: str, device):
    """Address of a contiguous tensor of this shape and type on `device`; None for None."""
    if x is None:
        return None
    if x.shape != shape or x.dtype is not dtype or not x.is_contiguous() or x.device != device:
        raise ValueError(f"{what} must be a contiguous {dtype} tensor of shape {shape} on {device}")
    return x.data_ptr()


class KVCache:
    """An 8-bit key/value cache (pxq_kv_cache) for `sequences` sequences of up
    to `capacity` tokens; its memory is a torch tensor of its own."""

    def __init__(self, sequences: int, capacity: int, kv_heads: int, head_dim: int, stream=None):
        torch = _torch()
        lib = load()
        nbytes = int(lib.pxq_kv_cache_bytes(sequences, capacity, kv_heads, head_dim))
        if not nbytes:
            raise PxqError(ERR_UNSUPPORTED, last_error())
        self.sequences, self.capacity, self.kv_heads, self.head_dim = sequences, capacity, kv_heads, head_dim
        with _on(stream):
            self.memory = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
        self.device = self.memory.device
        h = C.c_void_p()
        at = _kv_stream(stream, self.device)
        self._streams = {at}  # that torch knows to work on the memory
        _check(lib.pxq_kv_cache_create(self.memory.data_ptr(), sequences, capacity, kv_heads, head_dim, C.byref(h), at))
        self.handle = h

    def release(self) -> None:
        """Forget the cache; its memory goes back to torch, which hands it out
        again when every stream that worked on it is done.  (cudaStreamPerThread
        is another stream in every thread, and torch only knows the releasing one's: wait for the others first.)"""
        if self.handle:
            _check(load().pxq_kv_cache_release(self.handle))
            self.handle, self.memory = C.c_void_p(), None

    def _on_stream(self, stream):
        """Address of the stream that a call runs on, which torch is told of where the memory is another stream's."""
        at = _kv_stream(stream, self.device)
        if at not in self._streams:
            self.memory.record_stream(stream if stream is not None else _torch().cuda.current_stream(self.device))
            self._streams.add(at)
        return at

    def __del__(self):
        if getattr(self, "handle", None) and _lib is not None:
            _lib.pxq_kv_cache_release(self.handle)
            self.handle = C.c_void_p()

    def _live(self):
        if not self.handle:
            raise ValueError("the cache was released")
        return self.handle

    def _per_sequence(self, x, what: str, more: int = 0):
        return None if x is None else _whole(x, (self.sequences + more,), _torch().int32, what, self.device)

    def lengths(self, stream=None):
        """The sequences' lengths: int32 cuda tensor."""
        h = self._live()
        with _on(stream):
            out = _torch().empty(self.sequences, dtype=_torch().int32, device=self.device)
        _check(load().pxq_kv_cache_lengths(h, out.data_ptr(), self._on_stream(stream)))
        return out

    def append(self, k, v, starts=None, stream=None) -> None:
        """Append rows k, v [rows, kv_heads*d]; rows [starts[s], starts[s+1]) go to sequence s."""
        h = self._live()
        width = self.kv_heads * self.head_dim
        k, ldk = _rows(k, width, "k", self.device, stream)
        v, ldv = _rows(v, width, "v", self.device, stream)
        if k.shape[0] != v.shape[0]:
            raise ValueError(f"k has {k.shape[0]} rows, v {v.shape[0]}")
        _check(load().pxq_kv_append(h, k.data_ptr(), ldk, v.data_ptr(), ldv, k.shape[0], self._per_sequence(starts, "starts", 1),
                                    self._on_stream(stream)))

    def truncate(self, lengths=None, stream=None) -> None:
        """Shorten the sequences to `lengths` (int32 cuda tensor; None: empty them).
        Running totals of weights stay: set those of the dropped tokens to zero."""
        _check(load().pxq_kv_truncate(self._live(), self._per_sequence(lengths, "lengths"), self._on_stream(stream)))

    def read(self, first=None, count: Optional[int] = None, k=None, v=None, stream=None):
        """The values of tokens [first[s], first[s] + count) of every sequence:
        k, v [sequences, count, kv_heads*d].  Rows past a sequence's length are
        not written (zeros in tensors made here)."""
        torch = _torch()
        h = self._live()
        count = self.capacity if count is None else count
        shape = (self.sequences, count, self.kv_heads * self.head_dim)
        if k is None or v is None:
            with _on(stream):
                k = torch.zeros(shape, device=self.device) if k is None else k
                v = torch.zeros(shape, device=self.device) if v is None else v
        _check(load().pxq_kv_read(h, self._per_sequence(first, "first"), count, _whole(k, shape, torch.float32, "k", self.device),
                                  _whole(v, shape, torch.float32, "v", self.device), self._on_stream(stream)))
        return k, v


def kv_attention(q, cache: KVCache, heads: int, starts=None, max_rows: Optional[int] = None, causal: bool = True, weights=None,
                 weights_out=None, out=None, stream=None):
    """Attention of q [rows, heads*d] over the cache (pxq_kv_attention): rows
    [starts[s], starts[s+1]) are sequence s's, at most max_rows of them each
    (None: no bound but rows, which plans for a prompt).  weights_out = weights + what each cached token
    received, [sequences, kv_heads, capacity]."""
    torch = _torch()
    h, device = cache._live(), cache.device
    width = heads * cache.head_dim
    q, ldq = _rows(q, width, "q", device, stream)
    rows, ldo = q.shape[0], width
    if out is None:
        if stream is None:
            out = q.new_empty((rows, width))
        else:
            with _on(stream):
                out = q.new_empty((rows, width))
    elif out.shape != (rows, width) or out.dtype is not torch.float32 or out.device != device or out.stride(1) != 1 or \
            (rows > 1 and out.stride(0) < width):
        raise ValueError(f"out must be fp32 [{rows}, {width}] on {device}, its rows contiguous")
    elif rows > 1:
        ldo = out.stride(0)
    wi = wo = None
    if weights is not None or weights_out is not None:
        shape = (cache.sequences, cache.kv_heads, cache.capacity)
        wi = _whole(weights, shape, torch.float32, "weights", device)
        wo = _whole(weights_out, shape, torch.float32, "weights_out", device)
    _check(load().pxq_kv_attention(h, q.data_ptr(), ldq, rows, cache._per_sequence(starts, "starts", 1), rows if max_rows is None else max_rows, heads,
                                   1 if causal else 0, out.data_ptr(), ldo, wi, wo, cache._on_stream(stream)))
    return out


def kv_evict(src: KVCache, dst: KVCache, weights, keep: Optional[int] = None, recent: int = 0, weights_out=None, kept=None,
             stream=None) -> None:
    """Into dst: the last `recent` tokens of src's every (sequence, kv head) and
    the heaviest others, `keep` in all (None: dst's capacity) (pxq_kv_evict)."""
    torch = _torch()
    a, b = src._live(), dst._live()
    keep = dst.capacity if keep is None else keep
    if weights is None:
        raise ValueError("weights are needed")
    heads = (src.sequences, src.kv_heads)
    dst._on_stream(stream)
    _check(load().pxq_kv_evict(a, b, _whole(weights, heads + (src.capacity,), torch.float32, "weights", src.device), keep, recent,
                               _whole(weights_out, (dst.sequences, dst.kv_heads, dst.capacity), torch.float32, "weights_out", src.device),
                               _whole(kept, heads + (keep,), torch.int32, "kept", src.device), src._on_stream(stream)))


class _Uploaded:
    """A weight uploaded from a model file (pxq_gguf_upload*)."""

    def __init__(self, handle, wtype: int, inner: int, rows: int):
        self.handle, self.wtype, self.inner, self.rows = handle, wtype, inner, rows

    def release(self) -> None:
        if self.handle:
            _check(load().pxq_weight_release(self.handle))
            self.handle = C.c_void_p()


class GGUF:
    """A GGUF model file opened with pxq_gguf_open (a read-only mapping)."""

    def __init__(self, path: str):
        h = C.c_void_p()
        _check(load().pxq_gguf_open(path.encode(), C.byref(h)))
        self.handle, self.path = h, path

    def close(self) -> None:
        if self.handle:
            load().pxq_gguf_close(self.handle)
            self.handle = C.c_void_p()

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    @property
    def metadata_count(self) -> int:
        return int(load().pxq_gguf_metadata_count(self.handle))

    def tensors(self) -> list:
        lib = load()
        out = []
        for i in range(int(lib.pxq_gguf_tensor_count(self.handle))):
            t = GGUFTensor()
            _check(lib.pxq_gguf_tensor_at(self.handle, i, C.byref(t)))
            out.append(t.as_dict())
        return out

    def find(self, name: str) -> dict:
        t = GGUFTensor()
        _check(load().pxq_gguf_find(self.handle, name.encode(), C.byref(t)))
        return t.as_dict()

    def upload(self, name: str, row_first: int = 0, row_count: int = 0) -> _Uploaded:
        t = self.find(name)
        rows = 1
        for v in t["shape"][1:]:
            rows *= v
        h = C.c_void_p()
        _check(load().pxq_gguf_upload(self.handle, name.encode(), row_first, row_count, C.byref(h)))
        return _Uploaded(h, t["type"], t["shape"][0], row_count or rows - row_first)

    def upload_gated(self, gate: str, gate_first: int, up: str, up_first: int, rows: int) -> _Uploaded:
        t = self.find(gate)
        h = C.c_void_p()
        _check(load().pxq_gguf_upload_gated(self.handle, gate.encode(), gate_first, up.encode(), up_first, rows, C.byref(h)))
        return _Uploaded(h, t["type"], t["shape"][0], rows)


def matmul_gated(w: GatedWeight, x, out=None, ldy: Optional[int] = None, stream=None):
    """Y[c, r] = silu(x[c] . gate[r]) * (x[c] . up[r]) on the device."""
    torch = _torch()
    x = x.contiguous()
    columns, inner = x.shape
    if inner != w.inner:
        raise ValueError(f"input has {inner} features, weight expects {w.inner}")
    if out is None:
        out = torch.empty((columns, w.rows), dtype=torch.float32, device=x.device)
        ldy = w.rows
    elif ldy is None:
        ldy = out.stride(0)
    _check(load().pxq_matmul_gated(w.handle, _ptr(x), columns, _ptr(out), ldy, _stream_ptr(stream)))
    return out


def matmul(w: Weight, x, row_first: int = 0, row_count: Optional[int] = None, bias=None, out=None, ldy: Optional[int] = None,
           path: str = "auto", stream=None):
    """Y[c, r] = sum_k x[c, k] * W[row_first + r, k] (+ bias[r]) on the device."""
    torch = _torch()
    x = x.contiguous()
    columns, inner = x.shape
    if inner != w.inner:
        raise ValueError(f"input has {inner} features, weight expects {w.inner}")
    rc = w.rows - row_first if row_count is None else row_count
    if out is None:
        out = torch.empty((columns, rc), dtype=torch.float32, device=x.device)
        ldy = rc
    elif ldy is None:
        ldy = out.stride(0)
    fn = {"auto": load().pxq_matmul, "matvec": load().pxq_matvec, "gemm": load().pxq_gemm}[path]
    _check(fn(w.handle, row_first, rc, _ptr(x), columns, _ptr(out), ldy, _ptr(bias), _stream_ptr(stream)))
    return out


def gemm_block_dots(w: Weight, x, row_first: int = 0, row_count: Optional[int] = None, stream=None):
    """Exact per-block dots from the tensor-core GEMM: [items, columns, rows]."""
    torch = _torch()
    x = x.contiguous()
    columns, inner = x.shape
    rc = w.rows - row_first if row_count is None else row_count
    items = {TYPE_Q8_0: inner // 32, TYPE_Q5_K: 5 * (inner // 256), TYPE_Q6_K: 4 * (inner // 256)}[w.wtype]
    dump = torch.zeros((items, columns, rc), dtype=torch.float32, device=x.device)
    _check(load().pxq_gemm_block_dots(w.handle, row_first, rc, _ptr(x), columns, _ptr(dump), _stream_ptr(stream)))
    return dump


class Activation:
    """An activation quantized once for weights of one type (pxq_activation)."""

    def __init__(self, wtype: int, x, stream=None):
        self.x = x.contiguous()
        self.columns, self.inner = self.x.shape
        self.wtype = wtype
        h = C.c_void_p()
        _check(load().pxq_activation_quantize(wtype, _ptr(self.x), self.columns, self.inner, C.byref(h),
                                              _stream_ptr(stream)))
        self.handle = h

    def release(self, stream=None) -> None:
        if self.handle:
            _check(load().pxq_activation_release(self.handle, _stream_ptr(stream)))
            self.handle = C.c_void_p()


def matmul_quantized(w: Weight, a: Activation, row_first: int = 0, row_count: Optional[int] = None, bias=None, out=None,
                     ldy: Optional[int] = None, stream=None):
    torch = _torch()
    rc = w.rows - row_first if row_count is None else row_count
    if out is None:
        out = torch.empty((a.columns, rc), dtype=torch.float32, device=a.x.device)
        ldy = rc
    elif ldy is None:
        ldy = out.stride(0)
    _check(load().pxq_matmul_quantized(w.handle, row_first, rc, a.handle, _ptr(out), ldy, _ptr(bias), _stream_ptr(stream)))
    return out


def cache_limit(nbytes: int) -> None:
    """pxq_weight_cache_limit: the weight cache's budget on this device (0: default)."""
    _check(load().pxq_weight_cache_limit(nbytes))


def cache_usage() -> tuple[int, int, int]:
    """pxq_weight_cache_usage: (cached bytes, budget, entries) on this device."""
    b, l, n = C.c_uint64(), C.c_uint64(), C.c_uint64()
    _check(load().pxq_weight_cache_usage(C.byref(b), C.byref(l), C.byref(n)))
    return b.value, l.value, n.value


def kernel_launches() -> int:
    return int(load().pxq_kernel_launches())


def gather_shards(src, shards: int, columns: int, shard_rows: int, out=None, stream=None):
    torch = _torch()
    if out is None:
        out = torch.empty((columns, shards * shard_rows), dtype=torch.float32, device=src.device)
    _check(load().pxq_gather_shards(_ptr(src), shards, columns, shard_rows, _ptr(out), out.stride(0), _stream_ptr(stream)))
    return out


IPC_HANDLE_BYTES = 64


class IpcBuffer:
    """fp32 device buffer [rows][cols] that other processes of the node can
    map (pxq_ipc_alloc); ``handle`` is its 64-byte CUDA IPC handle and
    ``tensor`` a torch view of it on this device."""

    def __init__(self, rows: int, cols: int):
        torch = _torch()
        ptr, handle = C.c_void_p(), (C.c_uint8 * IPC_HANDLE_BYTES)()
        _check(load().pxq_ipc_alloc(rows * cols * 4, C.byref(ptr), C.cast(handle, C.c_void_p)))
        self.ptr, self.handle, self.shape = ptr.value, bytes(handle), (rows, cols)
        self.tensor = torch.as_tensor(_CudaArray(self.ptr, self.shape), device="cuda")

    def free(self) -> None:
        if self.ptr:
            self.tensor = None
            _check(load().pxq_ipc_free(C.c_void_p(self.ptr)))
            self.ptr = None


class IpcPeer:
    """Another process's IpcBuffer opened in this one (pxq_ipc_open)."""

    def __init__(self, handle: bytes):
        ptr = C.c_void_p()
        buf = (C.c_uint8 * IPC_HANDLE_BYTES).from_buffer_copy(handle)
        _check(load().pxq_ipc_open(C.cast(buf, C.c_void_p), C.byref(ptr)))
        self.ptr = ptr.value

    def close(self) -> None:
        if self.ptr:
            _check(load().pxq_ipc_close(C.c_void_p(self.ptr)))
            self.ptr = None


class _CudaArray:
    """Minimal __cuda_array_interface__ over a raw fp32 device pointer."""

    def __init__(self, ptr: int, shape):
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": "<f4", "data": (ptr, False), "version": 2}


def matmul_scatter(W: "Weight", x, dst_ptrs, ldy: int, col_offset: int, row_first: int = 0, row_count=None, stream=None):
    """pxq_matmul_scatter: rows [row_first, row_first + row_count) of W times
    x (device fp32 [M][K], M > 8), every element written to each pointer of
    ``dst_ptrs`` at [m][col_offset + n] with row stride ``ldy``; dst_ptrs[0]
    is this GPU's own buffer, the rest the other ranks' (pxq_ipc_open)."""
    x = x.contiguous()
    row_count = W.rows - row_first if row_count is None else row_count
    arr = (C.c_void_p * len(dst_ptrs))(*[C.c_void_p(p) for p in dst_ptrs])
    _check(load().pxq_matmul_scatter(W.handle, row_first, row_count, _ptr(x), x.shape[0], C.cast(arr, C.c_void_p), len(dst_ptrs),
                                     ldy, col_offset, _stream_ptr(stream)))


def synchronize(stream=None) -> None:
    _check(load().pxq_synchronize(_stream_ptr(stream)))


# --------------------------------------------------------------- host side ---

def quant_matmul(weights: np.ndarray, wtype: int, x: np.ndarray, rows: int):
    """cpu_quant_matmul with host buffers: returns (handled, Y[columns, rows])."""
    x = np.ascontiguousarray(x, dtype=np.float32)
    columns, inner = x.shape
    w = np.ascontiguousarray(weights, dtype=np.uint8)
    y = np.empty((columns, rows), dtype=np.float32)
    rc = load().pxq_quant_matmul(w.ctypes.data_as(C.c_void_p), wtype, x.ctypes.data_as(C.c_void_p),
                                 y.ctypes.data_as(C.c_void_p), rows, columns, inner)
    if rc == ERR_UNSUPPORTED:
        return False, y
    _check(rc)
    return True, y


def quant_matmul_ptr(weights_ptr: int, wtype: int, x_ptr: int, y_ptr: int, rows: int, columns: int, inner: int) -> int:
    """Raw-pointer form of pxq_quant_matmul (host addresses); returns the status."""
    return int(load().pxq_quant_matmul(C.c_void_p(weights_ptr), wtype, C.c_void_p(x_ptr), C.c_void_p(y_ptr), rows, columns,
                                       inner))
