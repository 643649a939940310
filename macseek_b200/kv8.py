"""Grouped-query heads over a paged cache in 8 bits: writing new rows, reading rows back, attention (the msb_kv8_* calls;
no counterpart in the reference, whose attention is `attn`).  Codes are e4m3 with one power-of-two scale per block of tokens
and head; a batch of sequences is described by device arrays, so that a captured call follows them from replay to replay."""
import ctypes as C

import torch

from . import _lib
from .core import Enc

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}      # MSB_F32, MSB_F16, MSB_BF16


def _want(ok, what):
    if not ok:
        raise _lib.MsbError(what)


def _fits(what, *numbers):
    """Numbers that the C calls take in 32 bits, not negative."""
    for x in numbers:
        if not 0 <= x <= 0x7fffffff:
            raise _lib.MsbError("%s: %d is negative or does not fit 32 bits" % (what, x))


_current = torch.cuda.current_device


def _elsewhere(e, device, fn, *args):
    """fn(*args, stream) on a device that is not the current one (the library works on the current device); it has to be the stream's."""
    if e.stream.device_index != device.index:
        raise _lib.MsbError("tensors on %s, the stream on %s" % (device, e.stream.device))
    with torch.cuda.device(device):
        return fn(*args, e.stream.cuda_stream)


class Cache:
    """Codes uint8 [n_blocks][kv_heads][block][head_dim] and scales F32 [n_blocks][kv_heads] of keys and of values."""

    def __init__(self, n_blocks, kv_heads, head_dim, block=64, device="cuda"):
        codes = lambda: torch.zeros(n_blocks, kv_heads, block, head_dim, dtype=torch.uint8, device=device)  # noqa: E731
        scale = lambda: torch.ones(n_blocks, kv_heads, dtype=torch.float32, device=device)  # noqa: E731
        self._set(codes(), codes(), scale(), scale())

    @classmethod
    def of(cls, k, v, k_scale, v_scale):
        """Over tensors that exist."""
        c = cls.__new__(cls)
        c._set(k, v, k_scale, v_scale)
        return c

    def _set(self, k, v, k_scale, v_scale):
        self.device, self.index = k.device, k.device.index
        for name, t, dt, shape in (("k", k, torch.uint8, k.shape), ("v", v, torch.uint8, k.shape),
                                   ("k_scale", k_scale, torch.float32, k.shape[:2]), ("v_scale", v_scale, torch.float32, k.shape[:2])):
            _want(t.is_cuda and t.device == self.device, "kv8 cache: %s must be on one CUDA device" % name)
            _want(t.dtype == dt and t.shape == shape and t.is_contiguous() and k.dim() == 4,
                  "kv8 cache: %s must be contiguous %s %s" % (name, dt, tuple(shape)))
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.n_blocks, self.kv_heads, self.block, self.head_dim = k.shape
        self.c = _lib.Kv8CacheC(self.n_blocks, self.kv_heads, self.head_dim, self.block, k.data_ptr(), v.data_ptr(),
                                k_scale.data_ptr(), v_scale.data_ptr())
        self.ref, self.addr = C.byref(self.c), C.addressof(self.c)


class Batch:
    """seq_start int32 [n + 1], kv_len int32 [n] (new tokens included), table int32 [n][blocks]; n_tokens rows in a call's
    tensors, at most max_new new tokens and max_len tokens in any sequence."""

    def __init__(self, seq_start, kv_len, table, n_tokens, max_new, max_len):
        n = kv_len.shape[0]
        _fits("kv8 batch", n, n_tokens, max_new, max_len, table.shape[-1])
        self.device, self.index = kv_len.device, kv_len.device.index
        for name, t, shape in (("seq_start", seq_start, (n + 1,)), ("kv_len", kv_len, (n,)), ("table", table, (n, table.shape[-1]))):
            _want(t.is_cuda and t.device == self.device, "kv8 batch: %s must be on one CUDA device" % name)
            _want(t.dtype == torch.int32 and tuple(t.shape) == shape and t.is_contiguous(),
                  "kv8 batch: %s must be contiguous int32 %s" % (name, shape))
        self.seq_start, self.kv_len, self.table = seq_start, kv_len, table
        self.n_seq, self.n_tokens, self.max_new, self.max_len = n, n_tokens, max_new, max_len
        self.c = _lib.Kv8BatchC(n, n_tokens, max_new, max_len, seq_start.data_ptr(), kv_len.data_ptr(), table.data_ptr(),
                                table.shape[1])
        self.ref, self.addr = C.byref(self.c), C.addressof(self.c)


def _rows(name, t, n_tokens, heads, dim, device):
    """MSB type of rows [n_tokens][heads][dim] whose heads are dense (tokens may be apart)."""
    _want(t.device == device, "%s is on %s, not on %s" % (name, t.device, device))
    _want(tuple(t.shape) == (n_tokens, heads, dim) and t.stride(2) == 1 and (t.stride(1) == dim or heads == 1),
          "%s must be [%d][%d][%d] with dense heads" % (name, n_tokens, heads, dim))
    ty = DTYPES.get(t.dtype)
    _want(ty is not None, "%s must be float32, float16 or bfloat16" % name)
    return ty


_WRITE, _READ, _ATTN = (_lib.address(f) for f in (_lib.lib.msb_kv8_write, _lib.lib.msb_kv8_read, _lib.lib.msb_kv8_attn))


def _kv(e, cache, batch, k, v, call, what):
    i, st, dev = cache.index, e.stream, cache.device
    if batch.index != i:
        rc = 1
    elif st.device_index == i == _current():
        rc = _lib.host().msb_host_kv8_rows(k, v, cache.addr, batch.addr, i, call, st.cuda_stream)
    else:
        rc = _elsewhere(e, dev, _lib.host().msb_host_kv8_rows, k, v, cache.addr, batch.addr, i, call)
    if rc > 0:                     # not plainly right: say why
        _want(batch.device == dev, "%s: cache and batch on different devices" % what)
        ty = _rows("k", k, batch.n_tokens, cache.kv_heads, cache.head_dim, dev)
        _want(_rows("v", v, batch.n_tokens, cache.kv_heads, cache.head_dim, dev) == ty, "k and v must be of one type")
        _want(False, "%s: k and v must be rows of the batch and the cache" % what)
    _lib.check(rc)


def encode_kv8_write(e: Enc, cache: Cache, batch: Batch, k, v):
    """New rows k, v [n_tokens][kv_heads][head_dim] into the cache."""
    _kv(e, cache, batch, k, v, _WRITE, "kv8_write")


def encode_kv8_read(e: Enc, cache: Cache, batch: Batch, k, v):
    """The batch's rows of the cache into k, v."""
    _kv(e, cache, batch, k, v, _READ, "kv8_read")


def attn_scratch(cache: Cache, batch: Batch, heads):
    """Scratch of encode_kv8_attn for this cache and batch (any window); calls that overlap in time need one each."""
    _fits("kv8: heads", heads)
    with torch.cuda.device(cache.device):
        n = _lib.lib.msb_kv8_attn_scratch_bytes(cache.ref, batch.ref, heads)
    _want(n > 0, "kv8: " + _lib.lib.msb_last_error().decode())
    return torch.empty(n, dtype=torch.uint8, device=cache.device)


def encode_kv8_attn(e: Enc, cache: Cache, batch: Batch, q, out, scratch, scale=None, window=0, sinks=None):
    """Attention of the rows q [n_tokens][heads][head_dim] over the cache, which holds their tokens already, into out
    (scale: head_dim^-0.5 if None; window 0: everything up to the row's own token; sinks: F32 [heads] or None)."""
    if not 0 <= window <= 0x7fffffff:
        _fits("kv8_attn: window", window)
    i, st, dev = cache.index, e.stream, cache.device
    if scale is None:
        scale = cache.head_dim ** -0.5
    if batch.index != i:
        rc = 1
    elif st.device_index == i == _current():
        rc = _lib.host().msb_host_kv8_attn(q, out, scratch, sinks, cache.addr, batch.addr, i, scale, window, _ATTN, st.cuda_stream)
    else:
        rc = _elsewhere(e, dev, _lib.host().msb_host_kv8_attn, q, out, scratch, sinks, cache.addr, batch.addr, i, scale, window, _ATTN)
    if rc > 0:                     # not plainly right: say why
        _want(batch.device == dev and scratch.device == dev, "kv8_attn: cache, batch and scratch on different devices")
        _want(scratch.is_contiguous(), "kv8_attn: scratch must be contiguous")
        heads = q.shape[1] if q.dim() == 3 else 0
        ty = _rows("q", q, batch.n_tokens, heads, cache.head_dim, dev)
        _want(_rows("out", out, batch.n_tokens, heads, cache.head_dim, dev) == ty, "q and out must be of one type")
        _want(False, "kv8_attn: sinks must be contiguous float32 [%d] or None" % heads)
    _lib.check(rc)
