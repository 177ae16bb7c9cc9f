"""A layer's KV cache in 4- or 8-bit codes, and the decode step's operators over it.

A 16-bit cache costs ``4 d`` bytes a token and KV head, all of which a dense decode step and the
decode routing read; with 4-bit codes and groups of 32 it is ``1.25 d``, with groups of 128
``1.0625 d``. ``QuantKV`` owns the buffers; ``write`` quantises new rows into them (and can return the
values that the cache now holds, so that a prefill attends to what later steps will read) and
``read`` gives rows back. ``quant_decode``, ``quant_pooled_probs`` and ``quant_route`` are
``bigger_bird_decode``, ``pooled_probs`` and ``bigger_bird_route`` on such a cache, without a 16-bit copy
of it in between. The format and the arithmetic are described at ``bb_qkv_cache`` in
``include/bb_b200.h``.

Everything runs on the current stream of the cache's device without synchronising; ``n`` and ``at`` may be 1-element GPU
integer tensors that the kernels read at run time, so a captured CUDA graph follows a growing cache.
"""
from __future__ import annotations

import ctypes as C
import threading

import torch

from . import _lib, _ops

__all__ = ["QuantKV", "quant_decode", "quant_pooled_probs", "quant_route"]

_HALF = {torch.float16: _lib.BB_F16, torch.bfloat16: _lib.BB_BF16}


def _rows(x):
    """x [heads, rows, d] as the kernels can read it (a copy where they cannot), its address and strides."""
    sh, st, sd = x.stride()
    p, es = x.data_ptr(), x.element_size()
    if sd != 1 or (p | sh * es | st * es) & 15:
        # not contiguous(), which hands back what only an address or the stride of a single head or row is wrong with
        x = x.clone(memory_format=torch.contiguous_format)
        p, st = x.data_ptr(), x.shape[2]
        sh = x.shape[1] * st
    return x, p, sh, st


def _stream(device):
    """The current stream's handle (``torch.cuda.current_stream`` builds a Stream object for it)."""
    return torch._C._cuda_getCurrentRawStream(device.index)


def _elsewhere(device):
    """Whether another GPU than ``device`` is current: a launch would go there, with this one's pointers."""
    return device.type == "cuda" and torch._C._cuda_getDevice() != device.index


# Counters (zero between calls), a workspace and a lock, one set a stream, for calls that run one after the other on it. Their
# sizes are fixed: a call that needs a larger workspace (a routing over some 64K keys or more, which takes far longer than the
# allocation) has its own, and a call that needs more counters (only with explicit splits) takes two launches instead of
# one. A call holds the lock while it enqueues: its launches hand each other results in the
# workspace, and a call of another thread on the stream must come after the last of them. The kernels leave the counters at
# zero whatever happens, a routing wait that runs out (code 48 of bb_device_fault) included.
_scratch = {}
_TICKETS, _WORKSPACE = 1024, 8 << 20


def _take_scratch(device, stream):
    """Tickets, a workspace and the lock under which to use them, for a call on ``stream``. Calls under a graph capture get
    their own, which the graph zeroes and keeps."""
    if torch.cuda.is_current_stream_capturing():
        return (torch.zeros(_TICKETS, dtype=torch.int32, device=device),
                torch.empty(1, dtype=torch.uint8, device=device), threading.Lock())
    s = _scratch.get((device.index, stream))
    if s is None:
        s = _scratch[device.index, stream] = (torch.zeros(_TICKETS, dtype=torch.int32, device=device),
                                              torch.empty(_WORKSPACE, dtype=torch.uint8, device=device), threading.Lock())
    return s


def _run(what, run, size_of, a, device, stream, tickets):
    """One call of a C entry that takes a workspace: with the stream's, or one of its own if that is too small."""
    if _elsewhere(device):
        with torch.cuda.device(device):
            return _run(what, run, size_of, a, device, stream, tickets)
    ref = C.byref(a)
    t, ws, lock = _take_scratch(device, stream)
    a.tickets, a.n_tickets = t.data_ptr(), min(tickets, _TICKETS)
    with lock:
        status = run(ref, ws.data_ptr(), ws.numel(), stream)
    if status == _lib.BB_ERR_WORKSPACE:
        size = C.c_size_t(0)
        _lib.check(size_of(ref, C.byref(size)), what)
        ws = torch.empty(size.value, dtype=torch.uint8, device=device)
        with lock:
            status = run(ref, ws.data_ptr(), ws.numel(), stream)
    if status:
        _lib.check(status, what)


class QuantKV:
    """Codes and (step, low) pairs of ``kv_heads`` x ``capacity`` rows of keys and of values.

    ``bits``: 4 or 8. ``group``: dimensions that share a step and a low value (32, 64, 96 or 128, dividing
    ``head_dim``, which is a multiple of 32 up to 128). Buffers start at zero, which reads as 0."""

    def __init__(self, kv_heads, capacity, head_dim, *, bits=4, group=32, device="cuda"):
        if bits not in (4, 8):
            raise ValueError("QuantKV: bits must be 4 or 8")
        if head_dim <= 0 or head_dim > 128 or head_dim % 32:
            raise ValueError("QuantKV: head_dim must be a multiple of 32 up to 128")
        if group <= 0 or group % 32 or head_dim % group:
            raise ValueError("QuantKV: group must be a multiple of 32 that divides head_dim")
        if kv_heads <= 0 or capacity <= 0:
            raise ValueError("QuantKV: kv_heads and capacity must be positive")
        codes = [torch.zeros(kv_heads, capacity, head_dim * bits // 8, dtype=torch.uint8, device=device) for _ in "kv"]
        meta = [torch.zeros(kv_heads, capacity, head_dim // group, 2, dtype=torch.bfloat16, device=device) for _ in "kv"]
        self._adopt(codes[0], meta[0], codes[1], meta[1], bits)

    @classmethod
    def from_buffers(cls, k_codes, k_meta, v_codes, v_meta, *, bits):
        """A cache over the caller's buffers: codes uint8 [Hkv, cap, d * bits / 8], meta bf16
        [Hkv, cap, d / group, 2] as (step, low); rows dense, heads at any stride."""
        self = cls.__new__(cls)
        if bits not in (4, 8):
            raise ValueError("QuantKV: bits must be 4 or 8")
        for codes, meta in ((k_codes, k_meta), (v_codes, v_meta)):
            if codes.dtype != torch.uint8 or meta.dtype != torch.bfloat16 or codes.ndim != 3 or meta.ndim != 4:
                raise ValueError("QuantKV: codes must be uint8 [Hkv, cap, d*bits/8], meta bf16 [Hkv, cap, d/group, 2]")
            if meta.shape[:2] != codes.shape[:2] or meta.shape[3] != 2 or not meta.shape[2]:
                raise ValueError("QuantKV: codes and meta do not match")
            if codes.stride()[1:] != (codes.shape[2], 1) or meta.stride()[1:] != (2 * meta.shape[2], 2, 1):
                raise ValueError("QuantKV: rows must be dense")
            if codes.shape[0] > 1 and meta.stride(0) % 2:
                raise ValueError("QuantKV: heads of meta must be whole (step, low) pairs apart")
        if k_codes.shape != v_codes.shape or k_meta.shape != v_meta.shape:
            raise ValueError("QuantKV: keys and values do not match")
        if any(t.device != k_codes.device for t in (k_meta, v_codes, v_meta)):
            raise ValueError("QuantKV: buffers must be on one device")
        if k_codes.shape[2] * 8 // bits % k_meta.shape[2]:
            raise ValueError("QuantKV: group must divide head_dim")
        self._adopt(k_codes, k_meta, v_codes, v_meta, bits)
        return self

    def _adopt(self, k_codes, k_meta, v_codes, v_meta, bits):
        self.k_codes, self.k_meta, self.v_codes, self.v_meta, self.bits = k_codes, k_meta, v_codes, v_meta, bits
        self.kv_heads, self.capacity = k_codes.shape[:2]
        self.head_dim = k_codes.shape[2] * 8 // bits
        self.group = self.head_dim // k_meta.shape[2]
        self.device = k_codes.device
        self._struct = _lib.QkvCache(
            k_codes=k_codes.data_ptr(), k_meta=k_meta.data_ptr(), v_codes=v_codes.data_ptr(), v_meta=v_meta.data_ptr(),
            k_codes_h=k_codes.stride(0), k_meta_h=k_meta.stride(0) // 2, v_codes_h=v_codes.stride(0),
            v_meta_h=v_meta.stride(0) // 2, kv_heads=self.kv_heads, cap=self.capacity, d=self.head_dim, bits=bits,
            group=self.group)
        # Calls fill copies of these, so that threads may share a cache.
        self._attn = _lib.QkvAttnArgs(cache=self._struct)
        self._write = _lib.QkvWriteArgs(cache=self._struct)
        self._read = _lib.QkvReadArgs(cache=self._struct)

    @property
    def nbytes(self):
        return sum(t.numel() * t.element_size() for t in (self.k_codes, self.k_meta, self.v_codes, self.v_meta))

    def write(self, k, v, at, *, values=False):
        """Quantise k / v [Hkv, T, d] (fp16, bf16 or fp32) into rows at, at + 1, ...; ``at`` an int, or a
        1-element GPU integer tensor (rows that fall outside the cache are then skipped). With
        ``values``, returns what the rows now stand for, (k, v) [Hkv, T, d] in the input dtype, stored
        as [T, Hkv, d]."""
        dev = self.device
        if k.device != dev or v.device != dev or dev.type != "cuda":
            raise ValueError("QuantKV.write requires CUDA tensors on the cache's device")
        if _elsewhere(dev):
            with torch.cuda.device(dev):
                return self.write(k, v, at, values=values)
        dtype = _ops._DT.get(k.dtype)
        if dtype is None or v.dtype != k.dtype:
            raise ValueError("QuantKV.write: k and v must share one of f16/bf16/f32")
        shape = k.shape
        if len(shape) != 3 or v.shape != shape or shape[0] != self.kv_heads or shape[2] != self.head_dim:
            raise ValueError("QuantKV.write: k and v must be [Hkv, T, d] of the cache")
        hk, t, d = shape
        a = _lib.QkvWriteArgs.from_buffer_copy(self._write)
        k, a.k, a.sk_h, a.sk_t = _rows(k)
        v, a.v, a.sv_h, a.sv_t = _rows(v)
        a.t, a.dtype = t, dtype
        keep = None
        if isinstance(at, torch.Tensor):
            keep = _ops._n_arg(at, 0, dev)[2]
            a.at_dev = keep.data_ptr()
        else:
            a.at = at = int(at)
            if at < 0 or at + t > self.capacity:
                raise ValueError(f"QuantKV.write: rows [{at}, {at + t}) outside a cache of {self.capacity}")
        out = None
        if values:
            stride = (d, hk * d, 1)
            out = k.new_empty_strided(shape, stride), k.new_empty_strided(shape, stride)
            a.out_k, a.out_v = out[0].data_ptr(), out[1].data_ptr()
            a.sok_h = a.sov_h = d
            a.sok_t = a.sov_t = hk * d
        status = _lib.lib().bb_qkv_write(C.byref(a), _stream(dev))
        if status:
            _lib.check(status, "QuantKV.write")
        return out

    def read(self, positions=None, *, start=0, stop=None, dtype=torch.bfloat16):
        """Values of rows [start, stop), or of rows ``positions`` (int32 / int64 [Hkv, L]; positions outside the
        cache give zeros): (k, v) [Hkv, L, d]."""
        dt, dev = _ops._DT.get(dtype), self.device
        if dt is None:
            raise ValueError("QuantKV.read: dtype must be one of f16/bf16/f32")
        if dev.type != "cuda":
            raise ValueError("QuantKV.read requires a CUDA cache")
        if _elsewhere(dev):
            with torch.cuda.device(dev):
                return self.read(positions, start=start, stop=stop, dtype=dtype)
        a = _lib.QkvReadArgs.from_buffer_copy(self._read)
        hk, d = self.kv_heads, self.head_dim
        if positions is None:
            stop = self.capacity if stop is None else int(stop)
            if not 0 <= start <= stop <= self.capacity:
                raise ValueError(f"QuantKV.read: rows [{start}, {stop}) outside a cache of {self.capacity}")
            a.start, rows = start, stop - start
        else:
            wide = positions.dtype == torch.int64
            if positions.device != dev or not (wide or positions.dtype == torch.int32):
                raise ValueError("QuantKV.read: positions must be int32 or int64 on the cache's device")
            if positions.ndim != 2 or positions.shape[0] != hk:
                raise ValueError("QuantKV.read: positions must be [Hkv, L]")
            if positions.stride(1) != 1:
                positions = positions.contiguous()
            rows = positions.shape[1]
            a.positions, a.sp_h, a.pos_i64 = positions.data_ptr() if rows else None, positions.stride(0), wide
        shape, stride = (hk, rows, d), (rows * d, d, 1)
        k = torch.empty_strided(shape, stride, dtype=dtype, device=dev)
        v = torch.empty_strided(shape, stride, dtype=dtype, device=dev)
        if rows:
            a.dtype, a.rows, a.out_k, a.out_v = dt, rows, k.data_ptr(), v.data_ptr()
            a.sok_h = a.sov_h = rows * d
            a.sok_t = a.sov_t = d
            status = _lib.lib().bb_qkv_read(C.byref(a), _stream(dev))
            if status:
                _lib.check(status, "QuantKV.read")
        return k, v


def _args(q, kv, front, window, scale, n, splits, what):
    """The filled argument struct of an attention call, and the tensors that must outlive it."""
    dtype = _HALF.get(q.dtype)
    if dtype is None or not q.is_cuda:
        raise ValueError(f"{what} requires CUDA FP16/BF16 queries")
    if q.device != kv.device:
        raise ValueError(f"{what}: q and the cache must be on one device")
    shape, stride = q.shape, q.stride()
    if not shape[0] or shape[0] % kv.kv_heads or shape[-1] != kv.head_dim:
        raise ValueError(f"{what}: q must be [H, ..., {kv.head_dim}] with H a multiple of {kv.kv_heads}")
    if front < 0 or window < 0:
        raise ValueError(f"{what}: front and window must be >= 0")
    if stride[-1] != 1:
        q = q.contiguous()
        stride = q.stride()
    a = _lib.QkvAttnArgs.from_buffer_copy(kv._attn)
    a.q, a.sq_h, a.heads, a.dtype = q.data_ptr(), stride[0], shape[0], dtype
    a.t, a.front, a.window, a.scale, a.splits = 1, front, window, scale, splits or 0
    keep = None
    if isinstance(n, torch.Tensor):
        a.n, a.n_dev, keep = _ops._n_arg(n, kv.capacity, kv.device)
    else:
        a.n = kv.capacity if n is None else int(n)
        if not 0 <= a.n <= kv.capacity:
            raise ValueError(f"{what}: n must lie in [0, {kv.capacity}]")
    return a, (q, keep)


def quant_decode(q, kv, indices=None, *, front=64, window=4096, scale=1.0, n=None, splits=None):
    """Attention of the newest token, q [H, d], or of the newest T tokens, q [H, T, d], over the first ``n``
    keys of ``kv`` (their own rows written first). The token at position p attends to [0, front),
    [p - window + 1, p] and its ``indices`` (int32 / int64 [Hkv, R], or [H, R] for a list per query
    head; entries outside [front, p - window] are skipped), each key of the first two once;
    ``front=0, window=n`` is dense causal attention. ``n``: an int, a 1-element GPU integer tensor, or
    None for the whole capacity.

    Returns q's shape and dtype ([T, H, d] storage for T tokens). ``splits``: pieces that a key list is
    cut into (default: enough to fill the GPU). Any T up to 2^30 / H; every 8 query rows of a KV head
    (H / Hkv a token) take a pass over the keys."""
    if q.ndim not in (2, 3):
        raise ValueError("quant_decode: q must be [H, d] or [H, T, d]")
    a, keep = _args(q, kv, front, window, scale, n, splits, "quant_decode")
    q = keep[0]
    if q.ndim == 3:
        h, t, d = q.shape
        if not t or (keep[1] is None and t > a.n):
            raise ValueError("quant_decode: the tokens of q must be among the first n cached")
        a.t, a.sq_t = t, q.stride(1)
        out = torch.empty_strided((h, t, d), (d, h * d, 1), dtype=q.dtype, device=q.device)
        a.so_h, a.so_t = d, h * d
    else:
        h = q.shape[0]
        out = torch.empty_like(q)
        if out.stride(-1) != 1:
            out = out.contiguous()
        a.so_h = out.stride(0)
    a.out = out.data_ptr()
    if indices is not None and indices.shape[-1]:
        if indices.device != q.device or indices.dtype not in (torch.int32, torch.int64):
            raise ValueError("quant_decode: indices must be int32 or int64 on q's device")
        if indices.ndim != 2 or indices.shape[0] not in (kv.kv_heads, h):
            raise ValueError("quant_decode: indices must be [Hkv, R] (pooled) or [H, R] (per head)")
        if indices.stride(-1) != 1:
            indices = indices.contiguous()
        a.idx, a.si_r, a.route_rows, a.route_k = indices.data_ptr(), indices.stride(0), *indices.shape
        a.idx_i64 = int(indices.dtype == torch.int64)
    L = _lib.lib()
    _run("quant_decode", L.bb_qkv_decode, L.bb_qkv_decode_workspace_size, a, kv.device, _stream(kv.device),
         kv.kv_heads * -(-(h // kv.kv_heads * a.t) // 8))
    return out


def _route(a, kv, what):
    L = _lib.lib()
    _run(what, L.bb_qkv_route, L.bb_qkv_route_workspace_size, a, kv.device, _stream(kv.device), 2 * kv.kv_heads)


def quant_pooled_probs(q, kv, *, front=64, window=4096, scale=1.0, n=None, splits=None):
    """q [H, d] -> [Hkv, capacity] fp32: the softmax probability of each of the first ``n`` keys, averaged over the
    query heads of its KV head; -1 outside [front, n - window)."""
    if q.ndim != 2:
        raise ValueError("quant_pooled_probs: q must be [H, d]")
    a, keep = _args(q, kv, front, window, scale, n, splits, "quant_pooled_probs")
    hk, cap = kv.kv_heads, kv.capacity
    probs = torch.empty_strided((hk, cap), (cap, 1), dtype=torch.float32, device=kv.device)
    a.out_probs = probs.data_ptr()
    _route(a, kv, "quant_pooled_probs")
    return probs


def quant_route(q, kv, k_route, *, front=64, window=4096, scale=1.0, n=None, splits=None):
    """Positions [Hkv, k_route] (int64, ascending) of the keys with the highest pooled probabilities in
    [front, n - window). Where that range holds fewer than k_route keys, the rest lie outside it (and
    ``quant_decode`` with the same front and window skips them)."""
    if q.ndim != 2:
        raise ValueError("quant_route: q must be [H, d]")
    if not 0 <= k_route <= kv.capacity:
        raise ValueError("quant_route: k_route must lie in [0, capacity]")
    a, keep = _args(q, kv, front, window, scale, n, splits, "quant_route")
    idx = torch.empty(kv.kv_heads, k_route, dtype=torch.int64, device=kv.device)
    if not k_route:
        return idx
    a.out_idx, a.so_i, a.route_k, a.out_idx_i64 = idx.data_ptr(), k_route, k_route, 1
    _route(a, kv, "quant_route")
    return idx
