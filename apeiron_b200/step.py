"""The steps between the projections, on torch tensors: residual add + RMS norm into an 8-bit
activation, rotary positions with the append to a paged 4-bit KV cache, attention over that cache,
and the sampler (include/apeiron_cuda.h states each of them).

``StepOps`` checks its tensors, queues one asynchronous call on the current torch stream (or the
``stream`` given, a raw handle) and returns without waiting; outputs may be passed in and are
allocated otherwise, for the stream that the call goes to (as under ``torch.cuda.stream``: to use
them on another one, wait for it and tell the allocator with ``record_stream``).  A refused argument
raises ``ValueError``, a backend condition ``BackendError``.  What only the device sees (a page
number outside the cache, a value that has no 4-bit image) goes to the optional ``status`` words of
``new_status``, read with ``check_status``.
"""
from __future__ import annotations

import ctypes as C
import struct

import torch

from . import _abi
from .chart import Backend, BackendError

_TYPES = {torch.float32: _abi.DTYPE_F32, torch.float16: _abi.DTYPE_F16,
          torch.bfloat16: _abi.DTYPE_BF16}
_LAYOUTS = {"half": _abi.ROPE_HALF, "interleaved": _abi.ROPE_INTERLEAVED}
_SCALINGS = {None: _abi.ROPE_PLAIN, "linear": _abi.ROPE_LINEAR, "bands": _abi.ROPE_BANDS,
             "ramp": _abi.ROPE_RAMP}


# A call's argument struct, packed in one go (the mirrors in _abi hold the same layout).
_NORM = struct.Struct("@9P7Nfi").pack
_ROPE = struct.Struct("@8P5N4i").pack
_ATTN = struct.Struct("@3P2N2if3i0P").pack
_SAMPLE = struct.Struct("@9P3N").pack
# what packing raises for a number that its field does not hold
_PACK_ERRORS = (struct.error, OverflowError)
_INT_MAX = 2 ** 31 - 1

_raw_stream = torch._C._cuda_getCurrentRawStream
_F32, _I32, _I64 = torch.float32, torch.int32, torch.int64


def _need(ok, what):
    if not ok:
        raise ValueError(what)


def _vector(t, n, dtype, name, dev):
    """The address of a contiguous vector of n elements on GPU `dev`; 0 for None."""
    if t is None:
        return 0
    if not (t.dtype is dtype and t.numel() == n and t.get_device() == dev and t.is_contiguous()):
        raise ValueError(f"{name}: a contiguous tensor of {n} {dtype} elements on cuda:{dev} is "
                         "wanted")
    return t.data_ptr()


def _rows(t, shape, name, dtype, dev):
    """The elements between rows of a tensor of `shape` (2 or 3 dims, rows first) on GPU `dev` whose
    rows are each contiguous."""
    if t.dtype is dtype and t.get_device() == dev and t.shape == shape:
        st = t.stride()
        if len(st) == 2:
            width = shape[1]
            if st[1] == 1 or width == 1:
                if st[0] >= width:
                    return st[0]
                if shape[0] <= 1:
                    return width
        else:
            width = shape[1] * shape[2]
            if st[2] == 1 and (st[1] == shape[2] or shape[1] == 1):
                if st[0] >= width:
                    return st[0]
                if shape[0] <= 1:
                    return width
    raise ValueError(f"{name}: a tensor {tuple(shape)} of {dtype} on cuda:{dev} is wanted, its "
                     "rows contiguous and apart")


class DeviceAct:
    """An activation as the projections read it: int8 codes (k, padded n), exponent bytes and
    descriptors (k, 8 int32) of k columns (the layout of ``apx_quant_f32_cols_async``)."""

    __slots__ = ("codes", "exps", "descs", "k", "n", "dev")

    def __init__(self, codes, exps, descs, n):
        self.codes, self.exps, self.descs = codes, exps, descs
        self.k, self.n, self.dev = codes.shape[0], n, codes.get_device()
        pad = _abi.load().apx_act_padded_len(n)
        _need(self.dev >= 0 and codes.shape == (self.k, pad), f"codes: int8 ({self.k}, {pad}) on a "
              "GPU are wanted")
        _vector(codes, self.k * pad, torch.int8, "codes", self.dev)
        _vector(exps, self.k * (pad // 32), torch.uint8, "exps", self.dev)
        _vector(descs, self.k * 8, torch.int32, "descs", self.dev)

    @classmethod
    def empty(cls, ops: "StepOps", k: int, n: int, stream=None) -> "DeviceAct":
        pad = ops.lib.apx_act_padded_len(n)
        return cls(ops._empty((k, pad), torch.int8, stream),
                   ops._empty((k, pad // 32), torch.uint8, stream),
                   ops._empty((k, 8), torch.int32, stream), n)


class KV4Cache:
    """A layer's paged 4-bit cache over ``pages``: uint8 (n_pages, n_kv_heads, page bytes)."""

    __slots__ = ("pages", "struct", "ref", "n_kv_heads", "head_dim", "dev")

    def __init__(self, pages, n_kv_heads: int, head_dim: int, page_tokens: int):
        size = 0
        if 0 < head_dim <= _INT_MAX and 0 < page_tokens <= _INT_MAX:
            size = self.page_bytes(head_dim, page_tokens)
        _need(size > 0, f"head_dim {head_dim} with pages of {page_tokens} tokens is not served")
        _need(pages.is_cuda and pages.dtype is torch.uint8 and pages.is_contiguous()
              and pages.shape[1:] == (n_kv_heads, size) and pages.data_ptr() % 16 == 0,
              f"pages: a contiguous CUDA uint8 tensor (n, {n_kv_heads}, {size}) is wanted")
        self.pages, self.n_kv_heads, self.head_dim = pages, n_kv_heads, head_dim
        self.dev = pages.get_device()
        self.struct = _abi.Kv4Cache(pages.data_ptr(), pages.shape[0], n_kv_heads, head_dim,
                                    page_tokens, 0)
        self.ref = C.byref(self.struct)

    @staticmethod
    def page_bytes(head_dim: int, page_tokens: int) -> int:
        return _abi.load().apx_kv4_page_bytes(head_dim, page_tokens)

    @classmethod
    def empty(cls, n_pages, n_kv_heads, head_dim, page_tokens, device="cuda") -> "KV4Cache":
        size = cls.page_bytes(head_dim, page_tokens)
        return cls(torch.zeros(n_pages, n_kv_heads, size, dtype=torch.uint8, device=device),
                   n_kv_heads, head_dim, page_tokens)


class SeqBatch:
    """The requests of one call: ``cu`` (n + 1) query offsets, ``kv_len`` (n) cached tokens with
    the query tokens last, ``table`` (n, max_pages) page numbers, all int32; ``n_tokens`` query
    tokens in all, at most ``max_q`` of one request."""

    __slots__ = ("cu", "kv_len", "table", "n_tokens", "struct", "ref", "dev")

    def __init__(self, cu, kv_len, table, n_tokens: int, max_q: int):
        n, dev = kv_len.numel(), kv_len.get_device()
        _need(dev >= 0, "kv_len: a CUDA tensor is wanted")
        _need(0 <= n_tokens <= _INT_MAX and 0 <= max_q <= _INT_MAX,
              f"{n_tokens} query tokens, at most {max_q} of a request: not served")
        _need(table.dim() == 2 and table.shape[0] == n, "table: one row per request is wanted")
        self.cu, self.kv_len, self.table, self.n_tokens = cu, kv_len, table, n_tokens
        self.dev = dev
        self.struct = _abi.SeqBatch(_vector(cu, n + 1, torch.int32, "cu", dev),
                                    _vector(kv_len, n, torch.int32, "kv_len", dev),
                                    _vector(table, table.numel(), torch.int32, "table", dev),
                                    n_tokens, n, table.shape[1], max_q, 0)
        self.ref = C.byref(self.struct)


class StepOps:
    """The calls, on one backend context and its GPU, whichever is current.  Calls on one context
    must not overlap in time."""

    def __init__(self, backend: Backend):
        self.backend, self.lib = backend, backend.lib
        self.device = torch.device("cuda", backend.device)
        self._index = backend.device
        lib = self.lib
        self._norm, self._rope = lib.apx_add_rms_norm_quant_async, lib.apx_rope_kv4_append_async
        self._attn, self._sample = lib.apx_attn_kv4_async, lib.apx_sample_async

    @property
    def ctx(self):
        """The backend's context; None once it is closed, which the entry points refuse."""
        return self.backend.ctx

    def _stream(self, stream):
        return _raw_stream(self._index) if stream is None else stream

    def _here(self, cache, batch):
        if not (cache.dev == batch.dev == self._index):
            raise ValueError(f"cache and batch on cuda:{self._index} are wanted")

    def _empty(self, shape, dtype, stream):
        """An output of a call on `stream`: memory that earlier work on that stream is done with."""
        if stream is None:
            return torch.empty(shape, dtype=dtype, device=self.device)
        with torch.cuda.stream(torch.cuda.ExternalStream(stream, device=self.device)):
            return torch.empty(shape, dtype=dtype, device=self.device)

    @staticmethod
    def _failed(rc, name):
        if rc in (_abi.APX_ERR_INVALID_ARGUMENT, _abi.APX_ERR_LAYOUT_MISMATCH,
                  _abi.APX_ERR_TOO_LARGE):
            raise ValueError(f"{name}: refused with code {rc}")
        raise BackendError(f"{name}: backend error {rc}")

    # -- refusals that the device finds -------------------------------------------------------
    def new_status(self):
        """Status words with nothing refused, written on the current stream."""
        return torch.full((2,), -1, dtype=_I64, device=self.device)

    @staticmethod
    def check_status(status):
        """None, or (row, code) of the first refusal; waits for the current stream, which is to have
        waited for the calls' own where that is another."""
        word = int(status[0].item()) & ((1 << 64) - 1)
        return None if word == (1 << 64) - 1 else (word >> 24, word >> 16 & 0xFF)

    # -- the calls -------------------------------------------------------------------------------
    def add_rms_norm_quant(self, x, weight, eps, *, add=None, resid=None, act=None, deq=None,
                           y=None, stream=None):
        """h = x + add into ``resid`` (may be x), h * weight / rms(h) into ``y`` (f32), ``act``
        (a DeviceAct, allocated when no output is given) and ``deq`` (the activation's values,
        f32 or bf16).  x, add: (k, n) f32; weight: n f32, or None.  Returns act."""
        shape, dev = x.shape, self._index
        k, n = shape
        if act is None and deq is None and y is None:
            act = DeviceAct.empty(self, k, n, stream)
        codes = exps = descs = 0
        if act is not None:
            _need(act.n == n and act.k == k and act.dev == dev,
                  f"act: ({k}, {n}) on cuda:{dev} is wanted")
            codes, exps, descs = act.codes.data_ptr(), act.exps.data_ptr(), act.descs.data_ptr()
        try:
            rc = self._norm(self.backend.ctx, _NORM(
                x.data_ptr(), 0 if add is None else add.data_ptr(),
                _vector(weight, n, _F32, "weight", dev),
                0 if resid is None else resid.data_ptr(), 0 if y is None else y.data_ptr(),
                0 if deq is None else deq.data_ptr(), codes, exps, descs, n, k,
                _rows(x, shape, "x", _F32, dev),
                0 if add is None else _rows(add, shape, "add", _F32, dev),
                0 if resid is None else _rows(resid, shape, "resid", _F32, dev),
                0 if y is None else _rows(y, shape, "y", _F32, dev),
                0 if deq is None else _rows(deq, shape, "deq", deq.dtype, dev), eps,
                0 if deq is None else _TYPES.get(deq.dtype, -1)), self._stream(stream))
        except _PACK_ERRORS as e:
            raise ValueError(f"add_rms_norm_quant: {e}") from None
        if rc:
            self._failed(rc, "add_rms_norm_quant")
        return act

    def rope_table(self, n_pos, rot_dim, base=10000.0, *, scaling=None, factor=1.0, low=1.0,
                   high=4.0, original=0.0, mscale=1.0, stream=None):
        """(n_pos, rot_dim / 2, 2) f32 cosines and sines; ``scaling``: None, "linear", "bands" or
        "ramp" (``low`` and ``high``: turns within the ``original`` length)."""
        _need(0 <= n_pos <= _INT_MAX and 0 <= rot_dim <= _INT_MAX,
              f"a table of {n_pos} positions for {rot_dim} dims is not served")
        table = self._empty((n_pos, rot_dim // 2, 2), _F32, stream)
        _need(scaling in _SCALINGS, f"scaling: one of {list(_SCALINGS)} is wanted")
        f = _abi.RopeFreqs(base, factor, low, high, original, mscale, rot_dim,
                           _SCALINGS[scaling])
        rc = self.lib.apx_rope_table_async(self.ctx, C.byref(f), n_pos, table.data_ptr(),
                                           self._stream(stream))
        if rc:
            self._failed(rc, "rope_table")
        return table

    def rope_kv4_append(self, q, k, v, table, cache: KV4Cache, batch: SeqBatch, *, rot_dim,
                        layout="half", q_out=None, q_type=_F32, k_deq=None, v_deq=None,
                        status=None, stream=None):
        """q (tokens, heads, dim; None to leave out) turned into ``q_out`` (may be q); k turned and v
        (tokens, kv heads, dim) appended to the cache in 4 bits.  ``k_deq`` / ``v_deq`` (f16):
        the values the cache now holds.  Returns q_out."""
        self._here(cache, batch)
        t, heads, dim, dev = batch.n_tokens, cache.n_kv_heads, cache.head_dim, self._index
        kv = (t, heads, dim)
        ldq = ld_out = n_heads = kind = q_ptr = out_ptr = 0
        if q is not None:
            shape = (t, q.shape[1], dim)
            if q_out is None:
                q_out = self._empty(shape, q_type, stream)
            ldq, n_heads = _rows(q, shape, "q", _F32, dev), shape[1]
            ld_out = _rows(q_out, shape, "q_out", q_out.dtype, dev)
            kind = _TYPES.get(q_out.dtype, -1)
            q_ptr, out_ptr = q.data_ptr(), q_out.data_ptr()
        n_pos, n = table.shape[0], t * heads * dim
        try:
            rc = self._rope(self.backend.ctx, _ROPE(
                q_ptr, k.data_ptr(), v.data_ptr(),
                _vector(table, n_pos * rot_dim, _F32, "table", dev),
                out_ptr, _vector(k_deq, n, torch.float16, "k_deq", dev),
                _vector(v_deq, n, torch.float16, "v_deq", dev),
                _vector(status, 2, _I64, "status", dev), n_pos, ldq, _rows(k, kv, "k", _F32, dev), _rows(v, kv, "v", _F32, dev), ld_out,
                rot_dim, _LAYOUTS.get(layout, -1), n_heads, kind), cache.ref, batch.ref,
                self._stream(stream))
        except _PACK_ERRORS as e:
            raise ValueError(f"rope_kv4_append: {e}") from None
        if rc:
            self._failed(rc, "rope_kv4_append")
        return q_out

    def attn_kv4(self, q, cache: KV4Cache, batch: SeqBatch, scale, *, window=0, sinks=0,
                 out=None, status=None, stream=None):
        """softmax(scale * q k^T) v of q (tokens, heads, dim; f32, f16 or bf16) over the cache,
        causal, within ``window`` keys (0: all) and the first ``sinks``.  Returns out."""
        self._here(cache, batch)
        heads, dtype, dev = q.shape[1], q.dtype, self._index
        shape = (batch.n_tokens, heads, cache.head_dim)
        if out is None:
            out = self._empty(shape, dtype, stream)
        try:
            rc = self._attn(self.backend.ctx, _ATTN(
                q.data_ptr(), out.data_ptr(), _vector(status, 2, _I64, "status", dev),
                _rows(q, shape, "q", dtype, dev), _rows(out, shape, "out", dtype, dev),
                _TYPES.get(dtype, -1), heads, scale, window, sinks, 0), cache.ref, batch.ref,
                self._stream(stream))
        except _PACK_ERRORS as e:
            raise ValueError(f"attn_kv4: {e}") from None
        if rc:
            self._failed(rc, "attn_kv4")
        return out

    def sample(self, logits, u, *, temperature=None, top_k=None, top_p=None, min_p=None,
               token=None, prob=None, kept=None, stream=None):
        """One token per row of f32 ``logits`` (rows, vocab) from ``u`` (rows) in [0, 1); the
        filters are per row, None to leave out.  Returns token (int32)."""
        shape, dev = logits.shape, self._index
        rows, vocab = shape
        if token is None:
            token = self._empty(rows, _I32, stream)
        rc = self._sample(self.backend.ctx, _SAMPLE(
            logits.data_ptr(), _vector(u, rows, _F32, "u", dev),
            _vector(temperature, rows, _F32, "temperature", dev),
            _vector(top_p, rows, _F32, "top_p", dev), _vector(min_p, rows, _F32, "min_p", dev),
            _vector(top_k, rows, _I32, "top_k", dev),
            _vector(token, rows, _I32, "token", dev), _vector(prob, rows, _F32, "prob", dev),
            _vector(kept, rows, _I32, "kept", dev), rows, vocab,
            _rows(logits, shape, "logits", _F32, dev)), self._stream(stream))
        if rc:
            self._failed(rc, "sample")
        return token
