"""The steps between the projections, on torch tensors: residual add + RMS norm into an 8-bit
activation, rotary positions with the append to a paged 4-bit KV cache, attention over that cache,
and the sampler (include/apeiron_cuda.h states each of them).

``StepOps`` checks its tensors, queues one asynchronous call on the current torch stream (or the
``stream`` given, a raw handle) and returns without waiting; outputs may be passed in and are
allocated otherwise.  A refused argument raises ``ValueError``, a backend condition
``BackendError``.  What only the device sees (a page number outside the cache, a value that has no
4-bit image) goes to the optional ``status`` words of ``new_status``, read with ``check_status``.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _abi
from .chart import Backend, BackendError

_TYPES = {torch.float32: _abi.DTYPE_F32, torch.float16: _abi.DTYPE_F16,
          torch.bfloat16: _abi.DTYPE_BF16}
_LAYOUTS = {"half": _abi.ROPE_HALF, "interleaved": _abi.ROPE_INTERLEAVED}
_SCALINGS = {None: _abi.ROPE_PLAIN, "linear": _abi.ROPE_LINEAR, "bands": _abi.ROPE_BANDS,
             "ramp": _abi.ROPE_RAMP}


def _need(ok, what):
    if not ok:
        raise ValueError(what)


def _vector(t, n, dtype, name):
    """The address of a contiguous vector of n elements; 0 for None."""
    if t is None:
        return 0
    _need(t.is_cuda and t.dtype is dtype and t.numel() == n and t.is_contiguous(),
          f"{name}: a contiguous CUDA tensor of {n} {dtype} elements is wanted")
    return t.data_ptr()


def _rows(t, shape, name, dtype=None):
    """(address, elements between rows) of a tensor of `shape` (rows first) whose rows are each
    contiguous; (0, 0) for None."""
    if t is None:
        return 0, 0
    _need(t.is_cuda and t.shape == shape and (dtype is None or t.dtype is dtype),
          f"{name}: a CUDA tensor of shape {tuple(shape)}{f' and {dtype}' if dtype else ''} is "
          "wanted")
    width = 1
    for size, stride in zip(reversed(shape[1:]), reversed(t.stride()[1:])):
        _need(stride == width or size == 1, f"{name}: its rows are not contiguous")
        width *= size
    ld = t.stride(0) if shape[0] > 1 else width
    _need(ld >= width, f"{name}: its rows overlap")
    return t.data_ptr(), ld


class DeviceAct:
    """An activation as the projections read it: int8 codes, exponent bytes and descriptors of k
    columns (the layout of ``apx_quant_f32_cols_async``)."""

    __slots__ = ("codes", "exps", "descs", "k", "n")

    def __init__(self, codes, exps, descs, n):
        self.codes, self.exps, self.descs = codes, exps, descs
        self.k, self.n = codes.shape[0], n

    @classmethod
    def empty(cls, ops: "StepOps", k: int, n: int) -> "DeviceAct":
        pad = ops.lib.apx_act_padded_len(n)
        dev = ops.device
        return cls(torch.empty(k, pad, dtype=torch.int8, device=dev),
                   torch.empty(k, pad // 32, dtype=torch.uint8, device=dev),
                   torch.empty(k, 8, dtype=torch.int32, device=dev), n)


class KV4Cache:
    """A layer's paged 4-bit cache over ``pages``: uint8 (n_pages, n_kv_heads, page bytes)."""

    __slots__ = ("pages", "struct", "ref", "n_kv_heads", "head_dim")

    def __init__(self, pages, n_kv_heads: int, head_dim: int, page_tokens: int):
        size = self.page_bytes(head_dim, page_tokens)
        _need(size > 0, f"head_dim {head_dim} with pages of {page_tokens} tokens is not served")
        _need(pages.is_cuda and pages.dtype is torch.uint8 and pages.is_contiguous()
              and pages.shape[1:] == (n_kv_heads, size) and pages.data_ptr() % 16 == 0,
              f"pages: a contiguous CUDA uint8 tensor (n, {n_kv_heads}, {size}) is wanted")
        self.pages, self.n_kv_heads, self.head_dim = pages, n_kv_heads, head_dim
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

    __slots__ = ("cu", "kv_len", "table", "n_tokens", "struct", "ref")

    def __init__(self, cu, kv_len, table, n_tokens: int, max_q: int):
        n = kv_len.numel()
        _need(table.dim() == 2 and table.shape[0] == n, "table: one row per request is wanted")
        self.cu, self.kv_len, self.table, self.n_tokens = cu, kv_len, table, n_tokens
        self.struct = _abi.SeqBatch(_vector(cu, n + 1, torch.int32, "cu"),
                                    _vector(kv_len, n, torch.int32, "kv_len"),
                                    _vector(table, table.numel(), torch.int32, "table"),
                                    n_tokens, n, table.shape[1], max_q, 0)
        self.ref = C.byref(self.struct)


class StepOps:
    """The calls, on one backend context.  Calls on one context must not overlap in time."""

    def __init__(self, backend: Backend):
        self.backend, self.lib, self.ctx = backend, backend.lib, backend.ctx
        self.device = torch.device("cuda", backend.device)

    def _stream(self, stream):
        return torch.cuda.current_stream(self.device).cuda_stream if stream is None else stream

    @staticmethod
    def _done(rc, name):
        if rc in (_abi.APX_ERR_INVALID_ARGUMENT, _abi.APX_ERR_LAYOUT_MISMATCH,
                  _abi.APX_ERR_TOO_LARGE):
            raise ValueError(f"{name}: refused with code {rc}")
        if rc:
            raise BackendError(f"{name}: backend error {rc}")

    # -- refusals that the device finds -------------------------------------------------------
    def new_status(self):
        """Status words with nothing refused."""
        return torch.full((2,), -1, dtype=torch.int64, device=self.device)

    @staticmethod
    def check_status(status):
        """None, or (row, code) of the first refusal; waits for the work queued before."""
        word = int(status[0].item()) & ((1 << 64) - 1)
        return None if word == (1 << 64) - 1 else (word >> 24, word >> 16 & 0xFF)

    # -- the calls -------------------------------------------------------------------------------
    def add_rms_norm_quant(self, x, weight, eps, *, add=None, resid=None, act=None, deq=None,
                           y=None, stream=None):
        """h = x + add into ``resid`` (may be x), h * weight / rms(h) into ``y`` (f32), ``act``
        (a DeviceAct, allocated when no output is given) and ``deq`` (the activation's values).
        x, add: (k, n) f32.  Returns act."""
        k, n = x.shape
        if act is None and deq is None and y is None:
            act = DeviceAct.empty(self, k, n)
        a = _abi.NormArgs()
        f32 = torch.float32
        a.d_x, a.ldx = _rows(x, x.shape, "x", f32)
        a.d_weight = _vector(weight, n, f32, "weight")
        if add is not None:
            a.d_add, a.ld_add = _rows(add, x.shape, "add", f32)
        if resid is not None:
            a.d_resid, a.ld_resid = _rows(resid, x.shape, "resid", f32)
        if y is not None:
            a.d_y, a.ldy = _rows(y, x.shape, "y", f32)
        if deq is not None:
            a.d_deq, a.ld_deq = _rows(deq, x.shape, "deq")
            a.deq_type = _TYPES.get(deq.dtype, -1)
        if act is not None:
            _need(act.n == n and act.k == k, f"act: ({k}, {n}) is wanted")
            a.d_codes, a.d_exps = act.codes.data_ptr(), act.exps.data_ptr()
            a.d_descs = act.descs.data_ptr()
        a.n, a.k, a.eps = n, k, eps
        self._done(self.lib.apx_add_rms_norm_quant_async(self.ctx, C.byref(a),
                                                         self._stream(stream)),
                   "add_rms_norm_quant")
        return act

    def rope_table(self, n_pos, rot_dim, base=10000.0, *, scaling=None, factor=1.0, low=1.0,
                   high=4.0, original=0.0, mscale=1.0, stream=None):
        """(n_pos, rot_dim / 2, 2) f32 cosines and sines; ``scaling``: None, "linear", "bands" or
        "ramp" (``low`` and ``high``: turns within the ``original`` length)."""
        table = torch.empty(n_pos, rot_dim // 2, 2, dtype=torch.float32, device=self.device)
        _need(scaling in _SCALINGS, f"scaling: one of {list(_SCALINGS)} is wanted")
        f = _abi.RopeFreqs(base, factor, low, high, original, mscale, rot_dim,
                           _SCALINGS[scaling])
        self._done(self.lib.apx_rope_table_async(self.ctx, C.byref(f), n_pos, table.data_ptr(),
                                                 self._stream(stream)), "rope_table")
        return table

    def rope_kv4_append(self, q, k, v, table, cache: KV4Cache, batch: SeqBatch, *, rot_dim,
                        layout="half", q_out=None, q_type=torch.float32, k_deq=None, v_deq=None,
                        status=None, stream=None):
        """q (tokens, heads, dim; None to leave out) turned into ``q_out``; k turned and v
        (tokens, kv heads, dim) appended to the cache in 4 bits.  ``k_deq`` / ``v_deq`` (f16):
        the values the cache now holds.  Returns q_out."""
        f32, t = torch.float32, batch.n_tokens
        kv = (t, cache.n_kv_heads, cache.head_dim)
        a = _abi.RopeArgs()
        a.d_k, a.ldk = _rows(k, kv, "k", f32)
        a.d_v, a.ldv = _rows(v, kv, "v", f32)
        if q is not None:
            shape = (t, q.shape[1], cache.head_dim)
            if q_out is None:
                q_out = torch.empty(shape, dtype=q_type, device=q.device)
            a.d_q, a.ldq = _rows(q, shape, "q", f32)
            a.d_q_out, a.ldq_out = _rows(q_out, shape, "q_out")
            a.n_heads, a.q_type = shape[1], _TYPES.get(q_out.dtype, -1)
        n_pos = table.shape[0]
        a.d_table = _vector(table, n_pos * rot_dim, f32, "table")
        a.n_pos, a.rot_dim = n_pos, rot_dim
        a.layout = _LAYOUTS.get(layout, -1)
        if k_deq is not None:
            a.d_k_deq = _vector(k_deq, t * kv[1] * kv[2], torch.float16, "k_deq")
        if v_deq is not None:
            a.d_v_deq = _vector(v_deq, t * kv[1] * kv[2], torch.float16, "v_deq")
        if status is not None:
            a.d_status = _vector(status, 2, torch.int64, "status")
        self._done(self.lib.apx_rope_kv4_append_async(self.ctx, C.byref(a), cache.ref, batch.ref,
                                                      self._stream(stream)), "rope_kv4_append")
        return q_out

    def attn_kv4(self, q, cache: KV4Cache, batch: SeqBatch, scale, *, window=0, sinks=0,
                 out=None, status=None, stream=None):
        """softmax(scale * q k^T) v of q (tokens, heads, dim; f32, f16 or bf16) over the cache,
        causal, within ``window`` keys (0: all) and the first ``sinks``.  Returns out."""
        shape = (batch.n_tokens, q.shape[1], cache.head_dim)
        if out is None:
            out = torch.empty(shape, dtype=q.dtype, device=q.device)
        a = _abi.AttnArgs()
        a.d_q, a.ldq = _rows(q, shape, "q")
        a.d_out, a.ldo = _rows(out, shape, "out", q.dtype)
        a.type, a.n_heads = _TYPES.get(q.dtype, -1), shape[1]
        a.scale, a.window, a.sinks = scale, window, sinks
        if status is not None:
            a.d_status = _vector(status, 2, torch.int64, "status")
        self._done(self.lib.apx_attn_kv4_async(self.ctx, C.byref(a), cache.ref, batch.ref,
                                               self._stream(stream)), "attn_kv4")
        return out

    def sample(self, logits, u, *, temperature=None, top_k=None, top_p=None, min_p=None,
               token=None, prob=None, kept=None, stream=None):
        """One token per row of f32 ``logits`` (rows, vocab) from ``u`` (rows) in [0, 1); the
        filters are per row, None to leave out.  Returns token (int32)."""
        rows, vocab = logits.shape
        f32, i32 = torch.float32, torch.int32
        if token is None:
            token = torch.empty(rows, dtype=i32, device=logits.device)
        a = _abi.SampleArgs()
        a.d_logits, a.ld = _rows(logits, logits.shape, "logits", f32)
        a.d_u = _vector(u, rows, f32, "u")
        a.d_temperature = _vector(temperature, rows, f32, "temperature")
        a.d_top_k = _vector(top_k, rows, i32, "top_k")
        a.d_top_p = _vector(top_p, rows, f32, "top_p")
        a.d_min_p = _vector(min_p, rows, f32, "min_p")
        a.d_token = _vector(token, rows, i32, "token")
        a.d_prob = _vector(prob, rows, f32, "prob")
        a.d_kept = _vector(kept, rows, i32, "kept")
        a.rows, a.vocab = rows, vocab
        self._done(self.lib.apx_sample_async(self.ctx, C.byref(a), self._stream(stream)),
                   "sample")
        return token
