"""Paged 8-bit KV cache: rotary append and causal attention of ragged batches.

A ``PagedKV8Cache`` is the pool of one layer: pages of ``page_size`` tokens
whose keys and values are one-byte codes with one fp32 scale for each page and
kv head.  Sequences are lists of pages in a block table; their lengths, the
block table and the row starts of a ragged batch are device tensors that the
kernels read, so a step needs no host round trip and can be captured in a CUDA
graph.  One sequence brings one token (decoding), a few (drafted tokens to be
verified) or many (a prompt's chunk), mixed freely in a batch:

    q = cache.append(qkv, cos, sin, lengths=lengths, block_table=table)
    out = cache.attend(q, lengths=lengths, block_table=table)
    lengths += 1

``lengths`` counts the tokens held before the step: the append writes behind
them, and the attention sees the written tokens causally.  Advancing the
lengths afterwards, by as many tokens as are kept, is the caller's, so drafted
tokens that are rejected need no undoing.
"""

from __future__ import annotations

from ctypes import Structure, byref, c_int32, c_int64, c_size_t, c_void_p

import torch

from . import _lib
from .config import validate_head_dim

PAGE_SIZES = (16, 32, 64, 128)
MAX_SEQS = 2048  # TQ_PAGED_MAX_SEQS


class _KV(Structure):
    """tq_paged_kv"""
    _fields_ = [("k_pages", c_void_p), ("v_pages", c_void_p), ("k_scales", c_void_p), ("v_scales", c_void_p),
                ("num_pages", c_int64), ("kv_heads", c_int32), ("page_size", c_int32), ("head_dim", c_int32)]


class _Batch(Structure):
    """tq_paged_batch"""
    _fields_ = [("block_table", c_void_p), ("lengths", c_void_p), ("token_starts", c_void_p),
                ("table_stride", c_int64), ("rows", c_int64), ("table_width", c_int32), ("seqs", c_int32),
                ("max_new_tokens", c_int32)]


_scratch: dict[tuple[int, int], torch.Tensor] = {}


def scratch(nbytes: int, device: torch.device, stream: int) -> torch.Tensor:
    """Workspace of one stream, grown as needed: calls on a stream are ordered
    and share it, calls on different streams do not meet.  A captured call
    takes memory of its graph's pool instead."""
    if torch.cuda.is_current_stream_capturing():
        return torch.empty(nbytes, dtype=torch.uint8, device=device)
    key = (device.index, stream)
    buf = _scratch.get(key)
    if buf is None or buf.numel() < nbytes:
        buf = _scratch[key] = torch.empty(nbytes, dtype=torch.uint8, device=device)
    return buf


def rows_of(x: torch.Tensor) -> torch.Tensor:
    """``x`` with contiguous rows at 16-byte boundaries, copied only where it has none."""
    item = x.element_size()
    inner = 1
    for n, st in zip(reversed(x.shape[1:]), reversed(x.stride()[1:])):
        if n != 1 and st != inner:
            return x.contiguous()
        inner *= n
    if x.data_ptr() % 16 or (x.shape[0] > 1 and x.stride(0) * item % 16):
        return x.clone(memory_format=torch.contiguous_format)
    return x


class PagedKV8Cache:
    """Pool of ``num_pages`` pages of 8-bit keys and values of one layer."""

    def __init__(self, num_pages: int, *, kv_heads: int, head_dim: int, page_size: int = 64,
                 device: torch.device | str | None = None):
        if num_pages <= 0:
            raise ValueError("num_pages must be positive")
        if kv_heads <= 0:
            raise ValueError("kv_heads must be positive")
        validate_head_dim(head_dim)
        if page_size not in PAGE_SIZES:
            raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {page_size}")
        _lib.load()
        dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        shape = (num_pages, kv_heads, page_size, head_dim)
        self._bind(torch.full(shape, 128, dtype=torch.uint8, device=dev),
                   torch.full(shape, 128, dtype=torch.uint8, device=dev),
                   torch.zeros(shape[:2], dtype=torch.float32, device=dev),
                   torch.zeros(shape[:2], dtype=torch.float32, device=dev))

    @classmethod
    def from_pages(cls, key_pages: torch.Tensor, value_pages: torch.Tensor, key_scales: torch.Tensor,
                   value_scales: torch.Tensor) -> "PagedKV8Cache":
        """Cache over existing buffers, which it shares: codes ``[num_pages,
        kv_heads, page_size, d]`` uint8 (biased by 128) and scales ``[num_pages,
        kv_heads]`` fp32."""
        _lib.load()
        for t, name in ((key_pages, "key_pages"), (value_pages, "value_pages")):
            if t.dtype != torch.uint8 or t.dim() != 4 or not t.is_cuda or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous uint8 CUDA tensor [pages, kv_heads, page_size, head_dim]")
        for t, name in ((key_scales, "key_scales"), (value_scales, "value_scales")):
            if t.dtype != torch.float32 or tuple(t.shape) != tuple(key_pages.shape[:2]) or not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous fp32 [pages, kv_heads]")
            if t.device != key_pages.device:
                raise ValueError(f"{name} must be on {key_pages.device}")
        if value_pages.shape != key_pages.shape or value_pages.device != key_pages.device:
            raise ValueError("key_pages and value_pages must match in shape and device")
        validate_head_dim(int(key_pages.shape[3]))
        if key_pages.shape[2] not in PAGE_SIZES:
            raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {key_pages.shape[2]}")
        if key_pages.data_ptr() % 16 or value_pages.data_ptr() % 16:
            raise ValueError("key_pages and value_pages must start at 16-byte boundaries")
        self = cls.__new__(cls)
        self._bind(key_pages, value_pages, key_scales, value_scales)
        return self

    def _bind(self, kp: torch.Tensor, vp: torch.Tensor, ks: torch.Tensor, vs: torch.Tensor) -> None:
        self.key_pages, self.value_pages, self.key_scales, self.value_scales = kp, vp, ks, vs
        self.num_pages, self.kv_heads, self.page_size, self.head_dim = (int(n) for n in kp.shape)
        self.device = kp.device
        self._kv = _KV(kp.data_ptr(), vp.data_ptr(), ks.data_ptr(), vs.data_ptr(), self.num_pages, self.kv_heads,
                       self.page_size, self.head_dim)
        self._kv_ref = byref(self._kv)
        self._need: dict[tuple[int, int], int] = {}  # attention workspace by (q_heads, max_new_tokens)

    # ----------------------------------------------------------------- batch
    def _batch(self, rows: int, lengths: torch.Tensor, block_table: torch.Tensor, token_starts: torch.Tensor | None,
               max_new_tokens: int | None) -> _Batch:
        dev = self.device
        if lengths.dtype != torch.int32 or lengths.dim() != 1 or lengths.device != dev or not lengths.is_contiguous():
            raise ValueError(f"lengths must be contiguous int32 [seqs] on {dev}")
        seqs = lengths.shape[0]
        if seqs > MAX_SEQS:
            raise ValueError(f"at most {MAX_SEQS} sequences in a batch, got {seqs}")
        if (block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.device != dev
                or block_table.shape[0] != seqs or (block_table.shape[1] > 1 and block_table.stride(1) != 1)):
            raise ValueError(f"block_table must be int32 [{seqs}, pages] on {dev} with contiguous rows")
        starts = None
        if token_starts is None:
            if rows != seqs:
                raise ValueError(f"without token_starts every sequence brings one row: {seqs} sequences, {rows} rows")
            most = 1
        else:
            if (token_starts.dtype != torch.int32 or token_starts.dim() != 1 or token_starts.device != dev
                    or token_starts.shape[0] != seqs + 1 or not token_starts.is_contiguous()):
                raise ValueError(f"token_starts must be contiguous int32 [{seqs + 1}] on {dev}")
            starts = token_starts.data_ptr()
            most = rows if max_new_tokens is None else max_new_tokens
            if most < 0:
                raise ValueError("max_new_tokens must not be negative")
        width = block_table.shape[1]
        return _Batch(block_table.data_ptr(), lengths.data_ptr(), starts,
                      block_table.stride(0) if seqs > 1 else width, rows, width, seqs, min(most, rows))

    # ---------------------------------------------------------------- append
    def append(self, qkv: torch.Tensor, cos: torch.Tensor | None = None, sin: torch.Tensor | None = None, *,
               lengths: torch.Tensor, block_table: torch.Tensor, token_starts: torch.Tensor | None = None,
               max_new_tokens: int | None = None, interleaved: bool = True,
               out: torch.Tensor | None = None) -> torch.Tensor:
        """Write the rows' keys and values behind each sequence's tokens and
        return the rotated queries ``[rows, q_heads, d]`` (tq_paged_append).

        ``qkv`` is ``[rows, (q_heads + 2 kv_heads) * d]`` (fp16, bf16 or fp32,
        row stride free); rows ``token_starts[s]`` to ``token_starts[s + 1]``
        belong to sequence ``s`` (row ``s`` without ``token_starts``) and take
        the positions from ``lengths[s]`` on.  ``cos`` / ``sin`` are fp32
        ``[positions, rotary_dim / 2]`` tables; pairs are ``(2i, 2i + 1)``, or
        ``(i, i + rotary_dim / 2)`` with ``interleaved=False``.  Without them
        nothing is rotated.  The lengths are not advanced.  Rows that belong to
        no sequence leave their part of the result unwritten; a row whose
        position has no table row is not written and its query is NaN; a row
        whose page is missing is not written."""
        lib = _lib.load()
        d, Hkv = self.head_dim, self.kv_heads
        if qkv.dim() != 2 or qkv.device != self.device:
            raise ValueError(f"qkv must be [rows, (q_heads + {2 * Hkv}) * {d}] on {self.device}")
        rows, width = qkv.shape
        q_heads = width // d - 2 * Hkv
        if width % d or q_heads < 0 or q_heads % Hkv:
            raise ValueError(f"qkv width {width} must be (q_heads + {2 * Hkv}) * {d} with q_heads a multiple of {Hkv}")
        code = _lib.dtype_code(qkv.dtype)
        batch = self._batch(rows, lengths, block_table, token_starts, max_new_tokens)
        rotary, positions, cp, sp = 0, 0, None, None
        if cos is not None or sin is not None:
            if (cos is None or sin is None or cos.shape != sin.shape or cos.dim() != 2
                    or cos.dtype != torch.float32 or sin.dtype != torch.float32 or cos.device != self.device
                    or sin.device != self.device or not cos.is_contiguous() or not sin.is_contiguous()):
                raise ValueError(f"cos and sin must be contiguous fp32 tables [positions, rotary_dim / 2] on {self.device}")
            positions, rotary = cos.shape[0], 2 * cos.shape[1]
            if rotary % 16 or rotary > d:
                raise ValueError(f"rotary_dim must be a multiple of 16 up to {d}, got {rotary}")
            cp, sp = cos.data_ptr(), sin.data_ptr()
        qkv = rows_of(qkv)
        if out is None:
            out = torch.empty((rows, q_heads, d), dtype=qkv.dtype, device=self.device)
        elif (out.shape != (rows, q_heads, d) or out.dtype != qkv.dtype or out.device != self.device
              or not out.is_contiguous()):
            raise ValueError(f"out must be contiguous {qkv.dtype} [{rows}, {q_heads}, {d}]")
        with torch.cuda.device(self.device):
            _lib.check(lib.tq_paged_append(self._kv_ref, byref(batch), qkv.data_ptr(), code, qkv.stride(0), q_heads,
                                           cp, sp, positions, rotary, int(interleaved), out.data_ptr(),
                                           _lib.stream_ptr()), "paged append")
        return out

    # ---------------------------------------------------------------- attend
    def attend(self, q: torch.Tensor, *, lengths: torch.Tensor, block_table: torch.Tensor,
               token_starts: torch.Tensor | None = None, max_new_tokens: int | None = None,
               max_context: int | None = None, lengths_counted: bool = False, scale: float | None = None,
               return_lse: bool = False, out: torch.Tensor | None = None):
        """Causal attention of ``q`` ``[rows, q_heads, d]`` (fp16 or bf16) over
        the cache, which holds the rows' own tokens already (tq_paged_attend).
        Row t of sequence s sees positions up to ``lengths[s] + t``; with
        ``lengths_counted`` the lengths include the rows.  Returns q's shape and
        type, and with ``return_lse`` also the fp32 natural-log sum-exp
        ``[rows, q_heads]`` (-inf and a zero row where nothing is seen).
        ``max_context`` (a bound of any sequence's tokens, new ones included)
        sizes the launch; the result does not depend on it."""
        lib = _lib.load()
        d = self.head_dim
        if q.dim() != 3 or q.shape[2] != d or q.device != self.device:
            raise ValueError(f"q must be [rows, q_heads, {d}] on {self.device}")
        rows, q_heads, _ = q.shape
        if q_heads == 0 or q_heads % self.kv_heads:
            raise ValueError(f"q_heads {q_heads} must be a positive multiple of kv_heads {self.kv_heads}")
        if q.dtype != torch.bfloat16 and q.dtype != torch.float16:
            raise ValueError(f"q must be float16 or bfloat16, got {q.dtype}")
        batch = self._batch(rows, lengths, block_table, token_starts, max_new_tokens)
        if max_context is None:
            max_context = batch.table_width * self.page_size
        elif max_context < 0:
            raise ValueError("max_context must not be negative")
        q = rows_of(q)
        if out is None:
            out = torch.empty((rows, q_heads, d), dtype=q.dtype, device=self.device)
        elif out.shape != q.shape or out.dtype != q.dtype or out.device != self.device or not out.is_contiguous():
            raise ValueError(f"out must be contiguous {q.dtype} {tuple(q.shape)}")
        lse = torch.empty((rows, q_heads), dtype=torch.float32, device=self.device) if return_lse else None
        key = (q_heads, batch.max_new_tokens)
        with torch.cuda.device(self.device):
            need = self._need.get(key)
            if need is None:
                size = c_size_t()
                _lib.check(lib.tq_paged_attend_workspace_size(self._kv_ref, *key, byref(size)), "paged attend")
                need = self._need[key] = size.value
            stream = _lib.stream_ptr()
            ws = scratch(need, self.device, stream)
            _lib.check(lib.tq_paged_attend(
                self._kv_ref, byref(batch), q.data_ptr(), _lib.dtype_code(q.dtype), q.stride(0), q_heads,
                int(lengths_counted), float(d ** -0.5 if scale is None else scale), max_context, out.data_ptr(),
                _lib.ptr(lse), ws.data_ptr(), ws.numel(), stream), "paged attend")
        return (out, lse) if return_lse else out

    # ------------------------------------------------------------ dequantize
    def dequantize(self, page_ids: torch.Tensor, *, dtype: torch.dtype = torch.bfloat16):
        """The values of pages: ``(keys, values)``, each ``[n, kv_heads,
        page_size, d]`` (tq_paged_dequantize); NaN for an id outside the pool."""
        lib = _lib.load()
        if (page_ids.dtype != torch.int32 or page_ids.dim() != 1 or page_ids.device != self.device
                or not page_ids.is_contiguous()):
            raise ValueError(f"page_ids must be contiguous int32 [n] on {self.device}")
        code = _lib.dtype_code(dtype)
        both = torch.empty((2, page_ids.shape[0], self.kv_heads, self.page_size, self.head_dim), dtype=dtype,
                           device=self.device)
        k, v = both.unbind(0)
        with torch.cuda.device(self.device):
            _lib.check(lib.tq_paged_dequantize(self._kv_ref, page_ids.data_ptr(), page_ids.shape[0], k.data_ptr(),
                                               v.data_ptr(), code, _lib.stream_ptr()), "paged dequantize")
        return k, v
