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


def scratch(nbytes: int, device: torch.device) -> torch.Tensor:
    """Workspace of ``device``'s current stream, grown as needed: calls on a
    stream are ordered and share it, calls on different streams do not meet.  A
    captured call takes memory of its graph's pool instead."""
    if torch.cuda.is_current_stream_capturing():
        return torch.empty(nbytes, dtype=torch.uint8, device=device)
    key = (device.index, _lib.stream_of(device.index))
    buf = _scratch.get(key)
    if buf is None or buf.numel() < nbytes:
        buf = _scratch[key] = torch.empty(nbytes, dtype=torch.uint8, device=device)
    return buf


def rows_of(x: torch.Tensor) -> torch.Tensor:
    """``x`` with contiguous rows at 16-byte boundaries, copied only where it has none."""
    if not x.is_contiguous():
        inner = 1
        for n, st in zip(reversed(x.shape[1:]), reversed(x.stride()[1:])):
            if n != 1 and st != inner:
                return x.contiguous()
            inner *= n
    if x.data_ptr() % 16 or (x.shape[0] > 1 and x.stride(0) * x.element_size() % 16):
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
        if key_pages.shape[0] == 0 or key_pages.shape[1] == 0:
            raise ValueError("the pool has no pages or no heads")
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
        self.device, self._index = kp.device, kp.get_device()
        self._kv = _KV(kp.data_ptr(), vp.data_ptr(), ks.data_ptr(), vs.data_ptr(), self.num_pages, self.kv_heads,
                       self.page_size, self.head_dim)
        self._kv_ref = byref(self._kv)
        self._need: dict[tuple[int, int], int] = {}  # attention workspace by (q_heads, max_new_tokens)

    # ----------------------------------------------------------------- batch
    def _batch(self, rows: int, lengths: torch.Tensor, block_table: torch.Tensor, token_starts: torch.Tensor | None,
               max_new_tokens: int | None) -> _Batch:
        dev, index = self.device, self._index
        if (lengths.dtype is not torch.int32 or lengths.dim() != 1 or lengths.get_device() != index
                or not lengths.is_contiguous()):
            raise ValueError(f"lengths must be contiguous int32 [seqs] on {dev}")
        seqs = lengths.numel()
        if seqs > MAX_SEQS:
            raise ValueError(f"at most {MAX_SEQS} sequences in a batch, got {seqs}")
        table_seqs, width = block_table.shape if block_table.dim() == 2 else (-1, 0)
        if (block_table.dtype is not torch.int32 or table_seqs != seqs or block_table.get_device() != index
                or (width > 1 and block_table.stride(1) != 1)):
            raise ValueError(f"block_table must be int32 [{seqs}, pages] on {dev} with contiguous rows")
        starts = None
        if token_starts is None:
            if rows != seqs:
                raise ValueError(f"without token_starts every sequence brings one row: {seqs} sequences, {rows} rows")
            most = 1
        else:
            if (token_starts.dtype is not torch.int32 or token_starts.dim() != 1
                    or token_starts.get_device() != index or token_starts.numel() != seqs + 1
                    or not token_starts.is_contiguous()):
                raise ValueError(f"token_starts must be contiguous int32 [{seqs + 1}] on {dev}")
            starts = token_starts.data_ptr()
            most = rows if max_new_tokens is None else max_new_tokens
            if most < 0:
                raise ValueError("max_new_tokens must not be negative")
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
        if _lib.current_device() != self._index:
            with torch.cuda.device(self.device):
                return self.append(qkv, cos, sin, lengths=lengths, block_table=block_table, token_starts=token_starts,
                                   max_new_tokens=max_new_tokens, interleaved=interleaved, out=out)
        d, Hkv = self.head_dim, self.kv_heads
        if qkv.dim() != 2 or qkv.get_device() != self._index:
            raise ValueError(f"qkv must be [rows, (q_heads + {2 * Hkv}) * {d}] on {self.device}")
        rows, width = qkv.shape
        q_heads = width // d - 2 * Hkv
        if width % d or q_heads < 0 or q_heads % Hkv:
            raise ValueError(f"qkv width {width} must be (q_heads + {2 * Hkv}) * {d} with q_heads a multiple of {Hkv}")
        code = _lib.dtype_code(qkv.dtype)
        batch = self._batch(rows, lengths, block_table, token_starts, max_new_tokens)
        rotary, positions, cp, sp = 0, 0, None, None
        if cos is not None or sin is not None:
            if (cos is None or sin is None or cos.dim() != 2 or cos.shape != sin.shape
                    or cos.dtype is not torch.float32 or sin.dtype is not torch.float32
                    or cos.get_device() != self._index or sin.get_device() != self._index
                    or not cos.is_contiguous() or not sin.is_contiguous()):
                raise ValueError(f"cos and sin must be contiguous fp32 tables [positions, rotary_dim / 2] on {self.device}")
            positions, rotary = cos.shape
            rotary *= 2
            if rotary % 16 or rotary > d:
                raise ValueError(f"rotary_dim must be a multiple of 16 up to {d}, got {rotary}")
            cp, sp = cos.data_ptr(), sin.data_ptr()
        qkv = rows_of(qkv)
        if out is None:
            out = qkv.new_empty((rows, q_heads, d))
        elif (out.shape != (rows, q_heads, d) or out.dtype is not qkv.dtype or out.get_device() != self._index
              or not out.is_contiguous()):
            raise ValueError(f"out must be contiguous {qkv.dtype} [{rows}, {q_heads}, {d}]")
        status = lib.tq_paged_append(self._kv_ref, byref(batch), qkv.data_ptr(), code, qkv.stride(0), q_heads, cp, sp,
                                     positions, rotary, interleaved, out.data_ptr(), _lib.stream_of(self._index))
        if status:
            _lib.check(status, "paged append")
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
        if _lib.current_device() != self._index:
            with torch.cuda.device(self.device):
                return self.attend(q, lengths=lengths, block_table=block_table, token_starts=token_starts,
                                   max_new_tokens=max_new_tokens, max_context=max_context,
                                   lengths_counted=lengths_counted, scale=scale, return_lse=return_lse, out=out)
        d = self.head_dim
        rows, q_heads, width = q.shape if q.dim() == 3 else (0, 0, 0)
        if width != d or q.get_device() != self._index:
            raise ValueError(f"q must be [rows, q_heads, {d}] on {self.device}")
        if q_heads == 0 or q_heads % self.kv_heads:
            raise ValueError(f"q_heads {q_heads} must be a positive multiple of kv_heads {self.kv_heads}")
        dtype = q.dtype
        if dtype is not torch.bfloat16 and dtype is not torch.float16:
            raise ValueError(f"q must be float16 or bfloat16, got {dtype}")
        batch = self._batch(rows, lengths, block_table, token_starts, max_new_tokens)
        if max_context is None:
            max_context = batch.table_width * self.page_size
        elif max_context < 0:
            raise ValueError("max_context must not be negative")
        q = rows_of(q)
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        elif (out.shape != (rows, q_heads, d) or out.dtype is not dtype or out.get_device() != self._index
              or not out.is_contiguous()):
            raise ValueError(f"out must be contiguous {dtype} {(rows, q_heads, d)}")
        lse = torch.empty((rows, q_heads), dtype=torch.float32, device=self.device) if return_lse else None
        need = self._workspace(q_heads, batch.max_new_tokens)
        ws = scratch(need, self.device)
        status = lib.tq_paged_attend(
            self._kv_ref, byref(batch), q.data_ptr(), _lib.TQ_BF16 if dtype is torch.bfloat16 else _lib.TQ_F16,
            q.stride(0), q_heads, lengths_counted, d ** -0.5 if scale is None else scale, max_context, out.data_ptr(),
            None if lse is None else lse.data_ptr(), ws.data_ptr(), need, _lib.stream_of(self._index))
        if status:
            _lib.check(status, "paged attend")
        return (out, lse) if return_lse else out

    def _workspace(self, q_heads: int, max_new_tokens: int) -> int:
        """Bytes of an attention's workspace, asked once for each pair."""
        key = (q_heads, max_new_tokens)
        need = self._need.get(key)
        if need is None:
            size = c_size_t()
            _lib.check(_lib.load().tq_paged_attend_workspace_size(self._kv_ref, q_heads, max_new_tokens, byref(size)),
                       "paged attend")
            need = self._need[key] = size.value
        return need

    # ------------------------------------------------------------ dequantize
    def dequantize(self, page_ids: torch.Tensor, *, dtype: torch.dtype = torch.bfloat16):
        """The values of pages: ``(keys, values)``, each ``[n, kv_heads,
        page_size, d]`` (tq_paged_dequantize); NaN for an id outside the pool."""
        lib = _lib.load()
        if _lib.current_device() != self._index:
            with torch.cuda.device(self.device):
                return self.dequantize(page_ids, dtype=dtype)
        if (page_ids.dtype is not torch.int32 or page_ids.dim() != 1 or page_ids.get_device() != self._index
                or not page_ids.is_contiguous()):
            raise ValueError(f"page_ids must be contiguous int32 [n] on {self.device}")
        code = _lib.dtype_code(dtype)
        n = page_ids.numel()
        shape = (n, self.kv_heads, self.page_size, self.head_dim)
        k = torch.empty(shape, dtype=dtype, device=self.device)
        v = torch.empty_like(k)
        status = lib.tq_paged_dequantize(self._kv_ref, page_ids.data_ptr(), n, k.data_ptr(), v.data_ptr(), code,
                                         _lib.stream_of(self._index))
        if status:
            _lib.check(status, "paged dequantize")
        return k, v
