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
lengths afterwards, by as many tokens as are kept, is the caller's: drafted
tokens that are rejected are simply written over.  They may leave a trace: one
of larger magnitude than a page's scale covers raises that scale, and the
tokens that the page held before are rounded again to it (each value stays
within half of the new scale of what it was).  So drafting is not neutral to
the last bits of what the cache holds.
"""

from __future__ import annotations

from ctypes import Structure, addressof, byref, c_int32, c_int64, c_uint32, c_void_p

import torch

from . import _lib
from .config import validate_head_dim

PAGE_SIZES = (16, 32, 64, 128)


class _KV(Structure):
    """tq_paged_kv"""
    _fields_ = [("k_pages", c_void_p), ("v_pages", c_void_p), ("k_scales", c_void_p), ("v_scales", c_void_p),
                ("num_pages", c_int64), ("kv_heads", c_int32), ("page_size", c_int32), ("head_dim", c_int32)]


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
        kv_heads]`` fp32.  The scales of pages in use must be 0 or more: a page
        of negative key scale is not attended."""
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
        self.device = kp.device
        self._kv = _KV(kp.data_ptr(), vp.data_ptr(), ks.data_ptr(), vs.data_ptr(), self.num_pages, self.kv_heads,
                       self.page_size, self.head_dim)
        self._at, self._index = addressof(self._kv), kp.get_device()

    # ---------------------------------------------------------------- append
    def append(self, qkv: torch.Tensor, cos: torch.Tensor | None = None, sin: torch.Tensor | None = None, *,
               lengths: torch.Tensor, block_table: torch.Tensor, token_starts: torch.Tensor | None = None,
               max_new_tokens: int | None = None, interleaved: bool = True,
               out: torch.Tensor | None = None) -> torch.Tensor:
        """Write the rows' keys and values behind each sequence's tokens and
        return the rotated queries ``[rows, q_heads, d]`` (tq_paged_append).

        ``qkv`` is ``[rows, (q_heads + 2 kv_heads) * d]`` (fp16, bf16 or fp32,
        row stride free; the queries come back in its type, of which ``attend``
        takes fp16 and bf16); rows ``token_starts[s]`` to ``token_starts[s + 1]``
        belong to sequence ``s`` (row ``s`` without ``token_starts``) and take
        the positions from ``lengths[s]`` on.  ``cos`` / ``sin`` are fp32
        ``[positions, rotary_dim / 2]`` tables; pairs are ``(2i, 2i + 1)``, or
        ``(i, i + rotary_dim / 2)`` with ``interleaved=False``.  Without them
        nothing is rotated.  The lengths are not advanced.  Rows that belong to
        no sequence leave their part of the result unwritten; a row whose
        position has no table row is not written and its query is NaN; a row
        whose page is missing is not written."""
        return _lib.binding().paged_append(self._at, self._index, qkv, cos, sin, lengths, block_table, token_starts,
                                           max_new_tokens, interleaved, out)

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
        ``[rows, q_heads]`` (-inf and a zero row where nothing is seen).  Rows
        that belong to no sequence leave their part of the results unwritten.
        ``max_context`` (a bound of any sequence's tokens, new ones included)
        sizes the launch; the result does not depend on it."""
        return _lib.binding().paged_attend(self._at, self._index, q, lengths, block_table, token_starts, max_new_tokens,
                                           max_context, lengths_counted, scale, return_lse, out)

    def attend_gave_up(self) -> int:
        """Thread blocks of many-row attentions on the cache's device that gave
        up a wait and left NaN behind (tq_paged_attend_gave_up), since the
        library was loaded: 0 unless something is wrong.  Waits for the current
        stream."""
        count = c_uint32()
        with torch.cuda.device(self.device):
            _lib.check(_lib.load().tq_paged_attend_gave_up(byref(count), _lib.stream_ptr()), "paged attend")
        return count.value

    # ------------------------------------------------------------ dequantize
    def dequantize(self, page_ids: torch.Tensor, *, dtype: torch.dtype = torch.bfloat16):
        """The values of pages: ``(keys, values)``, each ``[n, kv_heads,
        page_size, d]`` (tq_paged_dequantize); NaN for an id outside the pool."""
        return _lib.binding().paged_dequantize(self._at, self._index, page_ids, dtype)
