"""Linear layers with 4-bit weights and group scales, for a few tokens.

``W4Weight`` holds a weight ``[n, k]`` as codes ``0..15`` and a bf16 scale for
each row and group of columns, ``w = scale * (code - 8)``, in the order that
the product's kernel reads (laid out once).  ``gemv_w4`` multiplies it with one
to a few tokens; like ``ops.gemv`` it can build its input from an fp32 row, an
RMSNorm or a SwiGLU activation on the way and add a residual.
"""

from __future__ import annotations

from ctypes import byref, c_size_t

import torch

from . import _lib

GROUP_SIZES = (32, 64, 128)
_MODES = {"plain": 0, "f32": 1, "rms": 2, "silu": 3}


class W4Weight:
    """A 4-bit weight ``[n, k]`` laid out for ``gemv_w4``: the codes and scales
    as tq_w4_layout wrote them (``from_packed`` and ``quantize`` make them)."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, n: int, k: int, group_size: int):
        for t, name, size in zip((codes, scales), ("codes", "scales"), self._check_sizes(n, k, group_size)):
            if t.dtype != torch.uint8 or t.numel() != size or not t.is_cuda or not t.is_contiguous() or t.data_ptr() % 16:
                raise ValueError(f"{name} of a weight [{n}, {k}] must be {size} contiguous bytes (uint8) at a 16-byte "
                                 "boundary on a CUDA device")
        if scales.device != codes.device:
            raise ValueError(f"scales must be on {codes.device}")
        self.codes, self.scales = codes, scales
        self.n, self.k, self.group_size = n, k, group_size
        self.device = codes.device

    @staticmethod
    def _check_sizes(n: int, k: int, group_size: int) -> tuple[int, int]:
        lib = _lib.load()
        if group_size not in GROUP_SIZES:
            raise ValueError(f"group_size must be one of {GROUP_SIZES}, got {group_size}")
        code_bytes, scale_bytes = c_size_t(), c_size_t()
        _lib.check(lib.tq_w4_sizes(n, k, group_size, byref(code_bytes), byref(scale_bytes)), "w4 weight")
        return code_bytes.value, scale_bytes.value

    @classmethod
    def from_packed(cls, packed: torch.Tensor, scales: torch.Tensor, *, k: int, group_size: int) -> "W4Weight":
        """From bytes ``[n, ceil(k/2)]`` (column 2i in the low half) and bf16
        scales ``[n, ceil(k/group_size)]``."""
        lib = _lib.load()
        if packed.dtype != torch.uint8 or packed.dim() != 2 or not packed.is_cuda or packed.shape[1] != (k + 1) // 2:
            raise ValueError(f"packed must be uint8 [n, {(k + 1) // 2}] on a CUDA device")
        n = packed.shape[0]
        code_bytes, scale_bytes = cls._check_sizes(n, k, group_size)
        groups = -(-k // group_size)
        if scales.dtype != torch.bfloat16 or tuple(scales.shape) != (n, groups) or scales.device != packed.device:
            raise ValueError(f"scales must be bf16 [{n}, {groups}] on {packed.device}")
        packed, scales = packed.contiguous(), scales.contiguous()
        codes = torch.empty(code_bytes, dtype=torch.uint8, device=packed.device)
        laid = torch.empty(scale_bytes, dtype=torch.uint8, device=packed.device)
        with torch.cuda.device(packed.device):
            _lib.check(lib.tq_w4_layout(packed.data_ptr(), scales.data_ptr(), n, k, group_size, codes.data_ptr(),
                                        laid.data_ptr(), _lib.stream_ptr()), "w4 layout")
        return cls(codes, laid, n, k, group_size)

    @classmethod
    def quantize(cls, weight: torch.Tensor, *, group_size: int = 128) -> "W4Weight":
        """Nearest codes of a dense weight ``[n, k]`` (fp32, fp16 or bf16) with
        scale = max|w| / 7 of each group (tq_w4_quantize)."""
        packed, scales = quantize_w4(weight, group_size=group_size)
        return cls.from_packed(packed, scales, k=weight.shape[1], group_size=group_size)

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The dense weight ``[n, k]``."""
        lib = _lib.load()
        out = torch.empty((self.n, self.k), dtype=dtype, device=self.device)
        with torch.cuda.device(self.device):
            _lib.check(lib.tq_w4_dequantize(self.codes.data_ptr(), self.scales.data_ptr(), self.n, self.k,
                                            self.group_size, out.data_ptr(), _lib.dtype_code(dtype),
                                            _lib.stream_ptr()), "w4 dequantize")
        return out


def quantize_w4(weight: torch.Tensor, *, group_size: int = 128) -> tuple[torch.Tensor, torch.Tensor]:
    """``(packed [n, ceil(k/2)] uint8, scales [n, groups] bf16)`` of a dense weight."""
    lib = _lib.load()
    if weight.dim() != 2 or not weight.is_cuda:
        raise ValueError("weight must be a CUDA tensor [n, k]")
    code = _lib.dtype_code(weight.dtype)
    n, k = weight.shape
    W4Weight._check_sizes(n, k, group_size)
    weight = weight.contiguous()
    packed = torch.empty((n, (k + 1) // 2), dtype=torch.uint8, device=weight.device)
    scales = torch.empty((n, -(-k // group_size)), dtype=torch.bfloat16, device=weight.device)
    with torch.cuda.device(weight.device):
        _lib.check(lib.tq_w4_quantize(weight.data_ptr(), code, n, k, group_size, packed.data_ptr(), scales.data_ptr(),
                                      _lib.stream_ptr()), "w4 quantize")
    return packed, scales


def gemv_w4(weight: W4Weight, x: torch.Tensor, *, mode: str = "plain", norm_weight: torch.Tensor | None = None,
            eps: float = 0.0, residual: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``y = x' W^T (+ residual)`` for tokens ``x`` ``[tokens, k]`` (or one
    ``[k]``; tq_gemv_w4).  ``x'`` is ``x`` (mode "plain", fp16 or bf16), bf16 of
    an fp32 ``x`` ("f32"), its RMSNorm ("rms", with ``norm_weight`` / ``eps``)
    or the SwiGLU activation of ``[gate | up]`` rows of ``2k`` ("silu").
    Returns ``[tokens, n]`` (or ``[n]``) in x's type (bf16 for "f32").  Made for
    few tokens: the weight is read once for each 32 of them."""
    code = _MODES.get(mode)
    if code is None:
        raise ValueError(f"mode must be one of {sorted(_MODES)}")
    return _lib.binding().gemv_w4(weight.codes, weight.scales, weight.n, weight.k, weight.group_size, x, code, norm_weight,
                                  eps, residual, out)
