"""Host-side argument checks of the serving operators' C ABI (no GPU needed):
each is answered with a status before anything is launched."""

from __future__ import annotations

import ctypes

import pytest

from torque_mlx_b200 import _lib
from torque_mlx_b200.paged import _KV


class _Batch(ctypes.Structure):
    """tq_paged_batch"""
    _fields_ = [("block_table", ctypes.c_void_p), ("lengths", ctypes.c_void_p), ("token_starts", ctypes.c_void_p),
                ("table_stride", ctypes.c_int64), ("rows", ctypes.c_int64), ("table_width", ctypes.c_int32),
                ("seqs", ctypes.c_int32), ("max_new_tokens", ctypes.c_int32)]


@pytest.fixture(scope="module")
def lib():
    from torque_mlx_b200.build import build_library
    build_library()
    return _lib.load(require_cuda=False)


def kv(**kw):
    f = dict(k_pages=256, v_pages=256, k_scales=256, v_scales=256, num_pages=4, kv_heads=2, page_size=16, head_dim=64)
    f.update(kw)
    return _KV(*f.values())


def batch(**kw):
    f = dict(block_table=256, lengths=256, token_starts=None, table_stride=4, rows=2, table_width=4, seqs=2,
             max_new_tokens=1)
    f.update(kw)
    return _Batch(*f.values())


def attend(lib, k, b, q=256, dtype=_lib.TQ_BF16, stride=256, heads=4, out=256, ws=256, ws_bytes=1 << 30, context=64):
    return lib.tq_paged_attend(ctypes.byref(k), ctypes.byref(b), q, dtype, stride, heads, 0, 1.0, context, out, None, ws,
                               ws_bytes, None)


def test_attend_refusals(lib):
    for bad, status in ((dict(head_dim=96), _lib.TQ_E_HEAD_DIM), (dict(page_size=48), _lib.TQ_E_SHAPE),
                        (dict(kv_heads=0), _lib.TQ_E_SHAPE), (dict(num_pages=0), _lib.TQ_E_SHAPE),
                        (dict(k_pages=None), _lib.TQ_E_ARG), (dict(v_pages=8), _lib.TQ_E_SHAPE)):
        assert attend(lib, kv(**bad), batch()) == status, bad
    for bad, status in ((dict(seqs=-1), _lib.TQ_E_SHAPE), (dict(rows=3), _lib.TQ_E_SHAPE),
                        (dict(lengths=None), _lib.TQ_E_ARG), (dict(block_table=None), _lib.TQ_E_ARG),
                        (dict(table_stride=3), _lib.TQ_E_SHAPE), (dict(max_new_tokens=-1), _lib.TQ_E_SHAPE),
                        (dict(seqs=3000, rows=3000), _lib.TQ_E_SHAPE)):
        assert attend(lib, kv(), batch(**bad)) == status, bad
    for bad, status in ((dict(dtype=_lib.TQ_F32), _lib.TQ_E_ARG), (dict(heads=3), _lib.TQ_E_SHAPE),
                        (dict(stride=8), _lib.TQ_E_SHAPE), (dict(stride=260), _lib.TQ_E_SHAPE), (dict(q=None), _lib.TQ_E_ARG),
                        (dict(q=8), _lib.TQ_E_SHAPE), (dict(out=16), _lib.TQ_E_SHAPE), (dict(context=-1), _lib.TQ_E_SHAPE),
                        (dict(ws=None), _lib.TQ_E_WORKSPACE), (dict(ws_bytes=64), _lib.TQ_E_WORKSPACE)):
        assert attend(lib, kv(), batch(), **bad) == status, bad
    assert attend(lib, kv(), batch(seqs=0, rows=0)) == _lib.TQ_OK


def test_append_refusals(lib):
    def append(k=None, b=None, x=256, dtype=_lib.TQ_F16, stride=512, heads=4, cos=256, sin=256, rotary=64, q=256):
        return lib.tq_paged_append(ctypes.byref(k or kv()), ctypes.byref(b or batch()), x, dtype, stride, heads, cos, sin,
                                   10, rotary, 1, q, None)

    for bad, status in ((dict(dtype=9), _lib.TQ_E_ARG), (dict(heads=3), _lib.TQ_E_SHAPE), (dict(stride=100), _lib.TQ_E_SHAPE),
                        (dict(rotary=24), _lib.TQ_E_SHAPE), (dict(rotary=128), _lib.TQ_E_SHAPE), (dict(x=None), _lib.TQ_E_ARG),
                        (dict(q=None), _lib.TQ_E_ARG), (dict(cos=None), _lib.TQ_E_ARG), (dict(sin=4), _lib.TQ_E_SHAPE)):
        assert append(**bad) == status, bad
    assert append(b=batch(seqs=0, rows=0)) == _lib.TQ_OK


def test_w4_sizes_and_refusals(lib):
    code, scale = ctypes.c_size_t(), ctypes.c_size_t()

    def sizes(n, k, g):
        return lib.tq_w4_sizes(n, k, g, ctypes.byref(code), ctypes.byref(scale))

    assert sizes(17, 130, 64) == _lib.TQ_OK and code.value == 2 * 2 * 1024 and scale.value == 2 * 2 * 64
    for n, k, g in ((0, 64, 64), (4, 0, 64), (4, 64, 48)):
        assert sizes(n, k, g) == _lib.TQ_E_SHAPE

    def gemv(codes=256, x=256, dtype=_lib.TQ_BF16, stride=64, mode=0, tokens=2, group=64, norm=None, y=256):
        return lib.tq_gemv_w4(codes, 256, 32, 64, group, x, dtype, stride, mode, norm, 0.0, None, y, tokens, None, 0, None)

    for bad, status in ((dict(group=16), _lib.TQ_E_SHAPE), (dict(mode=4), _lib.TQ_E_ARG), (dict(dtype=_lib.TQ_F32), _lib.TQ_E_ARG),
                        (dict(dtype=_lib.TQ_F16, mode=2), _lib.TQ_E_ARG), (dict(stride=32), _lib.TQ_E_SHAPE),
                        (dict(tokens=-1), _lib.TQ_E_SHAPE), (dict(codes=None), _lib.TQ_E_ARG), (dict(codes=8), _lib.TQ_E_SHAPE),
                        (dict(mode=2), _lib.TQ_E_ARG), (dict(y=None), _lib.TQ_E_ARG)):
        assert gemv(**bad) == status, bad
    assert gemv(tokens=0) == _lib.TQ_OK
    need = ctypes.c_size_t()
    # 32 tokens of 8192 columns do not fit beside the ring: their columns are split, and the parts need room
    assert lib.tq_gemv_w4_workspace_size(64, 8192, 32, ctypes.byref(need)) == _lib.TQ_OK and need.value > 0
    assert lib.tq_gemv_w4(256, 256, 64, 8192, 64, 256, _lib.TQ_BF16, 8192, 0, None, 0.0, None, 256, 32, None, 0,
                          None) == _lib.TQ_E_WORKSPACE


def test_verify_refusals(lib):
    def verify(target=256, row=100, dtype=_lib.TQ_F32, noise=256, seqs=1, drafts=2, vocab=100, tokens=256):
        return lib.tq_verify_drafts(target, 300, row, None, 0, 0, dtype, tokens, None, 256, noise, vocab, seqs, drafts, vocab,
                                    256, 256, None)

    for bad, status in ((dict(dtype=5), _lib.TQ_E_ARG), (dict(vocab=0), _lib.TQ_E_SHAPE), (dict(seqs=-1), _lib.TQ_E_SHAPE),
                        (dict(row=50), _lib.TQ_E_SHAPE), (dict(target=None), _lib.TQ_E_ARG), (dict(noise=None), _lib.TQ_E_ARG),
                        (dict(tokens=None), _lib.TQ_E_ARG), (dict(drafts=-1), _lib.TQ_E_SHAPE)):
        assert verify(**bad) == status, bad
    assert verify(seqs=0) == _lib.TQ_OK
