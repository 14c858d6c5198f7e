"""Serving operators at the edges of what their arguments may be."""

from __future__ import annotations

import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

import torque_mlx_b200 as tq  # noqa: E402
from torque_mlx_b200 import _lib  # noqa: E402

from test_gpu_paged import batch_args, make_cache, tables  # noqa: E402


def test_rows_repeated_by_a_stride_of_zero():
    cache, table = make_cache(81, [40, 7, 90], [1, 1, 1], page=16, kv_heads=2, d=64)
    args = dict(lengths=torch.tensor([40, 7, 90], dtype=torch.int32, device="cuda"), block_table=table)
    one = torch.randn(1, 8 * 64, device="cuda").to(torch.bfloat16)
    cos, sin = tables(100, 64)
    many = one.expand(3, -1)
    assert torch.equal(cache.append(many, cos, sin, **args), cache.append(many.contiguous(), cos, sin, **args))
    q = one[:, :256].reshape(1, 4, 64).expand(3, -1, -1)
    assert torch.equal(cache.attend(q, **args), cache.attend(q.contiguous(), **args))
    step = torch.randn(8 * 64 + 2 * 8, device="cuda").to(torch.bfloat16).as_strided((3, 8 * 64), (8, 1))  # rows that overlap
    assert torch.equal(cache.append(step, cos, sin, **args), cache.append(step.contiguous(), cos, sin, **args))


@pytest.mark.parametrize("mode", ["plain", "f32", "rms", "silu"])
def test_product_of_rows_repeated_by_a_stride_of_zero(mode):
    w = tq.W4Weight.quantize(torch.randn(96, 256, device="cuda"), group_size=64)
    x = torch.randn(1, 512 if mode == "silu" else 256, device="cuda")
    x = (x if mode == "f32" else x.to(torch.bfloat16)).expand(5, -1)
    norm = torch.ones(256, device="cuda", dtype=torch.bfloat16) if mode == "rms" else None
    assert torch.equal(tq.gemv_w4(w, x, mode=mode, norm_weight=norm), tq.gemv_w4(w, x.contiguous(), mode=mode, norm_weight=norm))


def test_verification_of_rows_repeated_by_a_stride_of_zero():
    g = torch.Generator(device="cuda").manual_seed(4)
    p = torch.softmax(torch.randn(1, 1, 100, generator=g, device="cuda"), -1)
    noise = torch.empty(1, 100, device="cuda").exponential_(generator=g)
    tokens = torch.randint(0, 100, (3, 2), generator=g, device="cuda").to(torch.int32)
    uniform = torch.rand(3, 2, generator=g, device="cuda")
    got = tq.verify_drafts(p.expand(3, 3, 100), p.expand(3, 2, 100), tokens, uniform, noise.expand(3, 100))
    want = tq.verify_drafts(p.expand(3, 3, 100).contiguous(), p.expand(3, 2, 100).contiguous(), tokens, uniform,
                            noise.expand(3, 100).contiguous())
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_out_of_memory_has_its_own_type():
    """As torch's own allocations have it, so that a server may catch it and shed load."""
    cache = tq.PagedKV8Cache(1, kv_heads=64, head_dim=256, page_size=128)
    pages = torch.zeros(1 << 20, dtype=torch.int32, device="cuda")  # 4 TB of values
    with pytest.raises(torch.OutOfMemoryError):
        cache.dequantize(pages, dtype=torch.float16)


def test_truth_values_that_have_none():
    cache, table = make_cache(82, [4], [1], page=16, kv_heads=1, d=64)
    args = dict(lengths=torch.tensor([4], dtype=torch.int32, device="cuda"), block_table=table)
    both = torch.tensor([True, False])  # has no truth value
    q = torch.zeros(1, 1, 64, device="cuda", dtype=torch.bfloat16)
    for kw in (dict(lengths_counted=both), dict(return_lse=both)):
        with pytest.raises(ValueError):
            cache.attend(q, **kw, **args)
    with pytest.raises(ValueError):
        cache.append(torch.zeros(1, 3 * 64, device="cuda"), interleaved=both, **args)


def test_row_counts_announced_beyond_the_rows():
    """The largest number that the C ABI takes for `max_new_tokens`: no more rows are there than there are."""
    from test_paged_abi_cpu import _Batch
    lens, new = [20, 70], [3, 1]
    lib = _lib.load()
    x = torch.randn(4, 8 * 64, device="cuda").to(torch.bfloat16)
    results = []
    for most in (3, 2 ** 31 - 1):
        cache, table = make_cache(83, lens, new, page=16, kv_heads=2, d=64)
        a = batch_args(lens, new)
        b = _Batch(table.data_ptr(), a["lengths"].data_ptr(), a["token_starts"].data_ptr(), table.stride(0), 4,
                   table.shape[1], 2, most)
        q = torch.empty(4, 4, 64, device="cuda", dtype=torch.bfloat16)
        out = torch.empty_like(q)
        need = ctypes.c_size_t()
        stream = torch.cuda.current_stream().cuda_stream
        assert lib.tq_paged_append(cache._at, ctypes.byref(b), x.data_ptr(), _lib.TQ_BF16, x.stride(0), 4, None, None, 0, 0, 1,
                                   q.data_ptr(), stream) == 0
        assert lib.tq_paged_attend_workspace_size(cache._at, 4, most, ctypes.byref(need)) == 0
        ws = torch.empty(need.value, dtype=torch.uint8, device="cuda")
        assert lib.tq_paged_attend(cache._at, ctypes.byref(b), q.data_ptr(), _lib.TQ_BF16, q.stride(0), 4, 0, 0.125, 128,
                                   out.data_ptr(), None, ws.data_ptr(), need.value, stream) == 0
        results.append((q, out, cache.key_pages, cache.value_pages, cache.key_scales))
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("rows", [2, 60])
def test_a_page_of_negative_key_scale_is_not_attended(rows):
    """As the header has it, in either kernel: what such a page holds is seen no more than a missing page."""
    lens, new = [100], [rows]
    cache, table = make_cache(84, lens, new, page=16, kv_heads=1, d=64)
    cache.key_scales[table[0, 2].long()] *= -1
    q = torch.randn(rows, 2, 64, device="cuda").to(torch.bfloat16)
    got = cache.attend(q, block_table=table, **batch_args(lens, new))
    table[0, 2] = -1
    assert torch.equal(got, cache.attend(q, block_table=table, **batch_args(lens, new)))
