"""Attention over the 8-bit paged cache where weights and page scales are far apart in size."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from test_gpu_paged import UNIT, batch_args, dense, make_cache  # noqa: E402


def check(cache, table, q, lens, new, out, lse, scale):
    """Rows of every sequence against 64 bits.

    A weight is rounded to fp16 against a reference that lies 7 to 15 powers of two under the row's largest exponent
    (score and v's page scale): 2^-11 of the weight, or 2^-25 over 2^7 of the largest one where it is smaller.  A score is
    a sum of d products in fp32, and its error enters the weight as a factor."""
    d = q.shape[2]
    G = q.shape[1] // cache.kv_heads
    row = 0
    for s, (length, n) in enumerate(zip(lens, new)):
        for h in range(cache.kv_heads):
            k, v = dense(cache, table, s, h, length + n)
            pages = table[s].long()[torch.arange(length + n, device="cuda") // cache.page_size]
            vs = torch.where(pages >= 0, cache.value_scales[pages.clamp(min=0), h], 0).double()
            here = pages >= 0
            for t in range(n):
                seen = here & (torch.arange(length + n, device="cuda") <= length + t)
                qq = q[row + t, h * G:(h + 1) * G].double()
                x = qq @ k[seen].T * scale
                wide = float((qq.abs() @ k[seen].abs().T).max()) * abs(scale)
                p = torch.softmax(x, -1)
                want = p @ v[seen]
                size = p @ v[seen].abs()
                most = (p * vs[seen]).amax(-1, keepdim=True)
                tol = (2.0 ** -11 + 2.0 ** -15 + 2.0 ** -20 * (1 + wide)) * size + 2.0 ** -32 * 128 * int(seen.sum()) * most
                tol = tol + 1.01 * UNIT[q.dtype] * (want.abs() + tol)
                if q.dtype == torch.float16:
                    tol = tol + 2.0 ** -25
                err = (out[row + t, h * G:(h + 1) * G].double() - want).abs()
                assert bool((err <= tol).all()), (s, h, t, float((err / tol).max()))
                if lse is not None:
                    wl = torch.logsumexp(x, -1)
                    assert bool(((lse[row + t, h * G:(h + 1) * G].double() - wl).abs() <= 2e-5 * (1 + wl.abs())
                                 + 2.0 ** -20 * wide).all())
        row += n


def aimed(seed, lens, new, *, page, kv_heads, d):
    """A cache whose keys are zero but for dimension 0, so that scores are what is written there; the query's row is
    (1, 0, ...), and a score is code * key scale * the softmax scale."""
    cache, table = make_cache(seed, lens, new, page=page, kv_heads=kv_heads, d=d)
    cache.key_pages.fill_(128)
    cache.key_scales.fill_(0.01)
    return cache, table


def row_of_ones(rows, heads, d, dtype):
    q = torch.zeros(rows, heads, d, device="cuda", dtype=dtype)
    q[..., 0] = 1
    return q


@pytest.mark.parametrize("drop", [18, 22, 26])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("length,rows", [(250, 1), (200, 50)])
def test_many_small_weights_beside_large_ones(length, rows, d, drop):
    """A few tokens hold nearly all the weight and values of zero: the output is what 200 weights 2^-drop of theirs bring."""
    lens, new = [length], [rows]
    cache, table = aimed(71, lens, new, page=16, kv_heads=1, d=d)
    cache.value_scales.fill_(0.02)
    g = torch.Generator(device="cuda").manual_seed(drop)
    cache.key_pages[..., 0] = 128 + torch.randint(-3, 4, cache.key_pages.shape[:3], generator=g, device="cuda").to(torch.uint8)
    cache.value_pages.clamp_(min=200)
    for token in (0, 16, 32, 48):  # one for each of four neighbouring chunks of sixteen
        at = table[0, token // 16].long()
        cache.key_pages[at, :, token % 16, 0] = 255
        cache.value_pages[at, :, token % 16] = 128
    scale = drop * math.log(2) / (127 * 0.01)
    q = row_of_ones(rows, 1, d, torch.bfloat16)
    out, lse = cache.attend(q, block_table=table, scale=scale, return_lse=True, **batch_args(lens, new))
    check(cache, table, q, lens, new, out, lse, scale)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("rows", [6, 60])
def test_pages_of_much_larger_scale_that_causality_hides(rows, d):
    """Rows of a first page of ordinary values; what follows, unseen by them, is 2^50 as large."""
    lens, new = [13], [rows]
    cache, table = make_cache(72, lens, new, page=16, kv_heads=1, d=d)
    later = table[0, 1:]
    cache.value_scales[later[later >= 0].long()] *= 2.0 ** 50
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn(rows, 2, d, generator=g, device="cuda").to(torch.bfloat16)
    out, lse = cache.attend(q, block_table=table, return_lse=True, **batch_args(lens, new))
    check(cache, table, q, lens, new, out, lse, d ** -0.5)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("rows", [2, 60])
@pytest.mark.parametrize("small,large,gap", [(-10, 40, 60), (-110, 10, 30), (-100, 100, 150), (-100, 100, 215), (0, 90, 3),
                                             (-60, 60, 140), (-119, -119, 2), (110, 110, 2)])
@pytest.mark.parametrize("order", [0, 1])
def test_scores_that_prefer_the_smaller_values(order, small, large, gap, rows, d):
    """Pages of value scales 2^small and 2^large by turns, those of the small ones with scores `gap` powers of two above."""
    lens, new = [300], [rows]
    cache, table = aimed(73, lens, new, page=16, kv_heads=1, d=d)
    ids = table[0, :-(-(lens[0] + rows) // 16)].long()
    g = torch.Generator(device="cuda").manual_seed(2)
    for i, id_ in enumerate(ids.tolist()):
        low = (i // 3) % 2 == order
        cache.value_scales[id_] = 2.0 ** (small if low else large)
        cache.key_pages[id_, :, :, 0] = (128 + torch.randint(-2, 3, (1, 16), generator=g, device="cuda")
                                         + (100 if low else 0)).to(torch.uint8)
    scale = gap * math.log(2) / (100 * 0.01)
    q = row_of_ones(rows, 1, d, torch.bfloat16)
    args = dict(block_table=table, scale=scale, **batch_args(lens, new))
    out, lse = cache.attend(q, return_lse=True, **args)
    check(cache, table, q, lens, new, out, lse, scale)
    out = cache.attend(q, max_context=1 << 20, **args)
    check(cache, table, q, lens, new, out, None, scale)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_small_weights_of_values_without_scale(d):
    """Pages of zeros (scale 0 or the smallest) hold nearly all the weight: the sum counts them."""
    lens, new = [150], [60]
    cache, table = aimed(74, lens, new, page=16, kv_heads=1, d=d)
    for i, id_ in enumerate(table[0, :14].tolist()):
        if i % 3 < 2:
            cache.key_pages[id_, :, :, 0] = 228
            cache.value_pages[id_] = 128
            cache.value_scales[id_] = (0.0, 2.0 ** -120)[i % 3]
    scale = 9 * math.log(2)
    q = row_of_ones(60, 1, d, torch.float16)
    out, lse = cache.attend(q, block_table=table, scale=scale, return_lse=True, **batch_args(lens, new))
    check(cache, table, q, lens, new, out, lse, scale)
