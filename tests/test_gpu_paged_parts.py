"""Joins of many parts of the attention over the 8-bit paged cache."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from test_gpu_paged import attend64, batch_args  # noqa: E402
from test_gpu_paged_range import aimed, check, row_of_ones  # noqa: E402


@pytest.mark.parametrize("rows", [1, 45])
def test_many_parts_before_the_first_page_and_very_low_scores(rows):
    """A context in over 70 parts, the first 40 or so without pages, and scores of which two to their power vanishes."""
    lens, new = [20000], [rows]
    cache, table = aimed(75, lens, new, page=64, kv_heads=1, d=64)
    cache.value_scales.fill_(0.02)
    g = torch.Generator(device="cuda").manual_seed(3)
    cache.key_pages[..., 0] = 28 + torch.randint(-2, 3, cache.key_pages.shape[:3], generator=g, device="cuda").to(torch.uint8)
    table[0, :200] = -1
    scale = 300 * math.log(2)
    q = row_of_ones(rows, 1, 64, torch.bfloat16)
    out, lse = cache.attend(q, block_table=table, scale=scale, return_lse=True, **batch_args(lens, new))
    check(cache, table, q, lens, new, out, lse, scale)
    want, want_lse, _ = attend64(cache, table, q, lens, new, scale=scale)
    assert float(want.abs().max()) > 0 and float(want_lse.max()) < -126 * math.log(2)
