"""Waits of the many-row attention that run out: the rows are NaN, the caller can read it, and the GPU goes on."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

from torque_mlx_b200 import _lib  # noqa: E402

from test_gpu_paged import batch_args, check_attend, make_cache  # noqa: E402

TRIES = 20000


@pytest.fixture
def limit():
    lib = _lib.load()
    yield lib.tq_paged_attend_wait_limit
    lib.tq_paged_attend_wait_limit(TRIES)


@pytest.mark.parametrize("lens,new,hq,hkv,d", [
    ([20 + i % 100 for i in range(200)], [45] * 200, 2, 2, 64),   # more units than CTAs, none divided
    ([30, 0, 200] * 30, [60, 0, 41] * 30, 4, 4, 256),
    ([6000, 3000], [300, 50], 4, 2, 128),                   # few units in many parts
    ([9000], [70], 1, 1, 256),
])
def test_a_wait_that_gives_up_is_told(limit, lens, new, hq, hkv, d):
    cache, table = make_cache(61, lens, new, page=64, kv_heads=hkv, d=d)
    q = torch.randn(sum(new), hq, d, device="cuda").to(torch.bfloat16)
    most = max(a + b for a, b in zip(lens, new))
    args = dict(block_table=table, max_context=most, return_lse=True, **batch_args(lens, new))
    before = cache.attend_gave_up()
    want, want_lse = cache.attend(q, **args)
    assert cache.attend_gave_up() == before
    limit(0)
    out, lse = cache.attend(q, out=torch.ones_like(q), **args)
    count = cache.attend_gave_up()
    assert count > before
    assert bool(out.isnan().all()) and bool(lse.isnan().all())
    limit(TRIES)
    out, lse = cache.attend(q, out=torch.ones_like(q), **args)
    assert cache.attend_gave_up() == count
    assert torch.equal(out, want) and torch.equal(lse, want_lse)


def test_a_wait_that_gives_up_leaves_other_calls_alone(limit):
    """The stream, the workspace and the tensor memory serve the next calls, on either kernel."""
    lens, new = [700, 90], [50, 64]
    cache, table = make_cache(62, lens, new, page=32, kv_heads=2, d=128)
    q = torch.randn(sum(new), 4, 128, device="cuda").to(torch.float16)
    for _ in range(3):
        limit(0)
        cache.attend(q, block_table=table, **batch_args(lens, new))
        limit(TRIES)
        out, lse = cache.attend(q, block_table=table, return_lse=True, **batch_args(lens, new))
        check_attend(cache, table, q, lens, new, out, lse)
        few = cache.attend(q[:2], block_table=table, **batch_args(lens, [1, 1]))
        check_attend(cache, table, q[:2], lens, [1, 1], few)


def test_the_count_is_not_read_in_a_capture():
    cache, _ = make_cache(63, [10], [1], page=16, kv_heads=1, d=64)
    graph = torch.cuda.CUDAGraph()
    x = torch.zeros(4, device="cuda")
    with torch.cuda.graph(graph):
        x += 1
        with pytest.raises(ValueError):
            cache.attend_gave_up()
    graph.replay()
    assert float(x.sum()) == 4
