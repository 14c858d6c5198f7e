"""Serving operators called by two threads on one stream: a call's launches belong together."""

from __future__ import annotations

import sys
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu

import torque_mlx_b200 as tq  # noqa: E402

from test_gpu_paged import batch_args, make_cache  # noqa: E402


def attention(seed, length, rows):
    """A call whose few units fall to many thread blocks, so that a second launch joins their parts."""
    cache, table = make_cache(seed, [length], [rows], page=64, kv_heads=2, d=64)
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randn(rows, 4, 64, generator=g, device="cuda").to(torch.bfloat16)
    args = batch_args([length], [rows])
    return lambda: cache.attend(q, block_table=table, **args)


def product(seed, tokens):
    """A product whose columns are split, so that a second launch adds the parts."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = tq.W4Weight.quantize(torch.randn(256, 8192, generator=g, device="cuda"), group_size=64)
    x = torch.randn(tokens, 8192, generator=g, device="cuda").to(torch.bfloat16)
    return lambda: tq.gemv_w4(w, x)


PAIRS = [
    (lambda: attention(1, 4000, 2), lambda: attention(2, 4000, 2)),
    (lambda: attention(3, 5000, 60), lambda: attention(4, 5000, 60)),
    (lambda: product(5, 32), lambda: product(6, 32)),
    (lambda: attention(7, 4000, 1), lambda: product(8, 32)),
]


@pytest.mark.parametrize("pair", range(len(PAIRS)))
def test_two_threads_on_one_stream(pair):
    calls = [make() for make in PAIRS[pair]]
    want = [call() for call in calls]
    torch.cuda.synchronize()
    stream = torch.cuda.current_stream()
    start, off, errors = threading.Barrier(2), [0, 0], []

    def work(i):
        try:
            with torch.cuda.stream(stream):
                start.wait()
                for _ in range(40):
                    got = [calls[i]() for _ in range(50)]
                    off[i] += sum(not torch.equal(x, want[i]) for x in got)
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    old = sys.getswitchinterval()
    sys.setswitchinterval(1e-5)
    try:
        threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    finally:
        sys.setswitchinterval(old)
    assert not errors and off == [0, 0], (off, errors)
