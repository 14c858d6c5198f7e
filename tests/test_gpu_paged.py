"""8-bit paged cache (tq_paged_append / tq_paged_attend / tq_paged_dequantize)
against the definitions in 64 bits."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

import torque_mlx_b200 as tq  # noqa: E402

FLOOR = 2.0 ** -120
# largest relative error of one rounding: 8 and 11 significant bits (fp32 results are checked by their own terms)
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 0.0}


def make_cache(seed, lens, new, *, page, kv_heads, d, spare=3, v_spread=1.0):
    """A pool of random codes and a shuffled block table that holds lens + new tokens."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    pages = [-(-(a + b) // page) for a, b in zip(lens, new)]
    total = sum(pages) + spare
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lens), max(1, max(pages)) + 1), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(pages):
        table[s, :n] = order[at:at + n]
        at += n
    shape = (total, kv_heads, page, d)
    kp = torch.randint(1, 256, shape, generator=g, device="cuda", dtype=torch.uint8)
    vp = torch.randint(1, 256, shape, generator=g, device="cuda", dtype=torch.uint8)
    ks = 0.01 + 0.02 * torch.rand(shape[:2], generator=g, device="cuda")
    vs = 0.01 + 0.02 * torch.rand(shape[:2], generator=g, device="cuda")
    if v_spread != 1.0:
        vs *= v_spread ** torch.randint(-1, 2, shape[:2], generator=g, device="cuda").float()
    return tq.PagedKV8Cache.from_pages(kp, vp, ks, vs), table


def batch_args(lens, new):
    starts = np.concatenate([[0], np.cumsum(new)])
    return dict(lengths=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                token_starts=torch.tensor(starts, dtype=torch.int32, device="cuda"), max_new_tokens=max(new))


def dense(cache, table, s, h, n):
    """Values [n, d] of the first n tokens of sequence s in fp64, NaN where a page is missing."""
    P = cache.page_size
    ids = table[s, : -(-n // P)].long()
    out = []
    for codes, scales in ((cache.key_pages, cache.key_scales), (cache.value_pages, cache.value_scales)):
        x = (codes[ids.clamp(min=0), h].double() - 128) * scales[ids.clamp(min=0), h].double()[:, None, None]
        x[ids < 0] = math.nan
        out.append(x.reshape(-1, cache.head_dim)[:n])
    return out


def attend64(cache, table, q, lens, new, *, counted=False, scale=None):
    """(out, lse, bound of the rounded weights' effect) in 64 bits."""
    rows, Hq, d = q.shape
    G = Hq // cache.kv_heads
    out = torch.zeros((rows, Hq, d), dtype=torch.float64, device="cuda")
    lse = torch.full((rows, Hq), -math.inf, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(out)
    row = 0
    for s, (length, n) in enumerate(zip(lens, new)):
        base = length - n if counted else length
        total = base + n
        for h in range(cache.kv_heads):
            if n == 0 or total <= 0:
                continue
            k, v = dense(cache, table, s, h, total)
            here = ~k[:, 0].isnan()
            for t in range(n):
                seen = here & (torch.arange(total, device="cuda") <= base + t)
                if not bool(seen.any()):
                    continue
                x = q[row + t, h * G:(h + 1) * G].double() @ k[seen].T * (d ** -0.5 if scale is None else scale)
                p = torch.softmax(x, -1)
                out[row + t, h * G:(h + 1) * G] = p @ v[seen]
                lse[row + t, h * G:(h + 1) * G] = torch.logsumexp(x, -1)
                # weights rounded to fp16 (2^-11 of each) or, 2^-24 of the largest and below, to a subnormal
                size[row + t, h * G:(h + 1) * G] = (2.0 ** -11 + 2.0 ** -15) * (p @ v[seen].abs()) \
                    + 2.0 ** -25 * int(seen.sum()) * float(v[seen].abs().max()) * p.amax(-1, keepdim=True)
        row += n
    return out, lse, size


def check_attend(cache, table, q, lens, new, got, lse=None, **kw):
    want, want_lse, size = attend64(cache, table, q, lens, new, **kw)
    ulp = UNIT[q.dtype]
    tol = size + 1.01 * ulp * (want.abs() + size) + 1e-7
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())
    if lse is not None:
        # fp32 sums of d products and of the tokens' weights
        ok = (lse.double() - want_lse).abs() <= 2e-5 * (1 + want_lse.abs())
        assert bool((ok | (lse.double() == want_lse)).all())


ATTEND = [
    # lens, new, page, q_heads, kv_heads, d
    ([0], [1], 16, 1, 1, 128),
    ([511], [1], 64, 8, 8, 128),
    ([5, 0, 130, 77], [1, 1, 1, 1], 16, 8, 2, 64),
    ([1000, 3, 64, 63], [1, 1, 1, 1], 32, 16, 2, 256),
    ([40, 0, 333, 16, 2047], [3, 5, 0, 1, 4], 64, 8, 2, 128),
    ([9, 800], [16, 7], 128, 16, 4, 64),
    ([33, 0], [4, 2], 16, 32, 2, 256),
    ([100], [97], 32, 8, 4, 128),
    ([15, 0, 700], [65, 31, 8], 16, 4, 2, 256),
    ([3001, 2999, 5000], [1, 1, 1], 64, 16, 1, 128),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,new,page,hq,hkv,d", ATTEND)
def test_attend_matches_fp64(lens, new, page, hq, hkv, d, dtype):
    cache, table = make_cache(len(lens) + d, lens, new, page=page, kv_heads=hkv, d=d)
    g = torch.Generator(device="cuda").manual_seed(1)
    q = (2 * torch.randn(sum(new), hq, d, generator=g, device="cuda")).to(dtype)
    out, lse = cache.attend(q, block_table=table, return_lse=True, **batch_args(lens, new))
    check_attend(cache, table, q, lens, new, out, lse)
    # the launch's size does not change what comes out beyond rounding
    out2 = cache.attend(q, block_table=table, max_context=max(a + b for a, b in zip(lens, new)), **batch_args(lens, new))
    check_attend(cache, table, q, lens, new, out2)


def test_one_row_each_without_starts():
    lens = [7, 0, 250, 64, 65, 1]
    cache, table = make_cache(5, lens, [1] * 6, page=64, kv_heads=2, d=128)
    q = torch.randn(6, 8, 128, device="cuda").to(torch.bfloat16)
    args = batch_args(lens, [1] * 6)
    a = cache.attend(q, lengths=args["lengths"], block_table=table)
    b = cache.attend(q, block_table=table, **args)
    assert torch.equal(a, b)
    check_attend(cache, table, q, lens, [1] * 6, a)


def test_counted_lengths_and_rows_that_see_nothing():
    """With lengths that include the rows, more rows than tokens leave the first rows empty."""
    lens, new = [3, 0, 40, 2], [5, 2, 4, 2]
    cache, table = make_cache(6, lens, new, page=16, kv_heads=2, d=64)
    q = torch.randn(sum(new), 4, 64, device="cuda").to(torch.float16)
    out, lse = cache.attend(q, block_table=table, lengths_counted=True, return_lse=True, **batch_args(lens, new))
    check_attend(cache, table, q, lens, new, out, lse, counted=True)
    assert float(out[:2].abs().max()) == 0 and bool((lse[:2] == -math.inf).all())
    assert float(out[5:7].abs().max()) == 0 and bool((lse[5:7] == -math.inf).all())


@pytest.mark.parametrize("hkv,d", [(1, 128), (2, 64), (1, 256)])
def test_page_scales_far_apart(hkv, d):
    """Page scales 2^40 apart: the weights of v take the scale into their exponent."""
    lens, new = [200, 75], [1, 2]
    cache, table = make_cache(7, lens, new, page=16, kv_heads=hkv, d=d, v_spread=2.0 ** 20)
    q = torch.randn(3, 4 * hkv, d, device="cuda").to(torch.bfloat16)
    out = cache.attend(q, block_table=table, **batch_args(lens, new))
    check_attend(cache, table, q, lens, new, out)


def test_page_of_zeros_and_zero_scale():
    lens, new = [100], [1]
    cache, table = make_cache(8, lens, new, page=16, kv_heads=1, d=64)
    cache.value_pages[table[0, 2].long()] = 128
    cache.value_scales[table[0, 2].long()] = FLOOR
    cache.value_scales[table[0, 3].long()] = 0
    cache.key_scales[table[0, 4].long()] = 0
    q = torch.randn(1, 2, 64, device="cuda").to(torch.float16)
    out, lse = cache.attend(q, block_table=table, return_lse=True, **batch_args(lens, new))
    check_attend(cache, table, q, lens, new, out, lse)


def test_large_and_small_queries_keep_their_size():
    """bf16 rows far outside fp16's range: scores would overflow or vanish in fp16."""
    lens, new = [90, 90, 90], [1, 1, 1]
    cache, table = make_cache(9, lens, new, page=32, kv_heads=1, d=128)
    q = torch.randn(3, 4, 128, device="cuda")
    q[0] *= 2.0 ** 40
    q[1] *= 2.0 ** -40
    q[2, :, ::2] *= 2.0 ** -18  # small beside large elements of one row
    q = q.to(torch.bfloat16)
    for scale in (2.0 ** -43, 2.0 ** 37, None):
        i = {2.0 ** -43: 0, 2.0 ** 37: 1, None: 2}[scale]
        out = cache.attend(q, block_table=table, scale=scale, **batch_args(lens, new))
        want, _, size = attend64(cache, table, q, lens, new, scale=scale)
        tol = size[i] + 2.0 ** -8 * want[i].abs() + 1e-6
        assert bool(((out[i].double() - want[i]).abs() <= tol).all())


def test_nonfinite_query_stays_in_its_row():
    lens, new = [50, 50], [1, 1]
    cache, table = make_cache(10, lens, new, page=16, kv_heads=1, d=64)
    q = torch.randn(2, 2, 64, device="cuda").to(torch.bfloat16)
    clean = cache.attend(q, block_table=table, **batch_args(lens, new))
    q[1, 0, 3] = math.nan
    out = cache.attend(q, block_table=table, **batch_args(lens, new))
    assert bool(out[1, 0].isnan().all())
    assert torch.equal(out[0], clean[0]) and torch.equal(out[1, 1], clean[1, 1])


def test_garbage_behind_the_end_is_not_read():
    """Slots past a sequence's end and pages of others may hold anything, NaN scales among it."""
    lens, new = [37, 5], [1, 1]
    cache, table = make_cache(11, lens, new, page=16, kv_heads=2, d=128)
    q = torch.randn(2, 4, 128, device="cuda").to(torch.bfloat16)
    a = cache.attend(q, block_table=table, **batch_args(lens, new))
    used = table[table >= 0].long()
    other = torch.ones(cache.num_pages, dtype=torch.bool, device="cuda")
    other[used] = False
    for t in (cache.key_scales, cache.value_scales):
        t[other] = math.nan
    for t in (cache.key_pages, cache.value_pages):
        t[table[0, 2].long(), :, 6:] = 255
        t[table[1, 0].long(), :, 6:] = 0
    assert torch.equal(a, cache.attend(q, block_table=table, **batch_args(lens, new)))


def test_missing_pages_are_not_attended():
    lens, new = [100, 40], [1, 2]
    cache, table = make_cache(12, lens, new, page=16, kv_heads=2, d=64)
    table[0, 1] = -1
    table[0, 4] = cache.num_pages  # past the pool
    q = torch.randn(3, 4, 64, device="cuda").to(torch.float16)
    out, lse = cache.attend(q, block_table=table, return_lse=True, **batch_args(lens, new))
    ref = table.clone()
    ref[0, 4] = -1
    check_attend(cache, ref, q, lens, new, out, lse)


def test_strided_rows_other_stream_and_graph():
    lens, new = [70, 300, 0, 129], [2, 1, 3, 1]
    cache, table = make_cache(13, lens, new, page=64, kv_heads=2, d=128)
    wide = torch.randn(sum(new), 3, 8, 128, device="cuda").to(torch.bfloat16)
    q = wide[:, 1]
    args = batch_args(lens, new)
    want = cache.attend(q.contiguous(), block_table=table, **args)
    assert torch.equal(cache.attend(q, block_table=table, **args), want)
    assert torch.equal(cache.attend(q.transpose(0, 1).contiguous().transpose(0, 1), block_table=table, **args), want)
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device="cuda")[1:].view(q.shape).copy_(q)  # not at 16 bytes
    assert torch.equal(cache.attend(odd, block_table=table, **args), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(cache.attend(q, block_table=table, **args), want)
    side.synchronize()
    static = torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.attend(q, block_table=table, out=static, **args)
    args["lengths"][1] = 299  # the captured step follows the device's lengths
    graph.replay()
    check_attend(cache, table, q, [70, 299, 0, 129], new, static)


def test_same_result_every_time():
    lens, new = [5000, 17, 900], [1, 4, 2]
    cache, table = make_cache(14, lens, new, page=64, kv_heads=2, d=128)
    q = torch.randn(sum(new), 8, 128, device="cuda").to(torch.bfloat16)
    first = cache.attend(q, block_table=table, **batch_args(lens, new))
    for _ in range(5):
        assert torch.equal(first, cache.attend(q, block_table=table, **batch_args(lens, new)))


def test_many_short_sequences():
    rng = np.random.default_rng(0)
    lens = rng.integers(0, 40, 300).tolist()
    cache, table = make_cache(15, lens, [1] * 300, page=16, kv_heads=2, d=64)
    q = torch.randn(300, 4, 64, device="cuda").to(torch.float16)
    out = cache.attend(q, lengths=torch.tensor(lens, dtype=torch.int32, device="cuda"), block_table=table)
    check_attend(cache, table, q, lens, [1] * 300, out)


def test_pool_past_32_bit_offsets():
    """A pool of more than 2^32 bytes of keys whose last pages are in use."""
    P, Hkv, d = 128, 8, 256
    n = (1 << 32) // (P * Hkv * d) + 40
    kp = torch.full((n, Hkv, P, d), 128, dtype=torch.uint8, device="cuda")
    vp = torch.full((n, Hkv, P, d), 128, dtype=torch.uint8, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(3)
    kp[-8:] = torch.randint(1, 256, kp[-8:].shape, generator=g, device="cuda", dtype=torch.uint8)
    vp[-8:] = torch.randint(1, 256, vp[-8:].shape, generator=g, device="cuda", dtype=torch.uint8)
    sc = torch.full((n, Hkv), 0.02, device="cuda")
    cache = tq.PagedKV8Cache.from_pages(kp, vp, sc, sc.clone())
    table = torch.arange(n - 1, n - 9, -1, dtype=torch.int32, device="cuda").reshape(1, 8)
    lens, new = [900], [2]
    x = torch.randn(2, (16 + 16) * d, generator=g, device="cuda").to(torch.bfloat16)
    q = cache.append(x, block_table=table, **batch_args(lens, new))
    k, v = cache.dequantize(table[0, 7:], dtype=torch.float32)
    slot = 900 % P
    want = x.float().reshape(2, 32, d)
    for got, lo in ((k, 16), (v, 24)):
        have = got[0, :, slot:slot + 2].transpose(0, 1)
        step = have.abs().amax() / 100
        assert float((have - want[:, lo:lo + 8]).abs().max()) <= float(step)
    out = cache.attend(q, block_table=table, **batch_args(lens, new))
    check_attend(cache, table, q, lens, new, out)


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------
def rope64(x, cos, sin, pos, interleaved):
    """x [rows, heads, d] rotated at positions pos in fp64."""
    c, s = cos[pos].double()[:, None], sin[pos].double()[:, None]
    r = 2 * cos.shape[1]
    out = x.double().clone()
    if interleaved:
        a, b = x[..., 0:r:2].double(), x[..., 1:r:2].double()
        out[..., 0:r:2], out[..., 1:r:2] = a * c - b * s, a * s + b * c
    else:
        a, b = x[..., :r // 2].double(), x[..., r // 2:r].double()
        out[..., :r // 2], out[..., r // 2:r] = a * c - b * s, a * s + b * c
    return out


def tables(n, rotary):
    inv = 1.0 / (1e4 ** (torch.arange(0, rotary, 2, device="cuda", dtype=torch.float32) / rotary))
    angle = torch.arange(n, device="cuda", dtype=torch.float32)[:, None] * inv[None]
    return angle.cos(), angle.sin()


def check_codes(codes, scales, before_codes, before_scales, x, lens, new, table, page):
    """Codes and scales after an append of x [rows, kv_heads, d] (fp64) against the definition."""
    row = 0
    touched = torch.zeros(scales.shape[0], dtype=torch.bool, device="cuda")
    for s, (length, n) in enumerate(zip(lens, new)):
        for j in range(length // page, -(-(length + n) // page) if n else 0):
            id_ = int(table[s, j])
            if id_ < 0 or id_ >= scales.shape[0]:
                continue
            touched[id_] = True
            a, b = max(length, j * page), min(length + n, (j + 1) * page)
            had = max(0, length - j * page)
            rows = x[row + a - length:row + b - length].transpose(0, 1)
            scale = (rows.abs().amax((1, 2)) / 127).clamp(min=FLOOR)
            if had:
                scale = torch.maximum(scale, before_scales[id_].double())
            # a product or two in fp32: 2^-22 of the value
            assert bool(((scales[id_].double() - scale).abs() <= 2.0 ** -22 * scale).all())
            want = torch.zeros(codes.shape[1:], dtype=torch.float64, device="cuda")
            want[:] = before_codes[id_].double() - 128
            want[:, :had] = want[:, :had] * (before_scales[id_].double() / scale)[:, None, None]
            want[:, a - j * page:b - j * page] = rows / scale[:, None, None]
            got = codes[id_].double() - 128
            # nearest whole number of a value that fp32 has to 127 * 2^-21
            assert bool(((got - want.clamp(-127, 127)).abs() <= 0.5 + 1e-4).all())
            assert bool((got[:, b - j * page:] == before_codes[id_].double()[:, b - j * page:] - 128).all())
        row += n
    assert torch.equal(codes[~touched], before_codes[~touched]) and torch.equal(scales[~touched], before_scales[~touched])


APPEND = [
    # lens, new, page, q_heads, kv_heads, d, rotary
    ([0], [1], 16, 1, 1, 128, 128),
    ([63, 64, 65, 0], [1, 1, 1, 1], 64, 8, 2, 64, 64),
    ([15, 0, 100, 31], [3, 40, 0, 1], 16, 4, 2, 128, 64),
    ([7, 300], [130, 1], 128, 16, 2, 256, 256),
    ([0, 12], [5, 64], 32, 0, 3, 64, 16),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("lens,new,page,hq,hkv,d,rotary", APPEND)
def test_append_matches_fp64(lens, new, page, hq, hkv, d, rotary, interleaved, dtype):
    cache, table = make_cache(21, lens, new, page=page, kv_heads=hkv, d=d)
    # some scales below and some above what the new rows need
    cache.key_scales *= 4.0 ** torch.randint(-2, 3, cache.key_scales.shape, device="cuda").float()
    before = [t.clone() for t in (cache.key_pages, cache.key_scales, cache.value_pages, cache.value_scales)]
    rows = sum(new)
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.randn(rows, hq + 2 * hkv, d, generator=g, device="cuda").to(dtype)
    cos, sin = tables(max(a + b for a, b in zip(lens, new)), rotary)
    q = cache.append(x.reshape(rows, -1), cos, sin, block_table=table, interleaved=interleaved, **batch_args(lens, new))
    pos = torch.cat([torch.arange(a, a + b, device="cuda") for a, b in zip(lens, new)])
    ulp = UNIT[dtype]
    want_q = rope64(x[:, :hq], cos, sin, pos, interleaved)
    assert q.shape == (rows, hq, d) and q.dtype == dtype
    big = x.double().abs().amax() if rows else 0
    assert bool(((q.double() - want_q).abs() <= 1.01 * ulp * want_q.abs() + 2.0 ** -22 * big + 2.0 ** -25).all())
    k = rope64(x[:, hq:hq + hkv], cos, sin, pos, interleaved)
    check_codes(cache.key_pages, cache.key_scales, before[0], before[1], k, lens, new, table, page)
    check_codes(cache.value_pages, cache.value_scales, before[2], before[3], x[:, hq + hkv:].double(), lens, new, table,
                page)


def test_append_without_rotation_and_from_a_wider_tensor():
    lens, new = [10, 33], [2, 30]
    cache, table = make_cache(22, lens, new, page=32, kv_heads=2, d=64)
    before = [t.clone() for t in (cache.key_pages, cache.key_scales, cache.value_pages, cache.value_scales)]
    wide = torch.randn(32, 3 * 8 * 64, device="cuda").to(torch.bfloat16)
    x = wide[:, 8 * 64:16 * 64]
    q = cache.append(x, block_table=table, **batch_args(lens, new))
    assert torch.equal(q.reshape(32, -1), x[:, :4 * 64])
    heads = x.reshape(32, 8, 64).double()
    check_codes(cache.key_pages, cache.key_scales, before[0], before[1], heads[:, 4:6], lens, new, table, 32)
    check_codes(cache.value_pages, cache.value_scales, before[2], before[3], heads[:, 6:], lens, new, table, 32)


def test_append_token_by_token_keeps_values_near():
    """Growing magnitudes: every held token is rounded again whenever the scale grows, by half a step of each scale."""
    P, d = 16, 64
    cache = tq.PagedKV8Cache(2, kv_heads=1, head_dim=d, page_size=P)
    table = torch.tensor([[1, 0]], dtype=torch.int32, device="cuda")
    lengths = torch.zeros(1, dtype=torch.int32, device="cuda")
    xs = torch.randn(P, 3 * d, device="cuda") * (1 + torch.arange(P, device="cuda"))[:, None]
    err = torch.zeros(P, dtype=torch.float64, device="cuda")
    scale = 0.0
    for t in range(P):
        cache.append(xs[t:t + 1], lengths=lengths, block_table=table)
        lengths += 1
        now = float(cache.key_scales[1, 0])
        assert now >= scale
        err[:t] += 0.5001 * now * (now != scale)
        err[t] = 0.5001 * now
        scale = now
    k, _ = cache.dequantize(table[0, :1], dtype=torch.float32)
    off = (k[0, 0].double() - xs[:, d:2 * d].double()).abs().amax(1)
    assert bool((off <= err).all())


def test_append_zeros_and_nonfinite():
    cache = tq.PagedKV8Cache(3, kv_heads=1, head_dim=64, page_size=16)
    table = torch.tensor([[0], [1], [2]], dtype=torch.int32, device="cuda")
    lengths = torch.zeros(3, dtype=torch.int32, device="cuda")
    x = torch.zeros(3, 3 * 64, device="cuda")
    x[1, 64:] = torch.randn(128, device="cuda")
    x[1, 70] = math.nan
    x[2, 64:] = 1.0
    x[2, 71] = -math.inf
    cache.append(x, lengths=lengths, block_table=table)
    k, v = cache.dequantize(table[:, 0].contiguous(), dtype=torch.float32)
    assert float(k[0].abs().max()) == 0 and float(cache.key_scales[0, 0]) == FLOOR
    assert float(k[1, 0, 0, 6]) == 0 and float((k[1, 0, 0, 7:] - x[1, 71:128]).abs().max()) < 0.02
    assert float(k[2, 0, 0, 7]) < -3.3e38 and float(k[2, 0, 0, 8]) == 0
    assert bool(torch.isfinite(k).all()) and bool(torch.isfinite(v).all())


def test_append_past_table_pages_and_rotary_rows():
    """A missing page or rotary row drops the row's key and value; nothing else changes."""
    lens, new = [14, 40], [4, 3]
    cache, table = make_cache(23, lens, new, page=16, kv_heads=1, d=64)
    table[0, 1] = -1                       # positions 16, 17 of sequence 0
    before = [t.clone() for t in (cache.key_pages, cache.key_scales, cache.value_pages, cache.value_scales)]
    x = torch.randn(7, 4, 64, device="cuda").to(torch.bfloat16)
    cos, sin = tables(42, 64)              # position 42 of sequence 1 has no row
    q = cache.append(x.reshape(7, -1), cos, sin, block_table=table, **batch_args(lens, new))
    assert bool(q[6].isnan().all()) and not bool(q[:6].isnan().any())
    pos = torch.tensor([14, 15, 16, 17, 40, 41, 41], device="cuda")
    k = rope64(x[:, 2:3], cos, sin, pos, True)
    keep = [0, 1, 4, 5]
    check_codes(cache.key_pages, cache.key_scales, before[0], before[1], k[keep], [14, 40], [2, 2], table, 16)
    check_codes(cache.value_pages, cache.value_scales, before[2], before[3], x[:, 3:].double()[keep], [14, 40], [2, 2],
                table, 16)


def test_dequantize_types_and_unknown_ids():
    cache, _ = make_cache(24, [100], [1], page=16, kv_heads=2, d=128)
    ids = torch.tensor([3, 0, -1, cache.num_pages, 3], dtype=torch.int32, device="cuda")
    for dt in (torch.float32, torch.float16, torch.bfloat16):
        k, v = cache.dequantize(ids, dtype=dt)
        for got, codes, scales in ((k, cache.key_pages, cache.key_scales), (v, cache.value_pages, cache.value_scales)):
            want = ((codes[ids[[0, 1, 4]].long()].float() - 128) * scales[ids[[0, 1, 4]].long()][..., None, None]).to(dt)
            assert torch.equal(got[[0, 1, 4]], want)
            assert bool(got[2:4].isnan().all())
    empty = cache.dequantize(ids[:0])
    assert empty[0].shape == (0, 2, 16, 128)


def test_refusals():
    cache, table = make_cache(25, [10, 20], [1, 1], page=16, kv_heads=2, d=64)
    lengths = torch.tensor([10, 20], dtype=torch.int32, device="cuda")
    q = torch.randn(2, 4, 64, device="cuda").to(torch.bfloat16)
    ok = dict(lengths=lengths, block_table=table)
    cache.attend(q, **ok)
    starts = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    for bad in (dict(lengths=lengths.long()), dict(lengths=lengths.cpu()), dict(block_table=table[:1]),
                dict(block_table=table.long()), dict(token_starts=starts[:2]), dict(token_starts=starts.long()),
                dict(token_starts=starts, max_new_tokens=-1), dict(max_context=-1)):
        with pytest.raises(ValueError):
            cache.attend(q, **{**ok, **bad})
    for bad_q in (q.float(), q[:, :3], q[..., :32], q[:1], q.cpu(), q.reshape(2, -1)):
        with pytest.raises(ValueError):
            cache.attend(bad_q, **ok)
    with pytest.raises(ValueError):
        cache.attend(q, out=torch.empty(2, 4, 64, device="cuda"), **ok)
    x = torch.randn(2, 8 * 64, device="cuda")
    cos, sin = tables(32, 64)
    for args in ((x[:, :100],), (x[:, :3 * 64],), (x, cos), (x, cos, sin[:5]), (x, cos.half(), sin.half()),
                 (x, cos[:, :4].contiguous(), sin[:, :4].contiguous()), (x.int(),), (x.cpu(),)):
        with pytest.raises(ValueError):
            cache.append(*args, **ok)
    with pytest.raises(ValueError):
        cache.dequantize(torch.zeros(2, dtype=torch.int64, device="cuda"))
    for kw in (dict(num_pages=0, kv_heads=1, head_dim=64), dict(num_pages=1, kv_heads=0, head_dim=64),
               dict(num_pages=1, kv_heads=1, head_dim=96), dict(num_pages=1, kv_heads=1, head_dim=64, page_size=48)):
        with pytest.raises(ValueError):
            tq.PagedKV8Cache(**kw)
    with pytest.raises(ValueError):
        tq.PagedKV8Cache.from_pages(cache.key_pages, cache.value_pages[1:], cache.key_scales, cache.value_scales)
    with pytest.raises(ValueError):
        tq.PagedKV8Cache.from_pages(cache.key_pages.float(), cache.value_pages, cache.key_scales, cache.value_scales)


def test_empty_calls():
    cache, table = make_cache(26, [10, 20], [1, 1], page=16, kv_heads=2, d=64)
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert cache.attend(torch.empty(0, 4, 64, device="cuda", dtype=torch.float16), lengths=none,
                        block_table=table[:0]).shape == (0, 4, 64)
    starts = torch.zeros(3, dtype=torch.int32, device="cuda")
    lengths = torch.tensor([10, 20], dtype=torch.int32, device="cuda")
    empty = torch.empty(0, 4, 64, device="cuda", dtype=torch.float16)
    assert cache.attend(empty, lengths=lengths, block_table=table, token_starts=starts).shape == (0, 4, 64)
    assert cache.append(torch.empty(0, 8 * 64, device="cuda"), lengths=lengths, block_table=table,
                        token_starts=starts).shape == (0, 4, 64)


# ---------------------------------------------------------------------------
# many rows for each kv head: tiles of 128
# ---------------------------------------------------------------------------
MANY = [
    # lens, new, page, q_heads, kv_heads, d
    ([0], [129], 64, 2, 2, 128),
    ([0, 5], [33, 1], 16, 1, 1, 64),
    ([4000], [40], 128, 8, 2, 128),
    ([777, 0, 130, 12], [0, 64, 1, 100], 32, 4, 1, 64),
    ([250, 2000], [3, 90], 16, 16, 2, 256),
    ([127, 128, 129], [128, 127, 129], 64, 2, 1, 128),
    ([1], [300], 16, 12, 4, 64),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,new,page,hq,hkv,d", MANY)
def test_many_rows_match_fp64(lens, new, page, hq, hkv, d, dtype):
    cache, table = make_cache(31 + d, lens, new, page=page, kv_heads=hkv, d=d)
    g = torch.Generator(device="cuda").manual_seed(2)
    q = (2 * torch.randn(sum(new), hq, d, generator=g, device="cuda")).to(dtype)
    for most in (None, max(a + b for a, b in zip(lens, new))):
        out, lse = cache.attend(q, block_table=table, return_lse=True, max_context=most, **batch_args(lens, new))
        check_attend(cache, table, q, lens, new, out, lse)


def test_many_rows_counted_and_empty():
    lens, new = [20, 0, 200], [50, 40, 60]
    cache, table = make_cache(41, lens, new, page=16, kv_heads=2, d=64)
    q = torch.randn(sum(new), 4, 64, device="cuda").to(torch.float16)
    out, lse = cache.attend(q, block_table=table, lengths_counted=True, return_lse=True, **batch_args(lens, new))
    check_attend(cache, table, q, lens, new, out, lse, counted=True)
    assert float(out[:30].abs().max()) == 0 and bool((lse[:30] == -math.inf).all())
    assert float(out[50:90].abs().max()) == 0 and bool((lse[50:90] == -math.inf).all())


@pytest.mark.parametrize("d", [64, 128, 256])
def test_many_rows_page_scales_far_apart(d):
    lens, new = [200, 75], [60, 45]
    cache, table = make_cache(42, lens, new, page=16, kv_heads=1, d=d, v_spread=2.0 ** 20)
    cache.value_scales[table[0, 1].long()] = 0
    cache.key_scales[table[0, 2].long()] = 0
    cache.value_pages[table[0, 3].long()] = 128
    cache.value_scales[table[0, 3].long()] = FLOOR
    q = torch.randn(sum(new), 2, d, device="cuda").to(torch.bfloat16)
    out, lse = cache.attend(q, block_table=table, return_lse=True, **batch_args(lens, new))
    check_attend(cache, table, q, lens, new, out, lse)


def test_many_rows_only_zero_values():
    lens, new = [30], [40]
    cache, table = make_cache(43, lens, new, page=16, kv_heads=1, d=64)
    cache.value_pages.fill_(128)
    cache.value_scales.fill_(FLOOR)
    q = torch.randn(40, 2, 64, device="cuda").to(torch.bfloat16)
    out, lse = cache.attend(q, block_table=table, return_lse=True, **batch_args(lens, new))
    assert float(out.abs().max()) == 0
    _, want, _ = attend64(cache, table, q, lens, new)
    assert bool(((lse.double() - want).abs() <= 2e-5 * (1 + want.abs())).all())


def test_many_rows_missing_pages_garbage_and_nonfinite_rows():
    lens, new = [100, 40], [50, 70]
    cache, table = make_cache(44, lens, new, page=16, kv_heads=2, d=64)
    used = table[table >= 0].long()
    other = torch.ones(cache.num_pages, dtype=torch.bool, device="cuda")
    other[used] = False
    cache.key_scales[other] = math.nan
    cache.value_scales[other] = math.nan
    cache.value_pages[table[0, 9].long(), :, 6:] = 255  # past the end
    table[0, 1] = -1
    table[1, 4] = cache.num_pages
    ref = table.clone()
    ref[1, 4] = -1
    q = torch.randn(sum(new), 4, 64, device="cuda").to(torch.float16)
    out, lse = cache.attend(q, block_table=table, return_lse=True, **batch_args(lens, new))
    check_attend(cache, ref, q, lens, new, out, lse)
    bad = q.clone()
    bad[7, 1, 5] = math.nan
    again = cache.attend(bad, block_table=table, **batch_args(lens, new))
    assert bool(again[7, 1].isnan().all())
    keep = torch.ones(out.shape[:2], dtype=torch.bool, device="cuda")
    keep[7, 1] = False
    assert torch.equal(again[keep], out[keep])


def test_many_rows_scales_of_either_sign_stride_stream_graph_and_repeats():
    lens, new = [300, 20], [61, 35]
    cache, table = make_cache(45, lens, new, page=64, kv_heads=2, d=128)
    wide = torch.randn(sum(new), 3, 8, 128, device="cuda").to(torch.bfloat16)
    q = wide[:, 1]
    args = batch_args(lens, new)
    for scale in (0.05, -0.05, 0.0):
        check_attend(cache, table, q, lens, new, cache.attend(q, block_table=table, scale=scale, **args), scale=scale)
    want = cache.attend(q.contiguous(), block_table=table, **args)
    assert torch.equal(cache.attend(q, block_table=table, **args), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            assert torch.equal(cache.attend(q, block_table=table, **args), want)
    side.synchronize()
    static = torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.attend(q, block_table=table, out=static, **args)
    args["lengths"][0] = 299
    graph.replay()
    check_attend(cache, table, q, [299, 20], new, static)


def test_many_rows_large_and_small_queries():
    lens, new = [90], [40]
    cache, table = make_cache(46, lens, new, page=32, kv_heads=1, d=128)
    q = torch.randn(40, 2, 128, device="cuda")
    q[:20] *= 2.0 ** 40
    q[20:] *= 2.0 ** -40
    q = q.to(torch.bfloat16)
    for scale, rows in ((2.0 ** -43, slice(0, 20)), (2.0 ** 37, slice(20, 40))):
        out = cache.attend(q, block_table=table, scale=scale, **batch_args(lens, new))
        want, _, size = attend64(cache, table, q, lens, new, scale=scale)
        tol = size[rows] + 2.0 ** -8 * want[rows].abs() + 1e-6
        assert bool(((out[rows].double() - want[rows]).abs() <= tol).all())
