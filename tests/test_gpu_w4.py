"""Products with 4-bit weights (tq_gemv_w4) and their preparation against 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

import torque_mlx_b200 as tq  # noqa: E402
from torque_mlx_b200 import ops  # noqa: E402

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def make_weight(n, k, group, seed=0):
    """(W4Weight, dense fp64 weight) of random codes and scales."""
    g = torch.Generator(device="cuda").manual_seed(seed + n + k)
    packed = torch.randint(0, 256, (n, (k + 1) // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = (0.01 * (0.25 + torch.rand((n, -(-k // group)), generator=g, device="cuda"))).to(torch.bfloat16)
    codes = torch.stack([packed & 15, packed >> 4], -1).flatten(-2)[:, :k].double() - 8
    dense = codes * scales.double().repeat_interleave(group, 1)[:, :k]
    return tq.W4Weight.from_packed(packed, scales, k=k, group_size=group), dense


def check(got, x, dense, dtype, residual=None, extra=0.0):
    want = x.double() @ dense.T
    size = x.double().abs() @ dense.T.abs()
    if residual is not None:
        want = want + residual.double()
        size = size + residual.double().abs()
    # fp32 sums: a chain of k/16 products of sixteen, the warps' and the slabs' parts, one rounding each
    k = dense.shape[1]
    tol = (k / 16 + 64) * 2.0 ** -23 * size + extra * size
    tol = tol + 1.01 * UNIT[dtype] * (want.abs() + tol) + 1e-30
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25
    err = (got.double() - want).abs()
    assert got.dtype == dtype and got.shape == want.shape
    assert bool((err <= tol).all()), float((err / tol).max())


SHAPES = [(16, 64), (1, 32), (17, 96), (1000, 256), (4096, 2048), (2048, 6144), (77, 1000), (300, 8192), (33, 7), (640, 130),
          (5000, 1040)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,k", SHAPES)
def test_gemv_matches_fp64(n, k, group, dtype):
    w, dense = make_weight(n, k, group)
    g = torch.Generator(device="cuda").manual_seed(3)
    for tokens in (1, 5, 8, 9, 16, 31, 32, 45):
        x = torch.randn(tokens, k, generator=g, device="cuda").to(dtype)
        r = torch.randn(tokens, n, generator=g, device="cuda").to(dtype) if tokens % 2 else None
        check(tq.gemv_w4(w, x, residual=r), x, dense, dtype, r)


@pytest.mark.parametrize("tokens", [1, 4, 13])
@pytest.mark.parametrize("n,k", [(2048, 2048), (2048, 6144), (100, 320)])
def test_input_modes(n, k, tokens):
    w, dense = make_weight(n, k, 64)
    g = torch.Generator(device="cuda").manual_seed(5)
    bf = torch.bfloat16
    x = torch.randn(tokens, k, generator=g, device="cuda")
    check(tq.gemv_w4(w, x, mode="f32"), x.to(bf), dense, bf)
    gu = torch.randn(tokens, 2 * k, generator=g, device="cuda").to(bf)
    r = torch.randn(tokens, n, generator=g, device="cuda").to(bf)
    check(tq.gemv_w4(w, gu, mode="silu", residual=r), ops.silu_mul(gu), dense, bf, r)
    xb = (3 * x).to(bf)
    nw = (torch.rand(k, generator=g, device="cuda") + 0.5).to(bf)
    got = tq.gemv_w4(w, xb, mode="rms", norm_weight=nw, eps=1e-6)
    # an element on the edge of a bf16 rounding may fall to the other side: a hundredth of them by 2^-7
    check(got, ops.rmsnorm(xb, nw, 1e-6), dense, bf, extra=0.01 * 2.0 ** -7)


def test_one_vector_matches_one_row():
    w, _ = make_weight(50, 256, 32)
    x = torch.randn(256, device="cuda").to(torch.bfloat16)
    a = tq.gemv_w4(w, x)
    assert a.shape == (50,) and torch.equal(a, tq.gemv_w4(w, x[None])[0])


@pytest.mark.parametrize("n,k", [(640, 2048), (64, 8192)])
def test_tokens_do_not_see_each_other(n, k):
    """A token's result is its own: rows far apart in size, infinities and NaN beside it, and any position in the batch."""
    w, dense = make_weight(n, k, 128)
    x = torch.randn(12, k, device="cuda")
    x[1] *= 2.0 ** 90
    x[2] *= 2.0 ** -90
    x[3, 5] = math.inf
    x[4, 7] = math.nan
    x[5] = 0
    x[6, 3] = 2.0 ** 30
    x = x.to(torch.bfloat16)
    y = tq.gemv_w4(w, x)
    fine = [0, 1, 2, 5, 6, 7, 8, 9, 10, 11]
    check(y[fine], x[fine], dense, torch.bfloat16)
    assert bool(y[4].isnan().all())
    zero = dense[:, 5] == 0
    assert bool(torch.isinf(y[3])[~zero].all()) and bool(y[3].isnan()[zero].all())


def test_strides_alignment_other_stream_graph_and_repeats():
    w, dense = make_weight(1500, 1024, 64)
    wide = torch.randn(6, 3, 1024, device="cuda").to(torch.bfloat16)
    x = wide[:, 1]
    want = tq.gemv_w4(w, x.contiguous())
    check(want, x, dense, torch.bfloat16)
    assert torch.equal(tq.gemv_w4(w, x), want)
    odd = torch.empty(6 * 1024 + 1, dtype=x.dtype, device="cuda")[1:].view(6, 1024).copy_(x)
    assert torch.equal(tq.gemv_w4(w, odd), want)
    odd_rows = torch.empty(6, 1027, dtype=x.dtype, device="cuda")[:, :1024].copy_(x)
    assert torch.equal(tq.gemv_w4(w, odd_rows), want)
    assert torch.equal(tq.gemv_w4(w, x.T.contiguous().T), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(tq.gemv_w4(w, x), want)
    side.synchronize()
    static, out = x.contiguous(), torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tq.gemv_w4(w, static, out=out)
    static.copy_(x.flip(0))
    graph.replay()
    assert torch.equal(out, want.flip(0))
    for _ in range(4):
        assert torch.equal(tq.gemv_w4(w, x), want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,k,group", [(5, 256, 128), (33, 200, 32), (64, 65, 64), (16, 1, 32)])
def test_quantize_and_dequantize(n, k, group, dtype):
    g = torch.Generator(device="cuda").manual_seed(k)
    dense = torch.randn(n, k, generator=g, device="cuda") * 0.02
    dense[0] = 0
    dense = dense.to(dtype)
    packed, scales = tq.quantize_w4(dense, group_size=group)
    codes = torch.stack([packed & 15, packed >> 4], -1).flatten(-2)
    if k % 2:
        codes = codes[:, :k]
    padded = torch.zeros(n, -(-k // group) * group, device="cuda", dtype=torch.float64)
    padded[:, :k] = dense.double()
    top = padded.reshape(n, -1, group).abs().amax(-1)
    want_scale = (top / 7).clamp(min=2.0 ** -100)
    assert bool(((scales.double() - want_scale).abs() <= 2.0 ** -8 * want_scale).all())
    step = scales.double().repeat_interleave(group, 1)[:, :k]
    off = ((codes.double() - 8) * step - dense.double()).abs()
    # half a step, and what the rounded scale takes from the largest (code 7 stands for 7 scales)
    assert bool((off <= 0.5 * step + 7 * step * 2.0 ** -8 + 1e-30).all())
    w = tq.W4Weight.from_packed(packed, scales, k=k, group_size=group)
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        assert torch.equal(w.dequantize(dt), ((codes.float() - 8) * step.float()).to(dt))
    both = tq.W4Weight.quantize(dense, group_size=group)
    assert torch.equal(both.codes, w.codes) and torch.equal(both.scales, w.scales)


def test_weight_past_32_bit_offsets():
    """More than 2^32 codes; the last rows of the product are checked."""
    n, k, group = 540000, 8192, 128
    g = torch.Generator(device="cuda").manual_seed(1)
    packed = torch.zeros((n, k // 2), dtype=torch.uint8, device="cuda")
    packed[-64:] = torch.randint(0, 256, (64, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = torch.full((n, k // group), 0.01, device="cuda", dtype=torch.bfloat16)
    w = tq.W4Weight.from_packed(packed, scales, k=k, group_size=group)
    x = torch.randn(2, k, generator=g, device="cuda").to(torch.bfloat16)
    y = tq.gemv_w4(w, x)
    tail = packed[-64:]
    dense = (torch.stack([tail & 15, tail >> 4], -1).flatten(-2).double() - 8) * float(scales[0, 0])
    check(y[:, -64:], x, dense, torch.bfloat16)


def test_refusals():
    w, _ = make_weight(32, 128, 64)
    x = torch.randn(2, 128, device="cuda").to(torch.bfloat16)
    tq.gemv_w4(w, x)
    for args, kw in (((x[:, :64],), {}), ((x.float(),), {}), ((x.cpu(),), {}), ((x,), dict(mode="f32")),
                     ((x,), dict(mode="nope")), ((x,), dict(mode="rms")), ((x,), dict(mode="silu")),
                     ((x.half(),), dict(mode="rms", norm_weight=x[0])), ((x,), dict(residual=x)),
                     ((x,), dict(residual=torch.zeros(2, 32, device="cuda"))),
                     ((x,), dict(out=torch.zeros(2, 32, device="cuda"))), ((x[None],), {})):
        with pytest.raises(ValueError):
            tq.gemv_w4(w, *args, **kw)
    packed = torch.zeros(4, 64, dtype=torch.uint8, device="cuda")
    scales = torch.ones(4, 2, dtype=torch.bfloat16, device="cuda")
    tq.W4Weight.from_packed(packed, scales, k=128, group_size=64)
    for p, s, k, gs in ((packed, scales, 128, 48), (packed, scales, 130, 64), (packed, scales[:, :1], 128, 64),
                        (packed.int(), scales, 128, 64), (packed, scales.float(), 128, 64), (packed[:0], scales[:0], 128, 64)):
        with pytest.raises(ValueError):
            tq.W4Weight.from_packed(p, s, k=k, group_size=gs)
    with pytest.raises(ValueError):
        tq.quantize_w4(torch.zeros(4, 4, dtype=torch.int32, device="cuda"))
    assert tq.gemv_w4(w, x[:0]).shape == (0, 32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_infinite_weights_keep_their_sign(dtype):
    w = torch.randn(3, 64, device="cuda").to(dtype)
    w[0, 3], w[0, 4], w[0, 5] = math.inf, -math.inf, math.nan
    packed, scales = tq.quantize_w4(w, group_size=32)
    codes = torch.stack([packed & 15, packed >> 4], -1).flatten(-2)
    assert codes[0, 3:6].tolist() == [15, 0, 8]
    assert bool(torch.isfinite(scales).all())
    assert torch.equal(packed[1:], tq.quantize_w4(w[1:], group_size=32)[0])


def test_weight_of_buffers_that_do_not_hold_it():
    """The product reads by the sizes alone, so buffers of other sizes are refused where the weight is made."""
    w, _ = make_weight(64, 256, 64)
    again = tq.W4Weight(w.codes, w.scales, 64, 256, 64)
    x = torch.randn(2, 256, device="cuda").to(torch.bfloat16)
    assert torch.equal(tq.gemv_w4(again, x), tq.gemv_w4(w, x))
    for codes, scales, n, k, group in ((w.codes[:-1024], w.scales, 64, 256, 64), (w.codes, w.scales[:-16], 64, 256, 64),
                                       (w.codes, w.scales, 4096, 256, 64), (w.codes, w.scales, 64, 2560, 64),
                                       (w.codes, w.scales, 64, 256, 32), (w.codes.cpu(), w.scales, 64, 256, 64),
                                       (w.codes, w.scales.cpu(), 64, 256, 64), (w.codes, w.scales.float(), 64, 256, 64),
                                       (torch.zeros(w.codes.numel() + 1, dtype=torch.uint8, device="cuda")[1:], w.scales, 64, 256, 64),
                                       (w.codes, w.scales, 64, 256, 48), (w.codes, w.scales, 0, 256, 64)):
        with pytest.raises(ValueError):
            tq.W4Weight(codes, scales, n, k, group)
