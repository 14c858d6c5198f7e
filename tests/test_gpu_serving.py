"""The speculative serving example: the paged operators, the 4-bit products and
the verification of drafts run together as one decoder."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

from torque_mlx_b200.decoder import DecoderConfig  # noqa: E402
from torque_mlx_b200.serving import PagedDecoder, lookup_drafts  # noqa: E402

TINY = dict(num_layers=2, hidden=256, q_heads=4, kv_heads=2, head_dim=64, ffn=512, vocab=1000)


def plain_logits(m: PagedDecoder, tokens: torch.Tensor) -> torch.Tensor:
    """Logits of one sequence in fp64 on the dequantized weights, with an unquantized cache."""
    cfg = m.cfg
    H, Hkv, d, T = cfg.q_heads, cfg.kv_heads, cfg.head_dim, tokens.numel()

    def rms(x):
        return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + cfg.rms_eps)

    def rope(x):
        c, s = m.cos[:T].double()[:, None], m.sin[:T].double()[:, None]
        a, b = x[..., ::2], x[..., 1::2]
        return torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)

    x = m.embed[tokens].double()
    mask = torch.ones(T, T, dtype=torch.bool, device=x.device).tril()
    for lay in m.layers:
        w = {k: v.dequantize(torch.float32).double() for k, v in lay.items() if k.startswith("w")}
        q, k, v = (rms(x) @ w["wqkv"].T).reshape(T, H + 2 * Hkv, d).split([H, Hkv, Hkv], 1)
        q, k = rope(q), rope(k).repeat_interleave(H // Hkv, 1)
        v = v.repeat_interleave(H // Hkv, 1)
        s = torch.einsum("qhd,khd->hqk", q, k) / d ** 0.5
        p = torch.softmax(s.masked_fill(~mask, -torch.inf), -1)
        x = x + torch.einsum("hqk,khd->qhd", p, v).reshape(T, H * d) @ w["wo"].T
        gate, up = (rms(x) @ w["w_gate_up"].T).chunk(2, -1)
        x = x + (torch.nn.functional.silu(gate) * up) @ w["w_down"].T
    return rms(x) @ m.lm_head.dequantize(torch.float32).double().T


def test_forward_matches_plain_decoder():
    """Prompt in one go, in chunks and token by token: the logits are those of the plain decoder to the noise of bf16
    activations (as the packed decoder's test has it: 3% of the largest) and of the 8-bit cache."""
    cfg = DecoderConfig(**TINY, seed=5)
    m = PagedDecoder(cfg, batch=2, max_tokens=160, page_size=16)
    g = torch.Generator().manual_seed(1)
    tokens = torch.randint(0, cfg.vocab, (2, 90), generator=g).cuda()
    want = [plain_logits(m, t) for t in tokens]
    scale = float(max(w.abs().max() for w in want))
    for cuts in ([0, 90], [0, 70, 71, 74, 90], [0, *range(60, 91)]):
        m.lengths.zero_()
        for lo, hi in zip(cuts, cuts[1:]):
            starts = torch.tensor([0, hi - lo, 2 * (hi - lo)], dtype=torch.int32, device="cuda")
            got = m.forward(tokens[:, lo:hi].reshape(-1), starts, hi - lo).reshape(2, hi - lo, -1)
            m.lengths += hi - lo
            for s in range(2):
                assert float((got[s].double() - want[s][lo:hi]).abs().max()) <= 0.03 * scale


def test_drafting_does_not_change_greedy_text():
    """A repetitive prompt, so that drafts are proposed; what is emitted is what one token a step emits."""
    cfg = DecoderConfig(**TINY, seed=7)
    prompts = [[3, 1, 4, 1, 5, 9, 2, 6] * 6, [11, 12, 13] * 5, [42]]
    m = PagedDecoder(cfg, batch=3, max_tokens=256)
    plain, steps = m.generate(prompts, 24, drafts=0, temperature=0)
    drafted, fewer = m.generate(prompts, 24, drafts=4, temperature=0)
    assert steps == 24 and fewer <= steps
    assert drafted == plain


def test_sampling_is_repeatable_and_in_the_vocabulary():
    cfg = DecoderConfig(**TINY, seed=8)
    m = PagedDecoder(cfg, batch=2, max_tokens=128)
    a, _ = m.generate([[1, 2, 3, 1, 2], [9, 9, 9]], 12, drafts=3, temperature=0.8, seed=4)
    b, _ = m.generate([[1, 2, 3, 1, 2], [9, 9, 9]], 12, drafts=3, temperature=0.8, seed=4)
    assert a == b and all(len(t) == 12 and all(0 <= x < cfg.vocab for x in t) for t in a)


def test_refusals():
    m = PagedDecoder(DecoderConfig(**TINY), batch=1, max_tokens=32)
    for bad in ([], [[]], [[1], [2]], [[1] * 30]):
        with pytest.raises(ValueError):
            m.generate(bad, 8)
    with pytest.raises(ValueError):
        PagedDecoder(DecoderConfig(**TINY), batch=0, max_tokens=32)


def test_lookup_drafts():
    assert lookup_drafts([1, 2, 3, 9, 1, 2], 3) == [3, 9, 1]
    assert lookup_drafts([1, 2, 1, 2], 2) == [1, 2]
    assert lookup_drafts([5, 6, 7], 4) == [] and lookup_drafts([1, 2], 4) == [] and lookup_drafts([1, 2, 1, 2], 0) == []
