"""What rejected drafts leave behind in the 8-bit paged cache, and what drafting does to the text."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

import torque_mlx_b200 as tq  # noqa: E402
from torque_mlx_b200 import serving  # noqa: E402
from torque_mlx_b200.decoder import DecoderConfig  # noqa: E402

from test_gpu_serving import TINY, plain_logits  # noqa: E402


@pytest.mark.parametrize("loud", [0.5, 3.0, 1000.0])
@pytest.mark.parametrize("held,drafts", [(5, 3), (16, 3), (30, 5)])
def test_held_tokens_stay_within_half_of_the_raised_scale(held, drafts, loud):
    """Drafts up to a thousand times as large, appended behind tokens and dropped: each value held moves by half of its
    page's new scale at most, only where the scale rose, and what is appended next is as near as ever."""
    P, d = 16, 64
    cache = tq.PagedKV8Cache(4, kv_heads=2, head_dim=d, page_size=P)
    table = torch.tensor([[2, 0, 3]], dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(held)
    lengths = torch.zeros(1, dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, held], dtype=torch.int32, device="cuda")
    cache.append(torch.randn(held, 6 * d, generator=g, device="cuda"), lengths=lengths, block_table=table,
                 token_starts=starts)
    lengths += held
    before = [x.double() for x in cache.dequantize(table[0], dtype=torch.float32)]
    was = [cache.key_scales.clone(), cache.value_scales.clone()]
    rejected = loud * torch.randn(drafts, 6 * d, generator=g, device="cuda")
    cache.append(rejected, lengths=lengths, block_table=table,
                 token_starts=torch.tensor([0, drafts], dtype=torch.int32, device="cuda"))
    after = [x.double() for x in cache.dequantize(table[0], dtype=torch.float32)]
    for old, new, scales, now in zip(before, after, was, (cache.key_scales, cache.value_scales)):
        for page in range(-(-held // P)):
            n = min(P, held - page * P)
            id_ = int(table[0, page])
            for h in range(2):
                off = float((old[page, h, :n] - new[page, h, :n]).abs().max())
                if float(now[id_, h]) == float(scales[id_, h]):
                    assert off == 0
                else:
                    assert float(now[id_, h]) > float(scales[id_, h])
                    assert off <= 0.5001 * float(now[id_, h])
    # the drafts are dropped (the lengths stay) and written over
    x = torch.randn(1, 6 * d, generator=g, device="cuda")
    cache.append(x, lengths=lengths, block_table=table)
    k, _ = cache.dequantize(table[0], dtype=torch.float32)
    id_ = int(table[0, held // P])
    got = k[held // P, :, held % P].double()
    step = cache.key_scales[id_].double()[:, None]
    assert bool(((got - x[:, 2 * d:4 * d].double().reshape(2, d)).abs() <= 0.5001 * step).all())
    if held % P == 0:  # a page that held nothing before starts anew
        assert float(step.max()) < 5 / 127


def test_right_drafts_save_steps_and_wrong_ones_are_turned_down(monkeypatch):
    """Drafts that are the text which comes without them, and drafts that are not it.  What the cache holds and the order
    of sums depend on the tokens of a step, so a near tie may fall either way: every emitted token's logit is within twice
    the noise of the forward pass (3% of the largest, as its own test has it) of the best one's in 64 bits."""
    cfg = DecoderConfig(**TINY, seed=7)
    prompts = [[3, 1, 4, 1, 5, 9, 2, 6] * 6, [11, 12, 13] * 5, [42]]
    m = serving.PagedDecoder(cfg, batch=3, max_tokens=256)
    plain, steps = m.generate(prompts, 24, drafts=0, temperature=0)
    assert steps == 24
    proposed = []

    def known(shift):
        def draft(tokens, most, match=2):
            p, t = next((p, t) for p, t in zip(prompts, plain) if tokens[:len(p)] == p)
            at = len(tokens) - len(p)
            proposed.append([(x + shift) % cfg.vocab for x in t[at:at + max(most, 0)]])
            return proposed[-1]
        return draft

    def check(texts):
        for p, t in zip(prompts, texts):
            logits = plain_logits(m, torch.tensor(p + t, device="cuda"))[len(p) - 1:-1]
            best = logits.amax(1) - logits[torch.arange(24), torch.tensor(t, device="cuda")]
            assert len(t) == 24 and float(best.max()) <= 2 * 0.03 * float(logits.abs().max())

    check(plain)
    for shift in (0, 1):
        proposed.clear()
        monkeypatch.setattr(serving, "lookup_drafts", known(shift))
        text, taken = m.generate(prompts, 24, drafts=4, temperature=0)
        check(text)
        assert sum(map(len, proposed)) > 24
        assert taken < 24 if shift == 0 else taken <= 24
