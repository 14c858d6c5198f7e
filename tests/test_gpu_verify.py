"""Verification of drafted tokens (tq_verify_drafts) against the rule written with numpy."""

from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

import torque_mlx_b200 as tq  # noqa: E402


def rule(target, draft, tokens, uniform, noise, counts):
    """The acceptance and the draw, one sequence at a time, in single fp32 operations."""
    B, rows, V = target.shape
    accepted, out = np.zeros(B, np.int32), np.full((B, rows), -1, np.int32)
    for b in range(B):
        n = min(max(int(counts[b]), 0), rows - 1)
        a = 0
        while a < n:
            x = int(tokens[b, a])
            if not 0 <= x < V:
                break
            q = np.float32(1) if draft is None else draft[b, a, x]
            if not np.float32(uniform[b, a] * q) < target[b, a, x]:
                break
            a += 1
        w = target[b, a]
        if a < n:
            if draft is None:
                rest = w.copy()
                if 0 <= tokens[b, a] < V:
                    rest[tokens[b, a]] = 0
            else:
                rest = np.maximum(w - draft[b, a], np.float32(0))
            if (rest > 0).any():
                w = rest
        with np.errstate(divide="ignore", invalid="ignore"):
            score = np.where(w > 0, w / noise[b], np.float32(-1))
        out[b, :a] = tokens[b, :a]
        out[b, a] = int(np.argmax(score))
        accepted[b] = a
    return accepted, out


def make(seed, B, T, V, dtype=torch.float32, greedy=False, near=0.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    logits = 2 * torch.randn(B, T + 1, V, generator=g, device="cuda")
    target = torch.softmax(logits, -1).to(dtype)
    q = torch.softmax(logits[:, :T] + near * torch.randn(B, T, V, generator=g, device="cuda"), -1)
    tokens = (q / torch.empty_like(q).exponential_(generator=g)).argmax(-1).to(torch.int32)
    draft = None if greedy else q.to(dtype)
    uniform = torch.rand(B, T, generator=g, device="cuda")
    noise = torch.empty(B, V, device="cuda").exponential_(generator=g)
    return target, draft, tokens, uniform, noise


def check(target, draft, tokens, uniform, noise, counts=None):
    accepted, out = tq.verify_drafts(target, draft, tokens, uniform, noise, draft_counts=counts)
    B, rows, _ = target.shape
    n = np.full(B, rows - 1) if counts is None else counts.cpu().numpy()
    want = rule(target.float().cpu().numpy(), None if draft is None else draft.float().cpu().numpy(),
                tokens.cpu().numpy(), uniform.cpu().numpy(), noise.cpu().numpy(), n)
    assert np.array_equal(accepted.cpu().numpy(), want[0])
    assert np.array_equal(out.cpu().numpy(), want[1])
    return accepted, out


@pytest.mark.parametrize("greedy", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,T,V", [(1, 1, 1), (1, 4, 5000), (7, 3, 1000), (3, 8, 32001), (5, 0, 77), (2, 40, 515),
                                   (1, 2, 151936), (33, 5, 64)])
def test_matches_rule(B, T, V, dtype, greedy):
    args = make(B * 100 + T, B, T, V, dtype, greedy)
    check(*args)
    counts = torch.randint(0, T + 1, (B,), device="cuda", dtype=torch.int32)
    check(*args, counts=counts)


def test_counts_outside_their_range_are_taken_to_the_nearest():
    check(*make(1, 4, 3, 100), counts=torch.tensor([-5, 9, 2, 0], dtype=torch.int32, device="cuda"))


def test_all_accepted_and_nothing_left_over():
    target, draft, tokens, uniform, noise = make(2, 4, 3, 300)
    draft = target[:, :3].clone()  # p == q
    uniform[0] = 0.0               # everything accepted
    uniform[1:] = 0.9999
    uniform[2, 1] = 1.5            # rejected although p == q: the residual is zero everywhere
    accepted, _ = check(target, draft, tokens, uniform, noise)
    assert accepted[0] == 3 and accepted[2] == 1


def test_ties_go_to_the_lowest_token():
    V = 4096
    target = torch.full((2, 1, V), 1.0 / V, device="cuda")
    noise = torch.ones(2, V, device="cuda")
    noise[1, :3000] = 2.0
    none = torch.zeros(2, 0, device="cuda")
    _, out = check(target, None, none.int(), none, noise)
    assert out[0, 0] == 0 and out[1, 0] == 3000


def test_zero_and_infinite_scores():
    target = torch.zeros(3, 1, 100, device="cuda")
    target[0, 0, 40:42] = 0.5
    target[1, 0, 7] = 1e-38
    noise = torch.ones(3, 100, device="cuda")
    noise[0, 41] = 0.0   # infinite score
    noise[1, 7] = 1e30   # the score underflows to zero and is still the only positive weight
    none = torch.zeros(3, 0, device="cuda")
    _, out = tq.verify_drafts(target, None, none.int(), none, noise)
    assert out[:, 0].tolist() == [41, 7, 0]


def test_rows_that_are_not_reached_may_hold_anything():
    target, draft, tokens, uniform, noise = make(4, 3, 4, 500)
    counts = torch.tensor([0, 2, 1], dtype=torch.int32, device="cuda")
    want = check(target, draft, tokens, uniform, noise, counts)
    for b, n in enumerate(counts.tolist()):
        target[b, n + 1:] = float("nan")
        draft[b, n:] = float("nan")
        tokens[b, n:] = 10 ** 9
        uniform[b, n:] = float("nan")
    got = tq.verify_drafts(target, draft, tokens, uniform, noise, draft_counts=counts)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_unknown_tokens_are_rejected():
    target, draft, tokens, uniform, noise = make(5, 3, 2, 200)
    uniform[:] = 0
    tokens[0, 0], tokens[1, 1], tokens[2, 0] = -1, 200, 2 ** 31 - 1
    accepted, _ = check(target, draft, tokens, uniform, noise)
    assert accepted.tolist() == [0, 1, 0]
    check(target, None, tokens, uniform, noise)


def test_strided_rows_other_stream_and_graph():
    target, draft, tokens, uniform, noise = make(6, 4, 3, 801)
    want = check(target, draft, tokens, uniform, noise)
    wide = torch.zeros(4, 5, 900, device="cuda")
    wide[:, :4, :801] = target
    wide_q = torch.zeros(3, 4, 1000, device="cuda")
    wide_q[..., 100:901] = draft.transpose(0, 1)
    t, q = wide[:, :4, :801], wide_q[..., 100:901].transpose(0, 1)
    n = torch.zeros(4, 2, 801, device="cuda")
    n[:, 1] = noise
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = tq.verify_drafts(t, q, tokens.T.contiguous().T, uniform, n[:, 1])
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = tq.verify_drafts(target, draft, tokens, uniform, noise)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("greedy", [False, True])
def test_emitted_tokens_follow_the_target(greedy):
    """The first emitted token has the target's distribution, whatever the draft's: chi-square over 7 tokens, 6 degrees
    of freedom, 99.999% quantile 33.1 (the seed is fixed)."""
    B, V = 60000, 7
    g = torch.Generator(device="cuda").manual_seed(11)
    p = torch.softmax(torch.randn(V, generator=g, device="cuda"), -1)
    q = torch.softmax(torch.randn(V, generator=g, device="cuda"), -1)
    tokens = torch.multinomial(q, B, replacement=True, generator=g).to(torch.int32)[:, None]
    if greedy:
        tokens.fill_(2)
    target = p.expand(B, 2, V).contiguous()
    draft = None if greedy else q.expand(B, 1, V).contiguous()
    uniform = torch.rand(B, 1, generator=g, device="cuda")
    noise = torch.empty(B, V, device="cuda").exponential_(generator=g)
    _, out = tq.verify_drafts(target, draft, tokens, uniform, noise)
    seen = torch.bincount(out[:, 0].long(), minlength=V).double()
    want = p.double() * B
    assert float(((seen - want) ** 2 / want).sum()) < 33.1


def test_refusals():
    target, draft, tokens, uniform, noise = make(7, 2, 2, 50)
    counts = torch.ones(2, dtype=torch.int32, device="cuda")
    ok = [target, draft, tokens, uniform, noise]
    tq.verify_drafts(*ok, draft_counts=counts)
    for i, bad in ((0, target[0]), (0, target.cpu()), (0, target.double()), (0, target[:, :0]), (1, draft[:, :1]),
                   (1, draft.half()), (2, tokens.long()), (2, tokens[:, :1]), (3, uniform.double()), (3, uniform[:1]),
                   (4, noise[:, :-1]), (4, noise.half()), (0, target[..., :0])):
        with pytest.raises(ValueError):
            tq.verify_drafts(*(ok[:i] + [bad] + ok[i + 1:]))
    for bad in (counts.long(), counts[:1], counts.cpu()):
        with pytest.raises(ValueError):
            tq.verify_drafts(*ok, draft_counts=bad)
    accepted, out = tq.verify_drafts(*(x[:0] for x in ok))
    assert accepted.shape == (0,) and out.shape == (0, 3)


@pytest.mark.parametrize("B", [1, 14, 15, 400])
def test_most_of_a_cluster_without_columns(B):
    """Vocabularies of fewer columns than a cluster has CTAs times eight: those without a share have nothing to do
    before they hand over their keys, with and without drafts, so they are the first to meet the others' memory."""
    for i, (T, V) in enumerate([(0, 1), (0, 9), (1, 3), (2, 17), (0, 40), (3, 64)]):
        args = make(1000 * B + i, B, T, V)
        for _ in range(5):
            check(*args)
        if T:
            check(*args, counts=torch.zeros(B, dtype=torch.int32, device="cuda"))
