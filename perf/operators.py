"""Measured cases of the serving operators around the 8-bit paged cache.

Four operators that one speculative serving step runs in turn:

* ``append``: rotary positions on the q and k heads of ragged qkv rows, and the
  new keys and values quantised into an 8-bit paged cache (one scale for each
  page and head);
* ``attend``: causal grouped-query attention of ragged query tokens over that
  cache;
* ``gemv``: the product of a few tokens with a 4-bit weight with group scales;
* ``verify``: acceptance of drafted tokens by given random numbers, and the
  next token from the residual distribution.

``run`` computes an operator in elementary torch operations, or, where ``own``
is true, by the framework's public entry points.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
INV_127 = 1 / 127  # a page's scale is its largest magnitude times this, in 32 bits
SCALE_FLOOR = 2.0 ** -120  # smallest page scale: a page of zeros keeps a positive one


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _paged(op, name, seqs, tokens, ragged, ctx_lo, ctx_hi, q_heads, kv_heads, head_dim, page, dtype, interleaved=True):
    return {"op": op, "name": name, "seqs": seqs, "tokens": tokens, "ragged": ragged, "ctx_lo": ctx_lo,
            "ctx_hi": ctx_hi, "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": page,
            "dtype": dtype, "interleaved": interleaved}


def listed():
    return [
        # one new token for each of a batch of 64 sequences: the append of every generated token
        _paged("append", "append_decode", 64, 1, False, 1024, 4096, 32, 8, 128, 64, "bf16"),
        # prompts of uneven length entering together, two kv heads of 256, split-half rotary pairs
        _paged("append", "append_prompts", 7, 1531, True, 0, 700, 16, 2, 256, 32, "f16", False),
        # the smallest call: one sequence, a head for each query head
        _paged("attend", "attend_one", 1, 1, False, 511, 511, 8, 8, 128, 64, "bf16"),
        # a single 131072-token context, the longest one
        _paged("attend", "attend_long", 1, 1, False, 131071, 131071, 16, 2, 256, 64, "bf16"),
        # batched decode, 64 sequences of 16K to 32K tokens: the largest call
        _paged("attend", "attend_batch", 64, 1, False, 16384, 32767, 32, 8, 128, 64, "bf16"),
        # drafted tokens of uneven number over short and middling contexts, small pages
        _paged("attend", "attend_drafts", 16, 5, True, 1, 4001, 8, 2, 64, 16, "f16"),
        # a prompt's chunk over its own prefix
        _paged("attend", "attend_prompt", 1, 972, False, 4099, 4099, 16, 8, 128, 64, "bf16"),
        # a fused qkv projection for one token
        {"op": "gemv", "name": "gemv_qkv", "tokens": 1, "n": 4096, "k": 2048, "group": 128, "dtype": "bf16"},
        # the gate and up projections for the drafted tokens of three sequences
        {"op": "gemv", "name": "gemv_drafts", "tokens": 13, "n": 12288, "k": 2048, "group": 32, "dtype": "f16"},
        # the output head over the whole vocabulary
        {"op": "gemv", "name": "gemv_head", "tokens": 4, "n": 151936, "k": 2048, "group": 64, "dtype": "bf16"},
        # four drafted tokens of one sequence
        {"op": "verify", "name": "verify_one", "seqs": 1, "drafts": 4, "ragged": False, "vocab": 151936,
         "dtype": "f32", "greedy": False},
        # a batch with up to eight drafted tokens each
        {"op": "verify", "name": "verify_batch", "seqs": 64, "drafts": 8, "ragged": True, "vocab": 151936,
         "dtype": "f32", "greedy": False},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "gemv", "verify"])
    if op in ("append", "attend"):
        q_heads, kv_heads, d = rng.choice([(32, 8, 128), (16, 8, 128), (16, 2, 256), (8, 8, 128), (8, 2, 64),
                                           (4, 2, 64), (16, 1, 128), (12, 4, 64)])
        page = rng.choice([16, 32, 64, 128])
        dtype = rng.choice(["bf16", "f16"])
        if op == "append":
            tokens = _log_int(rng, 1, 1600)
            seqs = _log_int(rng, 1, max(1, min(96, 8192 // tokens)))
            hi = _log_int(rng, 1, 4096)
        elif rng.random() < 0.3:  # a prompt's chunk
            tokens = _log_int(rng, 17, 1024)
            seqs = _log_int(rng, 1, max(1, min(16, 1024 // tokens)))
            hi = _log_int(rng, 1, 6000)
        else:
            tokens = rng.choice([1, 1, _log_int(rng, 2, 16)])
            seqs = _log_int(rng, 1, 64)
            hi = _log_int(rng, 1, max(1, min(131072, (1 << 20) * 8 * 128 // (seqs * kv_heads * d))))
        lo = rng.choice([0, hi // 2, hi])
        return {k: v for k, v in _paged(op, "", seqs, tokens, rng.random() < 0.5, lo, hi, q_heads, kv_heads, d, page,
                                        dtype, rng.random() < 0.5).items() if k != "name"}
    if op == "gemv":
        k = 16 * _log_int(rng, 4, 512)
        return {"op": op, "tokens": _log_int(rng, 1, 32), "n": _log_int(rng, 64, min(151936, (1 << 29) // k)), "k": k,
                "group": rng.choice([32, 64, 128]), "dtype": rng.choice(["bf16", "f16"])}
    return {"op": op, "seqs": _log_int(rng, 1, 64), "drafts": rng.randint(1, 10), "ragged": rng.random() < 0.5,
            "vocab": _log_int(rng, 1000, 151936), "dtype": rng.choice(["f32", "f32", "bf16", "f16"]),
            "greedy": rng.random() < 0.25}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _ragged(rng, seqs, most, ragged):
    """How many tokens each sequence brings: ``most``, or 0 to ``most`` with one sequence at least at ``most``."""
    if not ragged:
        return [most] * seqs
    n = [rng.randint(0, most) for _ in range(seqs)]
    n[rng.randrange(seqs)] = most
    return n


def _lengths(c):
    """New tokens and tokens held of each sequence; they belong to the case, so that every seed has the same shapes."""
    rng = random.Random(1000003 * c["seqs"] + 101 * c["tokens"] + c["ctx_hi"])
    new = _ragged(rng, c["seqs"], c["tokens"], c["ragged"])
    return new, [rng.randint(c["ctx_lo"], c["ctx_hi"]) for _ in range(c["seqs"])]


def _paged_inputs(c, seed):
    """Cache, block table and rows of a paged case: what a serving loop holds before the call."""
    g = _gen(seed)
    S, P, Hq, Hkv, d = c["seqs"], c["page"], c["q_heads"], c["kv_heads"], c["head_dim"]
    dt = DTYPES[c["dtype"]]
    new, lens = _lengths(c)
    pages = [-(-(a + b) // P) for a, b in zip(lens, new)]
    total, widest = max(1, sum(pages)), max(1, max(pages))
    order = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
    seq_of = torch.repeat_interleave(torch.arange(S, device=DEV), torch.tensor(pages, device=DEV))
    firsts = [0]
    for n in pages:
        firsts.append(firsts[-1] + n)
    idx_of = torch.arange(sum(pages), device=DEV) - torch.tensor(firsts[:-1], device=DEV)[seq_of]
    table = torch.zeros((S, widest), dtype=torch.int32, device=DEV)
    table[seq_of, idx_of] = order[: sum(pages)]
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    # pages of codes as a quantised normal variable gives them: 127 stands for about four deviations
    kinds = min(total, max(1, (1 << 25) // (Hkv * P * d)))

    def codes():
        base = (torch.randn((kinds, Hkv, P, d), generator=g, device=DEV) * (127 / 4)).round_().clamp_(-127, 127)
        base = (base + 128).to(torch.uint8)
        return base[torch.randint(0, kinds, (total,), generator=g, device=DEV)]

    def scales():
        return (4 / 127) * (0.75 + 0.5 * torch.rand((total, Hkv), generator=g, device=DEV))

    s = {"case": c, "op": c["op"], "new": new, "lens": lens, "k_pages": codes(), "v_pages": codes(),
         "k_scales": scales(), "v_scales": scales(), "table": table,
         "starts": torch.tensor(starts, dtype=torch.int32, device=DEV),
         "lengths": torch.tensor(lens, dtype=torch.int32, device=DEV), "most": max(new), "longest": max(
             a + b for a, b in zip(lens, new)), "dtype": dt}
    N = sum(new)
    if c["op"] == "append":
        x = torch.randn((N, Hq + 2 * Hkv, d), generator=g, device=DEV)
        loud = torch.rand((Hq + 2 * Hkv, d), generator=g, device=DEV) < 0.01  # a few channels of large values
        s["qkv"] = torch.where(loud, x * 8, x).reshape(N, -1).to(dt)
        inv = 1.0 / (1e6 ** (torch.arange(0, d, 2, device=DEV, dtype=torch.float32) / d))
        angle = torch.arange(s["longest"] + 1, device=DEV, dtype=torch.float32)[:, None] * inv[None]
        s["cos"], s["sin"] = angle.cos(), angle.sin()
        first = [n // P for n in lens]
        count = [max(0, t - f) if n else 0 for t, f, n in zip(pages, first, new)]
        s["touched_seq"] = torch.repeat_interleave(torch.arange(S, device=DEV), torch.tensor(count, device=DEV))
        at = [0]
        for n in count:
            at.append(at[-1] + n)
        s["touched_idx"] = (torch.arange(at[-1], device=DEV) - torch.tensor(at[:-1], device=DEV)[s["touched_seq"]]
                            + torch.tensor(first, device=DEV)[s["touched_seq"]])
        s["touched"] = table[s["touched_seq"], s["touched_idx"]].contiguous()
    else:
        s["q"] = (1.5 * torch.randn((N, Hq, d), generator=g, device=DEV)).to(dt)
    s["row_seq"] = torch.repeat_interleave(torch.arange(S, device=DEV), torch.tensor(new, device=DEV))
    s["row_t"] = torch.arange(N, device=DEV) - s["starts"].long()[s["row_seq"]]
    return s


def _gemv_inputs(c, seed):
    g = _gen(seed)
    n, k, gs = c["n"], c["k"], c["group"]
    dt = DTYPES[c["dtype"]]
    groups = -(-k // gs)
    packed = torch.randint(0, 256, (n, k // 2), generator=g, device=DEV, dtype=torch.uint8)
    scales = ((0.02 * 3 / 7) * (0.5 + torch.rand((n, groups), generator=g, device=DEV))).to(torch.bfloat16)
    x = torch.randn((c["tokens"], k), generator=g, device=DEV).to(dt)
    return {"case": c, "op": "gemv", "packed": packed, "scales": scales, "x": x, "dtype": dt}


def _verify_inputs(c, seed):
    g = _gen(seed)
    B, T, V = c["seqs"], c["drafts"], c["vocab"]
    dt = DTYPES[c["dtype"]]
    target = torch.randn((B, T + 1, V), generator=g, device=DEV) * 3
    draft = target[:, :T] + 0.7 * torch.randn((B, T, V), generator=g, device=DEV)
    race = torch.empty((B, T, V), device=DEV).exponential_(generator=g)
    q = torch.softmax(draft, -1)
    tokens = (q / race).argmax(-1).to(torch.int32)
    del race, draft
    counts = torch.tensor(_ragged(random.Random(seed), B, T, c["ragged"]), dtype=torch.int32, device=DEV)
    return {"case": c, "op": "verify", "target": torch.softmax(target, -1).to(dt),
            "draft": None if c["greedy"] else q.to(dt), "tokens": tokens, "counts": counts,
            "uniform": torch.rand((B, T), generator=g, device=DEV),
            "noise": torch.empty((B, V), device=DEV).exponential_(generator=g)}


def _inputs(c, seed):
    return {"gemv": _gemv_inputs, "verify": _verify_inputs}.get(c["op"], _paged_inputs)(c, seed)


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        import torque_mlx_b200 as tq
        s["tq"] = tq
        if s["op"] == "gemv":
            s["weight"] = tq.W4Weight.from_packed(s["packed"], s["scales"], k=case["k"], group_size=case["group"])
        elif s["op"] != "verify":
            s["cache"] = tq.PagedKV8Cache.from_pages(s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"])
    return s


# ---------------------------------------------------------------------------
# plain forms: 32 bits, rounded once at the end
# ---------------------------------------------------------------------------
def _rope(x, cos, sin, interleaved):
    """Rotates the pairs of x [N, heads, d] by the angles of cos, sin [N, d/2]."""
    cos, sin = cos[:, None], sin[:, None]
    if interleaved:
        a, b = x[..., ::2], x[..., 1::2]
        return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


def _quantise_into(pages, scales, x, page_of, slot, touched, old):
    """Writes the rows x [N, Hkv, d] into their pages and slots; pages with ``old`` tokens keep at least their scale."""
    amax = torch.zeros_like(scales).index_reduce_(0, page_of, x.abs().amax(-1), "amax")
    before = scales[touched]
    after = (amax[touched] * INV_127).clamp(min=SCALE_FLOOR)
    after = torch.where((old > 0)[:, None], torch.maximum(after, before), after)
    ratio = (before / after)[:, :, None, None]
    kept = pages[touched]
    requantised = ((kept.float() - 128) * ratio).round().clamp(-127, 127) + 128
    live = torch.arange(pages.shape[2], device=DEV)[None, None, :, None] < old[:, None, None, None]
    pages[touched] = torch.where(live, requantised, kept.float()).to(torch.uint8)
    scales[touched] = after
    code = (x / scales[page_of][:, :, None]).round().clamp(-127, 127) + 128
    pages[page_of, :, slot] = code.to(torch.uint8)


def _plain_append(s):
    c = s["case"]
    Hq, Hkv, d, P = c["q_heads"], c["kv_heads"], c["head_dim"], c["page"]
    x = s["qkv"].float().reshape(-1, Hq + 2 * Hkv, d)
    pos = s["lengths"].long()[s["row_seq"]] + s["row_t"]
    cos, sin = s["cos"][pos], s["sin"][pos]
    q = _rope(x[:, :Hq], cos, sin, c["interleaved"]).to(s["dtype"])
    k = _rope(x[:, Hq:Hq + Hkv], cos, sin, c["interleaved"])
    touched = s["touched"].long()
    page_of, slot = s["table"][s["row_seq"], pos // P].long(), pos % P
    old = (s["lengths"].long()[s["touched_seq"]] - s["touched_idx"] * P).clamp(0, P)
    _quantise_into(s["k_pages"], s["k_scales"], k, page_of, slot, touched, old)
    _quantise_into(s["v_pages"], s["v_scales"], x[:, Hq + Hkv:], page_of, slot, touched, old)
    values = [((s[n + "_pages"][touched].float() - 128) * s[n + "_scales"][touched][:, :, None, None]).to(s["dtype"])
              for n in ("k", "v")]
    return {"q": q, "k": values[0], "v": values[1]}


def _dense(pages, scales, table):
    """The values [S, Hkv, T, d] of the pages of a block table, in 32 bits."""
    S, n = table.shape
    _, H, P, d = pages.shape
    at = table.long()
    x = pages[at].permute(0, 2, 1, 3, 4).float().sub_(128)
    return x.mul_(scales[at].permute(0, 2, 1)[..., None, None]).reshape(S, H, n * P, d)


def _plain_attend(s):
    c = s["case"]
    S, T, Hq, Hkv, d = c["seqs"], s["most"], c["q_heads"], c["kv_heads"], c["head_dim"]
    G = Hq // Hkv
    q = torch.zeros((S, T, Hkv, G, d), device=DEV)
    q[s["row_seq"], s["row_t"]] = s["q"].float().reshape(-1, Hkv, G, d)
    q = q.permute(0, 2, 1, 3, 4).reshape(S, Hkv, T * G, d)
    k = _dense(s["k_pages"], s["k_scales"], s["table"])
    score = (q @ k.transpose(-1, -2)).mul_(d ** -0.5).reshape(S, Hkv, T, G, -1)
    del k
    last = s["lengths"].long()[:, None] + torch.arange(T, device=DEV)  # the row's own position
    hidden = torch.arange(score.shape[-1], device=DEV) > last[:, :, None]
    score.masked_fill_(hidden[:, None, :, None], -math.inf)
    p = score.sub_(score.amax(-1, keepdim=True)).exp_()
    p = p.div_(p.sum(-1, keepdim=True)).reshape(S, Hkv, T * G, -1)
    out = (p @ _dense(s["v_pages"], s["v_scales"], s["table"])).reshape(S, Hkv, T, G, d)
    out = out.permute(0, 2, 1, 3, 4).reshape(S, T, Hq, d)
    return out[s["row_seq"], s["row_t"]].to(s["dtype"])


def _plain_gemv(s):
    c = s["case"]
    code = torch.stack([s["packed"] & 15, s["packed"] >> 4], -1).flatten(-2).float() - 8
    scale = s["scales"].float().repeat_interleave(c["group"], 1)[:, :c["k"]]
    return (s["x"].float() @ (code * scale).T).to(s["dtype"])


def _plain_verify(s):
    c = s["case"]
    B, T, V = c["seqs"], c["drafts"], c["vocab"]
    tokens, counts = s["tokens"].long(), s["counts"].long()
    p = s["target"][:, :T].gather(2, tokens[..., None])[..., 0].float()
    q = torch.ones_like(p) if s["draft"] is None else s["draft"].gather(2, tokens[..., None])[..., 0].float()
    step = torch.arange(T, device=DEV)
    good = (s["uniform"] * q < p) & (step < counts[:, None])
    accepted = good.long().cumprod(1).sum(1)
    row = torch.arange(B, device=DEV)
    final = s["target"][row, accepted].float()
    at = accepted.clamp(max=T - 1)
    if s["draft"] is None:
        taken = torch.zeros_like(final).scatter_(1, tokens[row, at][:, None], 1.0) * final
    else:
        taken = s["draft"][row, at].float()
    residual = (final - taken).clamp(min=0)
    whole = (accepted == counts) | (residual.amax(1) <= 0)  # every draft taken, or nothing left over
    weight = torch.where(whole[:, None], final, residual)
    best = torch.where(weight > 0, weight / s["noise"], -1.0)
    top = best.amax(1, keepdim=True)
    index = torch.where(best == top, torch.arange(V, device=DEV), V).amin(1)
    out = torch.cat([tokens, torch.full((B, 1), -1, device=DEV)], 1)
    out = torch.where(torch.arange(T + 1, device=DEV) < accepted[:, None], out, -1)
    out[row, accepted] = index
    return {"accepted": accepted.to(torch.int32), "tokens": out.to(torch.int32)}


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    s, op = state, state["op"]
    if not own:
        return {"append": _plain_append, "attend": _plain_attend, "gemv": _plain_gemv, "verify": _plain_verify}[op](s)
    if op == "append":
        c = s["case"]
        q = s["cache"].append(s["qkv"], s["cos"], s["sin"], lengths=s["lengths"], block_table=s["table"],
                              token_starts=s["starts"], max_new_tokens=s["most"], interleaved=c["interleaved"])
        k, v = s["cache"].dequantize(s["touched"], dtype=s["dtype"])
        return {"q": q, "k": k, "v": v}
    if op == "attend":
        return s["cache"].attend(s["q"], lengths=s["lengths"], block_table=s["table"], token_starts=s["starts"],
                                 max_new_tokens=s["most"], max_context=s["longest"])
    if op == "gemv":
        return s["tq"].gemv_w4(s["weight"], s["x"])
    accepted, tokens = s["tq"].verify_drafts(s["target"], s["draft"], s["tokens"], s["uniform"], s["noise"],
                                             draft_counts=s["counts"])
    return {"accepted": accepted, "tokens": tokens}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    c = case
    if c["op"] == "gemv":
        M, n, k = c["tokens"], c["n"], c["k"]
        return {"bytes": n * k / 2 + 2 * n * -(-k // c["group"]) + 2 * M * (n + k), "flops": 2 * M * n * k}
    if c["op"] == "verify":  # two rows at least decide the next token: the target's and the random numbers
        size = 4 if c["dtype"] == "f32" else 2
        return {"bytes": c["seqs"] * c["vocab"] * (size + 4), "flops": c["seqs"] * c["vocab"]}
    d, Hq, Hkv, P = c["head_dim"], c["q_heads"], c["kv_heads"], c["page"]
    new, lens = _lengths(c)
    N = sum(new)
    if c["op"] == "append":
        # rows read and q written; codes of the new tokens written; the touched pages' values, which come back with
        # the call's outputs, written from their codes
        pages = sum(-(-(a + n) // P) - a // P for a, n in zip(lens, new) if n)
        return {"bytes": N * (2 * (Hq + 2 * Hkv) * d + 2 * Hq * d + 2 * Hkv * d) + pages * 2 * Hkv * P * d * 3,
                "flops": N * 3 * (Hq + Hkv) * d}
    # each token's codes read once, q read and the output written; a product for each visible pair, twice
    pairs = sum(n * a + n * (n + 1) // 2 for a, n in zip(lens, new))
    held = sum(a + n for a, n in zip(lens, new) if n)
    return {"bytes": held * Hkv * 2 * d + 4 * N * Hq * d, "flops": 4 * pairs * Hq * d}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_append(s):
    c = s["case"]
    Hq, Hkv, d, P = c["q_heads"], c["kv_heads"], c["head_dim"], c["page"]
    dev = s["qkv"].device
    x = s["qkv"].double().reshape(-1, Hq + 2 * Hkv, d)
    N = x.shape[0]
    kv = {"k": torch.empty((N, Hkv, d), dtype=torch.float64, device=dev), "v": x[:, Hq + Hkv:]}
    q = torch.empty((N, Hq, d), dtype=torch.float64, device=dev)
    half = d // 2
    first = torch.arange(0, d, 2, device=dev) if c["interleaved"] else torch.arange(half, device=dev)
    second = first + 1 if c["interleaved"] else first + half
    row = 0
    out = {"k": [], "v": []}
    for i, (length, n) in enumerate(zip(s["lens"], s["new"])):
        if n == 0:
            continue
        cos = s["cos"][length:length + n].double()[:, None]
        sin = s["sin"][length:length + n].double()[:, None]
        r = slice(row, row + n)
        for src, dst in ((x[r, :Hq], q[r]), (x[r, Hq:Hq + Hkv], kv["k"][r])):
            dst[..., first] = src[..., first] * cos - src[..., second] * sin
            dst[..., second] = src[..., first] * sin + src[..., second] * cos
        for name in ("k", "v"):
            lo = length // P
            hi = (length + n - 1) // P
            for j in range(lo, hi + 1):
                page = int(s["table"][i, j])
                had = max(0, length - j * P)
                a, b = max(length, j * P), min(length + n, (j + 1) * P)
                rows = kv[name][row + a - length:row + b - length].transpose(0, 1)  # [Hkv, tokens, d]
                codes = s[name + "_pages"][page].double() - 128
                was = s[name + "_scales"][page].double()
                scale = (rows.abs().amax((1, 2)) / 127).clamp(min=SCALE_FLOOR)
                if had:
                    scale = torch.maximum(scale, was)
                    codes[:, :had] = (codes[:, :had] * (was / scale)[:, None, None]).round()
                codes[:, a - j * P:b - j * P] = (rows / scale[:, None, None]).round().clamp(-127, 127)
                out[name].append(codes * scale[:, None, None])
        row += n
    return {"q": q, "k": torch.stack(out["k"]), "v": torch.stack(out["v"])}


def _exact_attend(s):
    c = s["case"]
    Hq, Hkv, d, P = c["q_heads"], c["kv_heads"], c["head_dim"], c["page"]
    G = Hq // Hkv
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    row = 0
    for i, (length, n) in enumerate(zip(s["lens"], s["new"])):
        if n == 0:
            continue
        total = length + n
        pages = s["table"][i, :-(-total // P)].long()
        for h in range(Hkv):
            k, v = (((s[name + "_pages"][pages, h].double() - 128) * s[name + "_scales"][pages, h].double()[:, None, None])
                    .reshape(-1, d)[:total] for name in ("k", "v"))
            q = s["q"][row:row + n, h * G:(h + 1) * G].double()  # [n, G, d]
            score = torch.einsum("ngd,td->ngt", q, k) / math.sqrt(d)
            seen = torch.arange(total, device=q.device)[None] <= length + torch.arange(n, device=q.device)[:, None]
            score = torch.where(seen[:, None], score, torch.full_like(score, -math.inf))
            out[row:row + n, h * G:(h + 1) * G] = torch.einsum("ngt,td->ngd", torch.softmax(score, -1), v)
        row += n
    return out


def exact(case, seed):
    c = case
    if c["op"] == "verify":  # whole numbers: nothing is computed that a definition in 64 bits would sharpen
        return None
    s = _inputs(c, seed)
    if c["op"] == "append":
        return _exact_append(s)
    if c["op"] == "attend":
        return _exact_attend(s)
    k, gs = c["k"], c["group"]
    y = torch.zeros((c["tokens"], c["n"]), dtype=torch.float64, device=DEV)
    for lo in range(0, k, gs):  # group by group
        hi = min(k, lo + gs)
        byte = s["packed"][:, lo // 2:hi // 2]
        x = s["x"][:, lo:hi].double()
        part = x[:, ::2] @ ((byte & 15).double() - 8).T + x[:, 1::2] @ ((byte >> 4).double() - 8).T
        y += part * s["scales"][:, lo // gs].double()
    return y
