"""Speculative serving of a random-init GQA decoder on 4-bit weights and the
paged 8-bit cache: the model of ``decoder.py`` (pre-norm, RoPE, SwiGLU) for a
batch of sequences that bring uneven numbers of tokens.

One step takes the last token of every sequence and a few drafted ones and runs,
layer by layer,

    gemv_w4 (RMSNorm fused)  ->  PagedKV8Cache.append  ->  PagedKV8Cache.attend
    gemv_w4 (residual)       ->  gemv_w4 (RMSNorm)     ->  gemv_w4 (SwiGLU, residual)

then the output head and ``verify_drafts``.  The lengths advance by what was
accepted, and the next step writes over the rejected rest; a rejected token
that raised its page's scale leaves the page's tokens rounded to that scale
(see ``paged``).  Drafts come from the sequence itself: what followed the last occurrence
of its latest tokens.
"""

from __future__ import annotations

import torch

from . import ops
from .decoder import DecoderConfig
from .paged import PagedKV8Cache
from .verify import verify_drafts
from .w4 import W4Weight, gemv_w4

_FEW = 64  # rows up to which a product runs on the 4-bit weight itself


def lookup_drafts(tokens: list[int], most: int, match: int = 2) -> list[int]:
    """Up to ``most`` tokens that followed the last earlier occurrence of the
    sequence's ``match`` latest tokens."""
    if most <= 0 or len(tokens) <= match:
        return []
    tail = tokens[-match:]
    for i in range(len(tokens) - match - 1, -1, -1):
        if tokens[i:i + match] == tail:
            return tokens[i + match:i + match + most]
    return []


class PagedDecoder:
    """``batch`` sequences of up to ``max_tokens`` tokens."""

    def __init__(self, cfg: DecoderConfig, *, batch: int, max_tokens: int, page_size: int = 64, group_size: int = 128,
                 device: torch.device | str = "cuda"):
        if batch <= 0 or max_tokens <= 0:
            raise ValueError("batch and max_tokens must be positive")
        self.cfg, self.batch, self.max_tokens = cfg, batch, max_tokens
        self.dev = torch.device(device)
        g = torch.Generator(device=self.dev)
        g.manual_seed(cfg.seed)
        H, Hkv, d, D = cfg.q_heads, cfg.kv_heads, cfg.head_dim, cfg.hidden

        def dense(*shape):
            return (torch.randn(shape, generator=g, device=self.dev) * cfg.init_std).to(torch.bfloat16)

        def weight(n, k):
            return W4Weight.quantize(dense(n, k), group_size=group_size)

        def ones():
            return torch.ones(D, device=self.dev, dtype=torch.bfloat16)

        self.embed = dense(cfg.vocab, D)
        self.lm_head = weight(cfg.vocab, D)
        self.final_norm = ones()
        self.layers = [dict(attn_norm=ones(), mlp_norm=ones(), wqkv=weight((H + 2 * Hkv) * d, D), wo=weight(D, H * d),
                            w_gate_up=weight(2 * cfg.ffn, D), w_down=weight(D, cfg.ffn)) for _ in range(cfg.num_layers)]
        pages = -(-max_tokens // page_size)
        self.caches = [PagedKV8Cache(batch * pages, kv_heads=Hkv, head_dim=d, page_size=page_size, device=self.dev)
                       for _ in range(cfg.num_layers)]
        self.block_table = torch.arange(batch * pages, dtype=torch.int32, device=self.dev).reshape(batch, pages)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=self.dev)
        inv = 1.0 / (cfg.rope_theta ** (torch.arange(0, d, 2, device=self.dev, dtype=torch.float32) / d))
        angle = torch.arange(max_tokens, device=self.dev, dtype=torch.float32)[:, None] * inv[None]
        self.cos, self.sin = angle.cos(), angle.sin()

    # -- pieces ---------------------------------------------------------------------
    def _norm_linear(self, x, norm, weight):
        if x.shape[0] <= _FEW:
            return gemv_w4(weight, x, mode="rms", norm_weight=norm, eps=self.cfg.rms_eps)
        return ops.rmsnorm(x, norm, self.cfg.rms_eps) @ weight.dequantize().T

    def _linear_add(self, x, weight, residual, *, silu=False):
        if x.shape[0] <= _FEW:
            return gemv_w4(weight, x, mode="silu" if silu else "plain", residual=residual)
        return residual + (ops.silu_mul(x) if silu else x) @ weight.dequantize().T

    @torch.no_grad()
    def forward(self, tokens: torch.Tensor, token_starts: torch.Tensor, max_new_tokens: int,
                last: torch.Tensor | None = None) -> torch.Tensor:
        """Logits of the rows (or of rows ``last`` only): sequence ``s`` brings
        ``tokens[token_starts[s]:token_starts[s + 1]]`` behind its ``lengths[s]``
        tokens.  The lengths stay as they are."""
        batch = dict(lengths=self.lengths, block_table=self.block_table, token_starts=token_starts,
                     max_new_tokens=max_new_tokens)
        x = torch.index_select(self.embed, 0, tokens)
        for lay, cache in zip(self.layers, self.caches):
            qkv = self._norm_linear(x, lay["attn_norm"], lay["wqkv"])
            q = cache.append(qkv, self.cos, self.sin, **batch)
            att = cache.attend(q, max_context=self.max_tokens, **batch).flatten(1)
            x = self._linear_add(att, lay["wo"], x)
            x = self._linear_add(self._norm_linear(x, lay["mlp_norm"], lay["w_gate_up"]), lay["w_down"], x, silu=True)
        if last is not None:
            x = x.index_select(0, last)
        return self._norm_linear(x, self.final_norm, self.lm_head)

    def _starts(self, counts: list[int]) -> torch.Tensor:
        at = [0]
        for n in counts:
            at.append(at[-1] + n)
        return torch.tensor(at, dtype=torch.int32, device=self.dev)

    # -- generation -----------------------------------------------------------------
    @torch.no_grad()
    def generate(self, prompts: list[list[int]], new_tokens: int, *, drafts: int = 4, temperature: float = 1.0,
                 seed: int = 0) -> tuple[list[list[int]], int]:
        """``new_tokens`` tokens for each prompt, and the number of steps taken.
        ``temperature=0`` takes the most likely token (a target that is certain)."""
        if len(prompts) != self.batch or not all(prompts):
            raise ValueError(f"{self.batch} prompts of at least one token expected")
        if max(len(p) for p in prompts) + new_tokens + drafts > self.max_tokens:
            raise ValueError("max_tokens is too small for the prompts and the tokens asked for")
        g = torch.Generator(device=self.dev)
        g.manual_seed(seed)
        self.lengths.zero_()
        text = [list(p) for p in prompts]
        V, B = self.cfg.vocab, self.batch
        steps = 0
        pending = [list(p) for p in text]  # what each sequence brings to the next step
        guesses: list[list[int]] = [[] for _ in text]
        while min(len(t) - len(p) for t, p in zip(text, prompts)) < new_tokens:
            counts = [len(a) + len(b) for a, b in zip(pending, guesses)]
            starts = self._starts(counts)
            tokens = torch.tensor([t for a, b in zip(pending, guesses) for t in a + b], device=self.dev)
            # the rows behind which a token is wanted: the last given one and each guess, padded to `most` guesses
            most = max(len(b) for b in guesses)
            ends = [sum(counts[:s + 1]) for s in range(B)]
            rows = [max(0, min(ends[s] - 1 - len(guesses[s]) + i, ends[s] - 1)) for s in range(B) for i in range(most + 1)]
            logits = self.forward(tokens, starts, max(counts), torch.tensor(rows, device=self.dev))
            if temperature > 0:
                probs = torch.softmax(logits.float() / temperature, -1)
            else:
                probs = torch.zeros(logits.shape, device=self.dev).scatter_(1, logits.argmax(-1, keepdim=True), 1.0)
            guess = torch.zeros((B, most), dtype=torch.int32)
            for s, b in enumerate(guesses):
                guess[s, :len(b)] = torch.tensor(b, dtype=torch.int32)
            accepted, out = verify_drafts(
                probs.reshape(B, most + 1, V), None, guess.to(self.dev),
                torch.rand((B, most), generator=g, device=self.dev),
                torch.empty((B, V), device=self.dev).exponential_(generator=g),
                draft_counts=torch.tensor([len(b) for b in guesses], dtype=torch.int32, device=self.dev))
            given = torch.tensor([len(a) for a in pending], dtype=torch.int32, device=self.dev)
            self.lengths += given + accepted
            steps += 1
            for s, (a, row) in enumerate(zip(accepted.tolist(), out.tolist())):
                if not pending[s]:
                    continue
                text[s] += row[:a + 1]
                left = new_tokens - (len(text[s]) - len(prompts[s]))
                # a sequence that has its tokens brings no more rows
                pending[s] = [row[a]] if left > 0 else []
                guesses[s] = lookup_drafts(text[s], min(drafts, left - 1))
        return [t[len(p):len(p) + new_tokens] for t, p in zip(text, prompts)], steps
