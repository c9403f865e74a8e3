"""Serving a sliding-window decoder from a paged cache: the operators of
``paged`` and the sliding-window attention run together.

``Decoder`` is a random-init decoder-only language model (rotary positions,
grouped-query attention over a sliding window with sink tokens, RMSNorm,
SwiGLU).  ``generate`` answers prompts of different lengths with several
sampled continuations each:

1. all prompts go through the model once, packed behind each other (packed
   sliding-window attention), while each layer appends its keys and values to
   the cache;
2. every prompt branches off into its continuations (fork: whole pages are
   shared, the last partial page is copied);
3. pages that the window has passed are released (evict) and the pool, which
   had to hold whole prompts, is moved into one that holds windows (compact);
4. each step extends all rows by a token, appends and attends (paged decode),
   and releases what the window has passed.

Every operator here is batch invariant, so a prompt's continuations have the
same tokens whichever prompts it is served with.  Not in the reference, whose
models run no decoding loop.

    python -m batch_invariant_ops.decoder      # needs a B200
"""

from __future__ import annotations

import dataclasses
import math
import time

import torch
import torch.nn.functional as F

from .batch_invariant_ops import (
    gated_linear_batch_invariant,
    linear_batch_invariant,
    linear_residual_batch_invariant,
    rms_norm_batch_invariant,
    varlen_sliding_window_attention_batch_invariant,
)
from .paged import PagedKVCache


@dataclasses.dataclass(frozen=True)
class DecoderConfig:
    width: int = 2048
    layers: int = 18
    heads: int = 16
    kv_heads: int = 4
    head_dim: int = 128
    mlp: int = 8192
    vocab: int = 32000
    window: int = 1024
    sinks: int = 4
    page_size: int = 16
    dtype: torch.dtype = torch.bfloat16

    @staticmethod
    def tiny() -> "DecoderConfig":
        return DecoderConfig(width=128, layers=2, heads=4, kv_heads=2, head_dim=64, mlp=256,
                             vocab=512, window=48, sinks=4, page_size=16)

    def pages(self, tokens: int) -> int:
        return -(-tokens // self.page_size)

    def window_pages(self) -> int:
        """Pages that a row holds at most once its window has been evicted to:
        the window may begin and end inside a page, and a new page may begin."""
        return self.pages(self.sinks) + self.pages(self.window) + 2


class Decoder(torch.nn.Module):
    def __init__(self, cfg: DecoderConfig, device: torch.device | str = "cuda", seed: int = 0):
        super().__init__()
        self.cfg = c = cfg
        gen = torch.Generator(device=device).manual_seed(seed)

        def w(*shape, std=None):
            x = torch.randn(*shape, generator=gen, device=device)
            return torch.nn.Parameter((x * (std or shape[-1] ** -0.5)).to(c.dtype),
                                      requires_grad=False)

        def ones():
            return torch.nn.Parameter(torch.ones(c.width, dtype=c.dtype, device=device),
                                      requires_grad=False)

        self.embed = w(c.vocab, c.width, std=1.0)
        self.blocks = torch.nn.ModuleList(torch.nn.ParameterList([
            ones(), w((c.heads + 2 * c.kv_heads) * c.head_dim, c.width),
            w(c.width, c.heads * c.head_dim), ones(), w(2 * c.mlp, c.width), w(c.width, c.mlp),
        ]) for _ in range(c.layers))
        self.norm = ones()
        self.head = w(c.vocab, c.width)
        half = c.head_dim // 2
        self.register_buffer("freq", 10000.0 ** -(torch.arange(half, device=device) / half))

    def _rms(self, x, g):
        return rms_norm_batch_invariant(x, (self.cfg.width,), g, 1e-6)

    def _rotate(self, x, cos, sin):
        a, b = x.float().chunk(2, dim=-1)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(x.dtype)

    def _run(self, ids, positions, rows, cache, attend):
        """Tokens ids [T] at `positions` of table rows `rows`; their keys and values go
        into the cache, `attend(layer, q, k, v)` gives [T, heads, head_dim]."""
        c = self.cfg
        angle = positions[:, None].float() * self.freq
        cos, sin = angle.cos()[:, None], angle.sin()[:, None]
        x = F.embedding(ids, self.embed)
        for i, (n1, wqkv, wo, n2, w_in, w_out) in enumerate(self.blocks):
            qkv = linear_batch_invariant(self._rms(x, n1), wqkv).view(
                -1, c.heads + 2 * c.kv_heads, c.head_dim)
            q = self._rotate(qkv[:, :c.heads], cos, sin)
            k = self._rotate(qkv[:, c.heads:c.heads + c.kv_heads], cos, sin)
            v = qkv[:, c.heads + c.kv_heads:]
            cache.append(i, k, v, rows, positions)
            a = attend(i, q, k, v)
            x = linear_residual_batch_invariant(x, a.flatten(1), wo)
            h = gated_linear_batch_invariant(self._rms(x, n2), w_in, "silu")
            x = linear_residual_batch_invariant(x, h, w_out)
        return x

    def _logits(self, x):
        return linear_batch_invariant(self._rms(x, self.norm), self.head).float()

    def prefill(self, ids, offsets, rows, positions, cache):
        """Packed prompts: ids, rows and positions [T], offsets int32 [P + 1].
        Logits after the last token of each prompt [P, vocab]."""
        c = self.cfg

        def attend(_, q, k, v):
            return varlen_sliding_window_attention_batch_invariant(
                q[None], k[None], v[None], offsets, offsets, c.window, c.sinks)[0]

        x = self._run(ids, positions, rows, cache, attend)
        return self._logits(x[offsets[1:].long() - 1])

    def step(self, ids, rows, cache):
        """One new token of each row, which the cache has been extended by.
        Logits [R, vocab]."""
        c = self.cfg

        def attend(layer, q, _k, _v):
            return cache.attend(layer, q, rows=rows, window=c.window, sinks=c.sinks)

        positions = cache.seq_lens[rows.long()] - 1
        return self._logits(self._run(ids, positions, rows, cache, attend))


def generate(model: Decoder, prompts: list, steps: int, branches: int = 1,
             temperature: float = 1.0, seeds: list | None = None):
    """`branches` continuations of `steps` tokens for each prompt (1-D int64
    tensors of at least one token), drawn with one generator per prompt
    (`seeds[p]`, default p).  Returns tokens [P, branches, steps] on the model's
    device."""
    c, device = model.cfg, model.embed.device
    if not prompts or min(p.numel() for p in prompts) < 1 or branches < 1 or steps < 1:
        raise ValueError("generate needs prompts of at least one token, branches and steps")
    count, lens = len(prompts), [p.numel() for p in prompts]
    rows = count * branches
    # row p * branches holds the prompt, the rows behind it branch off it
    cache = PagedKVCache(
        c.layers, sum(map(c.pages, lens)) + rows, c.page_size, c.kv_heads, c.head_dim,
        rows=rows, max_tokens=max(lens) + steps, dtype=c.dtype, device=device)
    int32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    heads_of = int32([p * branches for p in range(count)])
    every = torch.arange(rows, dtype=torch.int32, device=device)
    lens_t = int32(lens)
    offsets = int32([0, *torch.tensor(lens).cumsum(0).tolist()])
    positions = torch.cat([torch.arange(n, dtype=torch.int32) for n in lens]).to(device)

    cache.extend(heads_of, lens_t)
    logits = model.prefill(torch.cat(prompts).to(device), offsets,
                           heads_of.repeat_interleave(lens_t), positions, cache)
    if branches > 1:
        others = every[every % branches != 0]
        cache.fork(others // branches * branches, others)
    cache.evict(every, c.window, c.sinks)
    # a row's sinks and window at most, and no more than the row will ever hold
    need = sum(branches * min(c.window_pages(), c.pages(n + steps)) for n in lens)
    cache = cache.compact(need)

    generators = [torch.Generator(device=device).manual_seed(p if seeds is None else seeds[p])
                  for p in range(count)]

    def draw(logits):  # [rows, vocab] -> [rows]
        noise = torch.stack([torch.rand(branches, c.vocab, generator=g, device=device)
                             for g in generators]).flatten(0, 1)
        gumbel = -torch.log(-torch.log(noise.clamp(1e-20, 1 - 1e-7)))
        return (logits / max(temperature, 1e-6) + gumbel).argmax(-1)

    out = [draw(logits.repeat_interleave(branches, 0))]
    for _ in range(steps - 1):
        cache.extend(every, cache.seq_lens + 1)
        logits = model.step(out[-1], every, cache)
        cache.evict(every, c.window, c.sinks)
        out.append(draw(logits))
    return torch.stack(out, 1).view(count, branches, steps)


def main() -> None:
    cfg = DecoderConfig()
    model = Decoder(cfg)
    gen = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, cfg.vocab, (n,), generator=gen) for n in (3000, 17, 1500, 777)]
    steps, branches = 64, 4
    generate(model, prompts, 2, branches)
    torch.cuda.synchronize()
    start = time.perf_counter()
    tokens = generate(model, prompts, steps, branches)
    torch.cuda.synchronize()
    seconds = time.perf_counter() - start
    alone = generate(model, prompts[2:3], steps, branches, seeds=[2])
    print(f"{len(prompts)} prompts of {[p.numel() for p in prompts]} tokens, {branches} "
          f"continuations of {steps} tokens each: {seconds * 1e3:.0f} ms, "
          f"{math.prod(tokens.shape) / seconds:.0f} tokens/s")
    print("same tokens alone and in the batch:", torch.equal(alone[0], tokens[2]))


if __name__ == "__main__":
    main()
