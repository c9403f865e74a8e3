"""The sliding-window decoder served from a paged cache: packed prefill, append,
fork, evict, compact and paged decode working together."""

from __future__ import annotations

import pytest
import torch

from batch_invariant_ops import PagedKVCache, _lib
from batch_invariant_ops.decoder import Decoder, DecoderConfig, generate

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model():
    return Decoder(DecoderConfig.tiny())


@pytest.fixture(autouse=True)
def clean_status():
    _lib.clear_device_status()
    yield
    assert _lib.device_status() == 0


def prompt(n, seed=0):
    return torch.randint(0, 512, (n,), generator=torch.Generator().manual_seed(100 * seed + n))


def int32(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def prefill(model, ids, pages=None):
    """A one-row cache that holds `ids`, and the logits after its last token."""
    c, n = model.cfg, ids.numel()
    cache = PagedKVCache(c.layers, pages or c.pages(n) + 4, c.page_size, c.kv_heads, c.head_dim,
                         rows=1, max_tokens=n + 64, dtype=c.dtype)
    cache.extend(int32(0), int32(n))
    logits = model.prefill(ids.cuda(), int32(0, n),
                           torch.zeros(n, dtype=torch.int32, device="cuda"),
                           torch.arange(n, dtype=torch.int32, device="cuda"), cache)
    return cache, logits


def test_a_prompt_gets_the_same_tokens_alone_and_in_a_batch(model):
    prompts = [prompt(n) for n in (1, 200, 47, 48, 133)]
    together = generate(model, prompts, 40, branches=3)
    assert together.shape == (5, 3, 40)
    for i, p in enumerate(prompts):
        alone = generate(model, [p], 40, branches=3, seeds=[i])
        assert torch.equal(alone[0], together[i]), i


def test_branches_do_not_disturb_each_other(model):
    # the first of three branches and a single one draw from generators in
    # different states, so compare greedy decoding: all branches agree
    out = generate(model, [prompt(150)], 30, branches=4, temperature=0.0)
    one = generate(model, [prompt(150)], 30, branches=1, temperature=0.0)
    for b in range(4):
        assert torch.equal(out[0, b], one[0, 0])


@pytest.mark.parametrize("n", [1, 16, 40, 90, 161])
def test_steps_agree_with_a_whole_prefill(model, n):
    """Token by token through the cache and all at once through the packed kernel
    are the same function: bf16 rounding of two layers apart."""
    ids = prompt(n + 20, 1)
    cache, _ = prefill(model, ids[:n], pages=model.cfg.pages(n + 20) + 1)
    for i in range(n, n + 20):
        cache.extend(int32(0), int32(i + 1))
        logits = model.step(ids[i:i + 1].cuda(), int32(0), cache)
    _, whole = prefill(model, ids)
    assert (logits - whole).norm() <= 0.05 * whole.norm()


def test_eviction_and_compaction_keep_the_bits(model):
    c, n = model.cfg, 300
    ids = prompt(n + 30, 2).cuda()
    plain, _ = prefill(model, ids[:n], pages=c.pages(n + 30))
    small, _ = prefill(model, ids[:n])
    small.evict(int32(0), c.window, c.sinks)
    small = small.compact(c.window_pages())
    for i in range(n, n + 30):
        logits = []
        for cache in (plain, small):
            cache.extend(int32(0), int32(i + 1))
            logits.append(model.step(ids[i:i + 1], int32(0), cache))
        small.evict(int32(0), c.window, c.sinks)
        assert torch.equal(*logits), i


def test_generate_refuses(model):
    for args in (([], 4), ([prompt(0)], 4), ([prompt(3)], 0), ([prompt(3)], 4, 0)):
        with pytest.raises(ValueError):
            generate(model, *args)
