"""The pages of a cache: appends, growth, branches, eviction, release and
compaction against the oracle's bookkeeping on plain lists.  Everything moves
values or counts, so everything is compared exactly."""

from __future__ import annotations

import random

import pytest
import torch

import batch_invariant_ops as bio
from batch_invariant_ops import _lib
from oracle import bio_oracle

pytestmark = pytest.mark.gpu

DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def i32(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def cache(layers=2, pages=40, page=4, heads=2, d=16, dv=None, rows=8, max_tokens=64,
          dtype=torch.float32, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    c = bio.PagedKVCache(layers, pages, page, heads, d, value_dim=dv, rows=rows,
                         max_tokens=max_tokens, dtype=dtype)
    c.key_pages.copy_(torch.randn(c.key_pages.shape, generator=gen, device="cuda"))
    c.value_pages.copy_(torch.randn(c.value_pages.shape, generator=gen, device="cuda"))
    return c


def book_of(c):
    return bio_oracle.PageBook(c.page_table.cpu(), c.seq_lens.cpu(), c.ref_counts.cpu(),
                               c.page_size)


def same(c, book):
    table, lens, refs = book.state()
    assert torch.equal(c.page_table.cpu(), table)
    assert torch.equal(c.seq_lens.cpu(), lens)
    assert torch.equal(c.ref_counts.cpu(), refs)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,d,dv,page", [(2, 16, 16, 4), (8, 128, 128, 16), (1, 256, 256, 16),
                                             (3, 72, 40, 5), (1, 1, 3, 1), (2, 33, 64, 100)])
def test_append_writes_exactly_its_slots(heads, d, dv, page, dtype):
    gen = torch.Generator(device="cuda").manual_seed(d)
    c = cache(1, 30, page, heads, d, dv, rows=4, max_tokens=6 * page, dtype=dtype)
    c.extend(i32(2, 0, 3), i32(5 * page, 2 * page + 1, 1))
    rows = i32(*([2] * (5 * page) + [0] * (2 * page + 1) + [3] + [1]))
    positions = i32(*range(5 * page), *range(2 * page + 1), 0, -1)
    n = rows.numel()
    # keys and values as slices of a fused projection, tokens in any order
    fused = torch.randn(n, 2 * heads + 3, max(d, dv), generator=gen, device="cuda").to(dtype)
    order = torch.randperm(n, generator=gen, device="cuda")
    fused, rows, positions = fused[order], rows[order], positions[order]
    k, v = fused[:, :heads, :d], fused[:, heads:2 * heads, :dv]
    want_k, want_v = c.key_pages.clone(), c.value_pages.clone()
    for t in range(n):
        r, p = int(rows[t]), int(positions[t])
        if p >= 0:
            at = int(c.page_table[r, p // page])
            want_k[0, at, :, p % page], want_v[0, at, :, p % page] = k[t], v[t]
    c.append(0, k, v, rows, positions)
    assert torch.equal(c.key_pages, want_k) and torch.equal(c.value_pages, want_v)


def test_append_skips_what_is_out_of_range():
    c = cache(1, 10, 4, 2, 16, rows=3, max_tokens=16)
    c.extend(i32(0), i32(6))
    c.page_table[2, 0] = 10
    before = c.key_pages.clone(), c.value_pages.clone()
    k = torch.ones(6, 2, 16, device="cuda")
    # no page yet, beyond the width, rows out of range, a page that the pool lacks
    c.append(0, k, k, i32(0, 0, -1, 3, 2, 1), i32(8, 16, 0, 0, 0, 0))
    assert torch.equal(c.key_pages, before[0]) and torch.equal(c.value_pages, before[1])
    assert _lib.device_status() == _lib.BIO_DEV_INDEX
    _lib.clear_device_status()
    c.append(0, k[:0], k[:0], i32(), i32())


@pytest.mark.parametrize("seed", range(6))
def test_a_random_life(seed):
    """Extends, forks, evictions, releases and compactions in random order."""
    rng = random.Random(seed)
    rows, page, width = 9, rng.choice([1, 3, 4, 16]), 12
    c = cache(2, 150, page, 2, 8, rows=rows, max_tokens=width * page, seed=seed)
    book = book_of(c)
    for _ in range(40):
        what = rng.choice(["extend", "extend", "fork", "evict", "free", "compact"])
        some = rng.sample(range(rows), rng.randint(1, rows))
        if what == "extend":
            to = [min(width * page, book.lens[r] + rng.randint(0, 3 * page)) for r in some]
            c.extend(i32(*some), i32(*to))
            book.extend(some, to)
        elif what == "fork":
            cut = rng.randint(1, max(1, len(some) - 1))
            src, dst = some[:cut], some[cut:]
            src = [rng.choice(src) for _ in dst]
            k, v = c.key_pages.clone(), c.value_pages.clone()
            c.fork(i32(*src), i32(*dst))
            for a, b, n in book.fork(src, dst):
                if a >= 0:
                    k[:, b, :, :n], v[:, b, :, :n] = k[:, a, :, :n], v[:, a, :, :n]
            for new, want in ((c.key_pages, k), (c.value_pages, v)):
                assert torch.equal(new.view(torch.int32), want.view(torch.int32))
        elif what == "evict":
            w, s = rng.randint(1, 3 * page), rng.randint(0, 2 * page)
            c.evict(i32(*some), w, s)
            book.evict(some, w, s)
        elif what == "free":
            c.free(i32(*some[:2]))
            book.free(some[:2])
        else:
            pages = rng.choice([150, 170, 140])
            old = c
            c = old.compact(pages)
            live = book.compact(pages)
            # as bits: pages that were never written hold anything
            for new, was in ((c.key_pages, old.key_pages), (c.value_pages, old.value_pages)):
                assert torch.equal(new[:, :len(live)].view(torch.int32),
                                   was[:, live].view(torch.int32))
        same(c, book)
    assert _lib.device_status() == 0


def test_extend_over_a_large_pool():
    """More pages than one sweep of the scan, some in use, more than 1024 rows."""
    pages, rows, page = 9000, 1500, 2
    c = cache(1, pages, page, 1, 2, rows=rows, max_tokens=12)
    gen = torch.Generator().manual_seed(1)
    c.ref_counts.copy_((torch.rand(pages, generator=gen) < 0.4).to(torch.int32))
    book = book_of(c)
    order = torch.randperm(rows, generator=gen)
    to = torch.randint(0, 8, (rows,), generator=gen)
    c.extend(order.to(torch.int32).cuda(), to.to(torch.int32).cuda())
    book.extend(order.tolist(), to.tolist())
    same(c, book)


def test_extend_when_the_pool_runs_out():
    c = cache(1, 5, 4, 1, 8, rows=3, max_tokens=32)
    book = book_of(c)
    c.extend(i32(1, 0, 2), i32(9, 14, 3))
    book.extend([1, 0, 2], [9, 14, 3])
    same(c, book)
    assert c.seq_lens.tolist() == [8, 9, 0]
    assert _lib.device_status() == _lib.BIO_DEV_PAGES
    _lib.clear_device_status()


def test_extend_refuses_bad_rows():
    c = cache(1, 20, 4, 1, 8, rows=3, max_tokens=16)
    c.extend(i32(1, 1, -1, 3, 0, 2), i32(5, 9, 4, 4, 17, -1))
    assert c.seq_lens.tolist() == [0, 5, 0] and int((c.ref_counts > 0).sum()) == 2
    assert _lib.device_status() == _lib.BIO_DEV_INDEX
    _lib.clear_device_status()


def test_fork_refuses_bad_pairs():
    c = cache(1, 20, 4, 1, 8, rows=6, max_tokens=16)
    c.extend(i32(0, 1), i32(5, 8))
    # 2 is twice a destination, 1 in both lists, -1 and 6 out of range: 1 -> 3 and 0 -> 4 stand
    c.fork(i32(0, 1, 0, 1, 0, -1, 0), i32(2, 2, 1, 3, 4, 5, 6))
    assert c.seq_lens.tolist() == [5, 8, 0, 8, 5, 0]
    assert c.page_table[3].tolist() == c.page_table[1].tolist()
    assert _lib.device_status() == _lib.BIO_DEV_INDEX
    _lib.clear_device_status()


def test_fork_without_a_free_page_ends_at_the_last_whole_page():
    c = cache(1, 4, 4, 1, 8, rows=4, max_tokens=16)
    c.extend(i32(0), i32(10))
    c.fork(i32(0, 0), i32(1, 2))
    assert c.seq_lens.tolist() == [10, 10, 8, 0]
    assert c.ref_counts.tolist() == [3, 3, 1, 1]
    assert _lib.device_status() == _lib.BIO_DEV_PAGES
    _lib.clear_device_status()


@pytest.mark.parametrize("heads,d,dv,page", [(2, 64, 64, 16), (3, 33, 72, 7)])
def test_many_branches_in_many_layers(heads, d, dv, page):
    """More branches and layers than blocks run at once."""
    c = cache(40, 200, page, heads, d, dv, rows=80, max_tokens=4 * page, dtype=torch.bfloat16)
    lens = [page - 1, 2 * page, 3 * page - 2, 1]
    c.extend(i32(0, 1, 2, 3), i32(*lens))
    book, keys, values = book_of(c), c.key_pages.clone(), c.value_pages.clone()
    src, dst = [i % 4 for i in range(64)], list(range(10, 74))
    c.fork(i32(*src), i32(*dst))
    for s, r in zip(src, dst):
        book.fork([s], [r])
    same(c, book)
    for s, r in zip(src, dst):
        for n in range(0, lens[s], page):
            have = min(page, lens[s] - n)
            a, b = c.page_table[s, n // page].item(), c.page_table[r, n // page].item()
            assert torch.equal(c.key_pages[:, b, :, :have], keys[:, a, :, :have])
            assert torch.equal(c.value_pages[:, b, :, :have], values[:, a, :, :have])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,d,dv,page", [(8, 128, 256, 64), (2, 256, 64, 256)])
def test_compact_of_large_pages(heads, d, dv, page, dtype):
    """Pages of more bytes than a block copies at once."""
    c = cache(3, 30, page, heads, d, dv, rows=4, max_tokens=12 * page, dtype=dtype)
    c.extend(i32(0, 1, 2), i32(4 * page, 5 * page - 3, 9 * page))
    c.free(i32(1))
    book = book_of(c)
    out, live = c.compact(16), book.compact(16)
    same(out, book)
    assert torch.equal(out.key_pages[:, :len(live)], c.key_pages[:, live])
    assert torch.equal(out.value_pages[:, :len(live)], c.value_pages[:, live])


def test_free_ignores_repeated_rows():
    c = cache(1, 10, 4, 1, 8, rows=3, max_tokens=16)
    c.extend(i32(0, 1), i32(9, 9))
    c.free(i32(1, 1, 7))
    assert c.seq_lens.tolist() == [9, 0, 0] and c.ref_counts.tolist() == [1] * 3 + [0] * 7
    assert _lib.device_status() == _lib.BIO_DEV_INDEX
    _lib.clear_device_status()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layers,heads,d,dv,page", [(3, 2, 16, 16, 4), (1, 8, 128, 128, 16),
                                                    (2, 1, 33, 7, 5), (2, 3, 72, 72, 100)])
def test_compact_into_other_strides(layers, heads, d, dv, page, dtype):
    """A pool laid out token-major and padded, into a dense smaller one and back."""
    c = cache(layers, 50, page, heads, d, dv, rows=5, max_tokens=8 * page, dtype=dtype)
    c.extend(i32(4, 1, 0), i32(7 * page, 3, 5 * page - 1))
    c.free(i32(1))
    c.fork(i32(0), i32(2))
    book = book_of(c)
    k = torch.zeros(layers, 50, page, heads, d + 1, dtype=dtype, device="cuda")
    k = k.transpose(2, 3)[..., 1:]
    k.copy_(c.key_pages)
    v = torch.zeros(layers, 50, heads, page, dv + 2, dtype=dtype, device="cuda")[..., :dv]
    v.copy_(c.value_pages)
    live = book.compact(20)
    out = bio.PagedKVCache(layers, 20, page, heads, d, value_dim=dv, rows=5,
                           max_tokens=8 * page, dtype=dtype)
    bio.paged_kv_compact(k, v, c.page_table, c.ref_counts, out.key_pages, out.value_pages,
                         out.page_table, out.ref_counts)
    out.seq_lens.copy_(c.seq_lens)
    same(out, book)
    assert torch.equal(out.key_pages[:, :len(live)], c.key_pages[:, live])
    assert torch.equal(out.value_pages[:, :len(live)], c.value_pages[:, live])
    bio.paged_kv_compact(out.key_pages, out.value_pages, out.page_table, out.ref_counts, k, v,
                         c.page_table, c.ref_counts)
    assert torch.equal(k[:, :len(live)], out.key_pages[:, :len(live)])


def test_compact_drops_what_does_not_fit():
    c = cache(1, 10, 4, 1, 8, rows=3, max_tokens=16)
    c.extend(i32(0, 1), i32(8, 8))
    out = c.compact(3)
    assert out.page_table[:2, :2].tolist() == [[0, 1], [2, -1]]
    assert out.ref_counts.tolist() == [1, 1, 1]
    assert _lib.device_status() == _lib.BIO_DEV_PAGES
    _lib.clear_device_status()


def test_compact_of_an_empty_pool():
    out = cache(1, 10, 4, 1, 8, rows=3, max_tokens=16).compact(2)
    assert out.ref_counts.tolist() == [0, 0] and int(out.page_table.max()) == -1


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_keeps_its_bits_through_the_cache_s_life(dtype):
    """A row's output is the same after a fork, after eviction under its window,
    and in a compacted pool; a branch goes on by itself."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    heads, d, page, window, sinks = 2, 64, 16, 40, 4
    c = cache(1, 60, page, heads, d, rows=4, max_tokens=300, dtype=dtype)
    new = lambda n: torch.randn(n, heads, d, generator=gen, device="cuda").to(dtype)  # noqa: E731
    c.extend(i32(0), i32(200))
    c.append(0, new(200), new(200), i32(*[0] * 200), i32(*range(200)))
    q = torch.randn(4, 8, d, generator=gen, device="cuda").to(dtype)
    q[1:] = q[0]
    one, zero = i32(0), q[:1]
    attend = lambda c, **k: c.attend(0, zero, rows=one, **k)  # noqa: E731
    plain, windowed = attend(c), attend(c, window=window, sinks=sinks)
    c.fork(i32(0, 0), i32(1, 3))
    both = c.attend(0, q[[0, 0, 0]], rows=i32(0, 1, 3))
    assert torch.equal(both, plain.expand(3, -1, -1))
    # the branch grows, its source does not notice
    c.extend(i32(1), i32(201))
    c.append(0, new(1), new(1), i32(1), i32(200))
    assert torch.equal(attend(c), plain)
    assert not torch.equal(c.attend(0, zero, rows=i32(1)), plain)
    c.evict(i32(0, 1, 3), window, sinks)
    assert int((c.page_table[0] >= 0).sum()) < 13
    assert torch.equal(attend(c, window=window, sinks=sinks), windowed)
    small = c.compact(int((c.ref_counts > 0).sum()))
    assert torch.equal(attend(small, window=window, sinks=sinks), windowed)


def test_streams_and_graphs():
    """A decode step captured once and replayed: extend, append, attend."""
    c = cache(1, 40, 4, 2, 64, rows=3, max_tokens=64, dtype=torch.bfloat16)
    gen = torch.Generator(device="cuda").manual_seed(2)
    rows, lens = i32(0, 1, 2), i32(5, 9, 1)
    k = torch.randn(3, 2, 64, generator=gen, device="cuda").bfloat16()
    q = torch.randn(3, 8, 64, generator=gen, device="cuda").bfloat16()
    eager = cache(1, 40, 4, 2, 64, rows=3, max_tokens=64, dtype=torch.bfloat16)

    def step(c, lens):
        c.extend(rows, lens)
        c.append(0, k, k, rows, lens - 1)
        return c.attend(0, q)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(c, lens)
        step(eager, lens)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(c, lens)
    for _ in range(5):
        lens += 1
        graph.replay()
        assert torch.equal(held, step(eager, lens))
        assert torch.equal(c.page_table, eager.page_table)
