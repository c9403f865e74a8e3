"""Attention over a paged cache against the 64-bit oracle.

Tolerances.  With u the unit roundoff of the dtype (2^-8 bf16, 2^-11 fp16,
2^-24 fp32), v* the largest |value| that a row sees and S the largest scale *
sum |q_i k_i| of its keys, the output is a weighted mean of values, so

* rounding the weights to the dtype, an exponential good to 2 u, and rounding
  the output cost at most 4 u v* (16-bit types);
* fp32 dot products of D terms move a score by at most D 2^-24 S, its weight
  by twice that; sums over n tokens cost 2 n 2^-24 relative;

which gives |out - oracle| <= v* (4 u + 2^-24 (2 D S + 2 n + 8)), for fp32
with u = 2^-24.  Rounding errors are independent, so the norm of the error of a
16-bit output stays under 2 u of the output's.
"""

from __future__ import annotations

import pytest
import torch

import batch_invariant_ops as bio
from batch_invariant_ops import _lib
from oracle import bio_oracle

pytestmark = pytest.mark.gpu

UNIT = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
DTYPES = tuple(UNIT)


def make(lens, heads, kv_heads, d, dv=None, page=16, dtype=torch.bfloat16, seed=0, width=None,
         fill=float("nan"), spread=1.0):
    """Query, pages, table and lengths; slots that hold no token get `fill`."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dv = dv or d
    need = [-(-n // page) for n in lens]
    width = width or max(max(need), 1)
    pages = sum(need) + 2
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    kp = torch.full((pages, kv_heads, page, d), fill, dtype=dtype, device="cuda")
    vp = torch.full((pages, kv_heads, page, dv), fill, dtype=dtype, device="cuda")
    at = 0
    for b, n in enumerate(lens):
        table[b, :need[b]] = order[at:at + need[b]]
        at += need[b]
        if n == 0:
            continue
        t = torch.arange(n, device="cuda")
        p, s = table[b, t // page].long(), t % page
        kp[p, :, s] = torch.randn(n, kv_heads, d, generator=gen, device="cuda").to(dtype)
        vp[p, :, s] = torch.randn(n, kv_heads, dv, generator=gen, device="cuda").to(dtype)
    q = (spread * torch.randn(len(lens), heads, d, generator=gen, device="cuda")).to(dtype)
    return q, kp, vp, table, torch.tensor(lens, dtype=torch.int32, device="cuda")


def check(out, args, window=None, sinks=0, scale=None, rows=None):
    q, kp, vp, table, lens = args
    ref = bio_oracle.paged_attention(q, kp, vp, table, lens, window, sinks, scale, rows)
    u, d = UNIT[q.dtype], q.shape[-1]
    scale = d ** -0.5 if scale is None else scale
    got = out.double().cpu()
    assert got.shape == ref.shape and out.dtype == q.dtype
    for b, r in enumerate(rows.tolist() if rows is not None else range(q.shape[0])):
        keys = bio_oracle.visible_keys(int(lens[r]) - 1, window, sinks).cuda()
        if keys.numel() == 0:
            assert torch.equal(got[b], torch.zeros_like(got[b]))
            continue
        page = kp.shape[2]
        p, s = table[r, keys // page].long(), keys % page
        k, v = kp[p, :, s].double(), vp[p, :, s].double()
        group = q.shape[1] // kp.shape[1]
        reach = abs(scale) * torch.einsum(
            "gad,ngd->gan", q[b].double().abs().view(kp.shape[1], group, d), k.abs()).max()
        top = v.abs().max().item()
        bound = top * (4 * u + 2.0**-24 * (2 * d * reach.item() + 2 * keys.numel() + 8))
        err = (got[b] - ref[b]).abs().max().item()
        assert err <= bound, f"row {b}: {err} > {bound}"
    if q.dtype != torch.float32 and ref.norm() > 0:
        assert ((got - ref).norm() / ref.norm()).item() <= 2 * u
    return ref


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,d", [
    (1, 1, 64), (8, 1, 256), (4, 4, 128), (32, 8, 128), (6, 2, 72), (10, 2, 80), (14, 2, 96),
    (16, 1, 128), (20, 1, 64), (40, 1, 128), (3, 1, 8), (2, 2, 1), (5, 1, 33), (4, 2, 100),
    (2, 1, 200),
])
def test_matches_the_oracle(heads, kv_heads, d, dtype):
    lens = [0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300, 1025]
    args = make(lens, heads, kv_heads, d, dtype=dtype, seed=d + heads)
    check(bio.paged_attention_decode_batch_invariant(*args), args)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,dv", [(64, 128), (128, 64), (256, 64), (40, 256), (24, 17)])
def test_value_dim_of_its_own(d, dv, dtype):
    args = make([5, 200, 0, 1300], 8, 2, d, dv, dtype=dtype, seed=dv)
    check(bio.paged_attention_decode_batch_invariant(*args), args)


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float32))
@pytest.mark.parametrize("page", (1, 3, 8, 16, 64, 100, 256, 1000))
def test_page_sizes_give_the_same_bits(page, dtype):
    lens = [1, 99, 100, 101, 800]
    args = make(lens, 8, 2, 64, page=page, dtype=dtype)
    out = bio.paged_attention_decode_batch_invariant(*args)
    check(out, args)
    # the same tokens in pages of 16
    q, kp, vp, table, ln = args
    other = make(lens, 8, 2, 64, page=16, dtype=dtype)
    for b, n in enumerate(lens):
        t = torch.arange(n, device="cuda")
        for a, x in ((kp, other[1]), (vp, other[2])):
            x[other[3][b, t // 16].long(), :, t % 16] = a[table[b, t // page].long(), :, t % page]
    assert torch.equal(bio.paged_attention_decode_batch_invariant(q, *other[1:]), out)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 0), (16, 4), (50, 100), (64, 17),
                                          (129, 3), (4096, 4)])
def test_window_and_sinks(window, sinks, dtype):
    lens = [0, 1, 15, 16, 17, 50, 51, 66, 150, 1025, 2000]
    args = make(lens, 8, 2, 128, dtype=dtype, seed=window)
    q, kp, vp, table, ln = args
    # what the window hides is poisoned: it must not be read into the result
    for b, n in enumerate(lens):
        t = torch.arange(n, device="cuda")
        t = t[(t < n - window) & (t >= sinks)]
        kp[table[b, t // 16].long(), :, t % 16] = float("inf")
        vp[table[b, t // 16].long(), :, t % 16] = float("nan")
    out = bio.paged_attention_decode_batch_invariant(*args, window=window, sinks=sinks)
    check(out, args, window, sinks)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", (8193, 32769, 40001))
def test_long_rows(n, dtype):
    args = make([n, 7, n // 2], 8, 2, 64, page=64, dtype=dtype, seed=n)
    check(bio.paged_attention_decode_batch_invariant(*args), args)
    check(bio.paged_attention_decode_batch_invariant(*args, window=n - 300, sinks=5), args,
          n - 300, 5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,d", [(8, 1, 256), (32, 8, 128), (4, 4, 64), (5, 1, 33)])
def test_a_row_does_not_depend_on_the_batch(heads, kv_heads, d, dtype):
    lens = [700, 1, 0, 64, 1024, 3000, 129, 9000]
    args = make(lens, heads, kv_heads, d, dtype=dtype, seed=3)
    q, kp, vp, table, ln = args
    full = bio.paged_attention_decode_batch_invariant(*args)
    for b in range(len(lens)):
        need = max(1, -(-lens[b] // 16))
        alone = bio.paged_attention_decode_batch_invariant(
            q[b:b + 1], kp, vp, table[b:b + 1, :need], ln[b:b + 1])
        assert torch.equal(alone, full[b:b + 1]), f"row {b} changed"
    order = torch.tensor([5, 0, 0, 7, 2], dtype=torch.int32, device="cuda")
    some = bio.paged_attention_decode_batch_invariant(q[order.long()], kp, vp, table, ln,
                                                      rows=order)
    assert torch.equal(some, full[order.long()])
    for _ in range(3):
        assert torch.equal(bio.paged_attention_decode_batch_invariant(*args), full)


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
def test_extreme_scores(dtype):
    """Scores of thousands, equal scores, one score far above the rest."""
    q, kp, vp, table, ln = make([500, 500, 500], 8, 2, 64, dtype=dtype, fill=0.0, spread=200.0)
    q[1] = 0
    args = (q, kp, vp, table, ln)
    check(bio.paged_attention_decode_batch_invariant(*args), args)
    check(bio.paged_attention_decode_batch_invariant(*args, scale=-0.3), args, scale=-0.3)
    check(bio.paged_attention_decode_batch_invariant(*args, scale=0.0), args, scale=0.0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_visible_nan_stays_in_its_row_and_heads(dtype):
    args = make([300, 300, 300], 8, 2, 64, dtype=dtype)
    clean = bio.paged_attention_decode_batch_invariant(*args)
    q, kp, vp, table, ln = args
    vp[table[1, 3].long(), 1, 2, 5] = float("nan")
    out = bio.paged_attention_decode_batch_invariant(*args)
    assert torch.isnan(out[1, 4:, 5]).all()
    out[1, 4:, 5] = clean[1, 4:, 5]
    assert torch.equal(out, clean)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_views(dtype):
    """Pages token-major and as a slice of a larger pool, the query as a slice
    of a fused projection, a table with padding between its rows."""
    q, kp, vp, table, ln = args = make([77, 300, 16, 1], 8, 2, 64, dtype=dtype)
    out = bio.paged_attention_decode_batch_invariant(*args)
    fused = torch.zeros(4, 12, 64, dtype=dtype, device="cuda")
    fused[:, 2:10] = q
    big_k = torch.zeros(kp.shape[0], 16, 2, 64, dtype=dtype, device="cuda")
    big_k.copy_(kp.transpose(1, 2))
    big_v = torch.zeros(3, *vp.shape[:3], 72, dtype=dtype, device="cuda")
    big_v[1, ..., :64] = vp
    wide = torch.full((4, 50), -1, dtype=torch.int32, device="cuda")
    wide[:, 3:3 + table.shape[1]] = table
    got = bio.paged_attention_decode_batch_invariant(
        fused[:, 2:10], big_k.transpose(1, 2), big_v[1, ..., :64], wide[:, 3:3 + table.shape[1]],
        ln)
    assert torch.equal(got, out)
    # rows that start off a 16-byte boundary take another kernel: same tolerance
    odd = torch.zeros(*kp.shape[:3], 67, dtype=dtype, device="cuda")
    odd[..., 3:] = kp
    args = (q, odd[..., 3:], vp, table, ln)
    check(bio.paged_attention_decode_batch_invariant(*args), args)


def test_out_of_range_rows_give_zeros_and_set_the_status():
    q, kp, vp, table, ln = make([40, 40, 40, 2000], 8, 2, 64)
    good = bio.paged_attention_decode_batch_invariant(q, kp, vp, table, ln)
    for what in ("page", "negative page", "length", "negative length", "row"):
        t, n, rows = table.clone(), ln.clone(), torch.arange(4, dtype=torch.int32, device="cuda")
        if what == "page":
            t[1, 2], t[3, 70] = kp.shape[0], kp.shape[0]
        elif what == "negative page":
            t[1, 0], t[3, 0] = -1, -7
        elif what == "length":
            n[1], n[3] = table.shape[1] * 16 + 1, 2**31 - 1
        elif what == "negative length":
            n[1], n[3] = -1, -5
        else:
            rows[1], rows[3] = -1, 4
        out = bio.paged_attention_decode_batch_invariant(q, kp, vp, t, n, rows=rows)
        assert torch.equal(out[::2], good[::2])
        assert torch.equal(out[1::2], torch.zeros_like(out[1::2])), what
        assert _lib.device_status() == _lib.BIO_DEV_INDEX
        _lib.clear_device_status()


def test_empty_inputs():
    q, kp, vp, table, ln = make([3, 4], 4, 2, 64)
    assert bio.paged_attention_decode_batch_invariant(
        q[:0], kp, vp, table[:0], ln[:0]).shape == (0, 4, 64)
    none = torch.zeros(2, 0, dtype=torch.int32, device="cuda")
    out = bio.paged_attention_decode_batch_invariant(q, kp[:0], vp[:0], none, ln * 0)
    assert torch.equal(out, torch.zeros_like(out))


def test_a_cache_beyond_32_bit_offsets():
    """Pages whose elements lie more than 2^32 from the start of the pool."""
    pages = 2**32 // (64 * 128) + 64
    kp = torch.zeros(pages, 1, 64, 128, dtype=torch.bfloat16, device="cuda")
    vp = torch.zeros(pages, 1, 64, 128, dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(1)
    kp[-3:] = torch.randn(3, 1, 64, 128, generator=gen, device="cuda").to(kp.dtype)
    vp[-3:] = torch.randn(3, 1, 64, 128, generator=gen, device="cuda").to(kp.dtype)
    q = torch.randn(1, 8, 128, generator=gen, device="cuda").to(kp.dtype)
    table = torch.tensor([[pages - 1, pages - 3, pages - 2]], dtype=torch.int32, device="cuda")
    ln = torch.tensor([190], dtype=torch.int32, device="cuda")
    out = bio.paged_attention_decode_batch_invariant(q, kp, vp, table, ln)
    args = (q, kp[-3:], vp[-3:], table - (pages - 3), ln)
    check(out, args)
    assert torch.equal(out, bio.paged_attention_decode_batch_invariant(*args))


def test_streams_and_graphs():
    args = make([700, 3, 2500], 8, 2, 64)
    want = bio.paged_attention_decode_batch_invariant(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = bio.paged_attention_decode_batch_invariant(*args)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = bio.paged_attention_decode_batch_invariant(*args)
    args[4][:] = torch.tensor([1, 3, 900], dtype=torch.int32)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held, bio.paged_attention_decode_batch_invariant(*args))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", (64, 128, 256))
def test_a_wide_table_changes_nothing(d, dtype):
    """The pieces of a row are joined by a warp or by a block, depending on how
    many pieces the table has room for; the bits do not depend on it."""
    args = make([3000, 31, 0, 700, 9000], 8, 2, d, dtype=dtype, seed=d)
    q, kp, vp, table, lens = args
    out = bio.paged_attention_decode_batch_invariant(*args)
    check(out, args)
    wide = torch.full((5, 5000), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    assert torch.equal(bio.paged_attention_decode_batch_invariant(q, kp, vp, wide, lens), out)


@pytest.mark.parametrize("dtype,longest", [(torch.bfloat16, 32), (torch.float16, 32),
                                           (torch.float32, 128)])
def test_rows_of_one_piece_are_written_before_the_next_kernel_reads(dtype, longest):
    """A table with room for many pieces whose rows have one each: nothing is left
    to join, and what follows in the graph or on the stream reads finished rows."""
    lens = [longest] * 200 + [0, 1, longest - 1, longest]
    q, kp, vp, table, ln = make(lens, 32, 2, 128, dtype=dtype, width=256)
    want = bio.paged_attention_decode_batch_invariant(q, kp, vp, table[:, :longest // 16], ln)
    check(want[-6:], (q[-6:], kp, vp, table[-6:], ln[-6:]))
    given, read = torch.zeros_like(q), torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        read.copy_(bio.paged_attention_decode_batch_invariant(given, kp, vp, table, ln))
    given.copy_(q)
    for turn in range(100):
        read.fill_(float("nan"))
        graph.replay()
        assert torch.equal(read, want), f"replay {turn}"
        got = bio.paged_attention_decode_batch_invariant(q, kp, vp, table, ln) + 0
        assert torch.equal(got, want), f"call {turn}"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", (64, 33))
def test_an_empty_pool_under_empty_rows_raises_nothing(d, dtype):
    q, kp, vp, table, ln = make([3, 40], 4, 2, d, dtype=dtype)
    for t in (table, table[:, :0]):
        out = bio.paged_attention_decode_batch_invariant(q, kp[:0], vp[:0], t, ln * 0)
        assert torch.equal(out, torch.zeros_like(out))
        assert _lib.device_status() == 0
    # a token in a pool without pages is still refused
    out = bio.paged_attention_decode_batch_invariant(q, kp[:0], vp[:0], table, ln)
    assert torch.equal(out, torch.zeros_like(out))
    assert _lib.device_status() == _lib.BIO_DEV_INDEX
    _lib.clear_device_status()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", (127, 64))
def test_lengths_up_to_the_last_position(page, dtype):
    """Positions next to 2^31: the longest row that is taken, and rows beyond it."""
    most, window, sinks = 2**31 - 65, 100, 40
    width = (2**31 - 1) // page
    lens = [most, most - 1, most - 33, most + 1, width * page]
    gen = torch.Generator(device="cuda").manual_seed(page)
    # pages 0.. hold the first tokens, the ones after them the last
    first, last = range(sinks // page + 1), range((most - 200) // page, width)
    table = torch.full((1, width), -1, dtype=torch.int32, device="cuda")
    table[0, :len(first)] = torch.arange(len(first))
    table[0, last[0]:] = len(first) + torch.arange(len(last))
    pages = len(first) + len(last)
    kp, vp = (torch.randn(pages, 2, page, 64, generator=gen, device="cuda").to(dtype)
              for _ in range(2))
    q = torch.randn(1, 8, 64, generator=gen, device="cuda").to(dtype)
    for n in lens:
        ln = torch.tensor([n], dtype=torch.int32, device="cuda")
        out = bio.paged_attention_decode_batch_invariant(q, kp, vp, table, ln, window=window,
                                                         sinks=sinks)
        if n > most:
            assert torch.equal(out, torch.zeros_like(out))
            assert _lib.device_status() == _lib.BIO_DEV_INDEX
            _lib.clear_device_status()
            continue
        assert _lib.device_status() == 0
        # the same tokens in a short cache of their own
        keys = torch.cat([torch.arange(sinks), torch.arange(n - window, n)]).cuda()
        p, s = table[0, keys // page].long(), keys % page
        short = -(-keys.numel() // page)
        own = [torch.zeros(short, 2, page, 64, dtype=dtype, device="cuda") for _ in range(2)]
        t = torch.arange(keys.numel(), device="cuda")
        for mine, theirs in zip(own, (kp, vp)):
            mine[t // page, :, t % page] = theirs[p, :, s]
        check(out, (q, *own, torch.arange(short, dtype=torch.int32, device="cuda")[None],
                    torch.tensor([keys.numel()], dtype=torch.int32, device="cuda")))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,d", [(8, 2, 64), (4, 1, 256)])
def test_more_rows_than_a_block_lists(heads, kv_heads, d, dtype):
    """700 rows under a wide table: the pieces that rows lack are passed over, and a
    row has the bits that it has among a few."""
    gen = torch.Generator().manual_seed(d)
    lens = torch.randint(0, 300, (700,), generator=gen)
    lens[torch.tensor([5, 80, 444, 699])] = torch.tensor([9000, 1100, 0, 2500])
    q, kp, vp, table, ln = make(lens.tolist(), heads, kv_heads, d, dtype=dtype, seed=d, width=640)
    out = bio.paged_attention_decode_batch_invariant(q, kp, vp, table, ln, window=6000, sinks=3)
    for some in (torch.arange(0, 12), torch.tensor([80, 444, 511, 512, 513, 698, 699])):
        at = some.to(torch.int32).cuda()
        few = bio.paged_attention_decode_batch_invariant(
            q[some.cuda()], kp, vp, table, ln, rows=at, window=6000, sinks=3)
        assert torch.equal(few, out[some.cuda()])
        check(few, (q[some.cuda()], kp, vp, table, ln), 6000, 3, rows=at)
    assert _lib.device_status() == 0
