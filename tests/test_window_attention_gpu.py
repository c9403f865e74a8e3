"""Sliding-window attention with sink tokens against the 64-bit oracle.

Tolerances are those of tests/test_paged_attention_gpu.py: |out - oracle| <=
v* (4 u + 2^-24 (2 D S + 2 n + 8)) per element, and 2 u in the norm for 16-bit
types."""

from __future__ import annotations

import pytest
import torch

import batch_invariant_ops as bio
from batch_invariant_ops import _lib
from oracle import bio_oracle

pytestmark = pytest.mark.gpu

UNIT = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
DTYPES = tuple(UNIT)


def make(b, h, hk, lq, lk, d, dv=None, dtype=torch.bfloat16, seed=0, spread=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    q = spread * torch.randn(b, lq, h, d, generator=gen, device="cuda")
    k = torch.randn(b, lk, hk, d, generator=gen, device="cuda")
    v = torch.randn(b, lk, hk, dv or d, generator=gen, device="cuda")
    return [t.to(dtype).transpose(1, 2) for t in (q, k, v)]


def bound_of(q, k, v, scale=None):
    """One bound for all rows, from the largest values that any of them sees."""
    u, d = UNIT[q.dtype], q.shape[-1]
    scale = d ** -0.5 if scale is None else abs(scale)
    k, v = torch.nan_to_num(k.double(), 0, 0, 0), torch.nan_to_num(v.double(), 0, 0, 0)
    k = k.abs().repeat_interleave(q.shape[1] // k.shape[1], 1)
    reach = scale * (q.double().abs() @ k.transpose(-1, -2)).max().item()
    return v.abs().max().item() * (4 * u + 2.0**-24 * (2 * d * reach + 2 * k.shape[2] + 8))


def check(out, q, k, v, window, sinks, scale=None):
    ref = bio_oracle.window_attention(q, k, v, window, sinks, scale)
    got = out.double().cpu()
    assert got.shape == ref.shape and out.dtype == q.dtype
    err = (got - ref).abs().max().item()
    assert err <= bound_of(q, k, v, scale), f"{err} > {bound_of(q, k, v, scale)}"
    if q.dtype != torch.float32 and ref.norm() > 0:
        assert ((got - ref).norm() / ref.norm()).item() <= 2 * UNIT[q.dtype]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,h,hk,lq,lk,d,window,sinks", [
    (1, 1, 1, 1, 1, 64, 1, 0),
    (2, 4, 2, 1, 300, 128, 100, 4),      # one token behind a cache
    (1, 2, 1, 7, 7, 64, 3, 1),
    (1, 2, 2, 127, 127, 128, 16, 4),
    (1, 2, 1, 128, 128, 64, 64, 0),
    (1, 2, 1, 129, 129, 128, 128, 2),
    (2, 3, 1, 255, 300, 64, 129, 5),
    (1, 2, 1, 257, 257, 128, 1, 0),      # each token sees itself
    (1, 4, 2, 400, 400, 128, 1000, 0),   # plain causal
    (1, 2, 1, 520, 1100, 64, 257, 130),  # more sinks than a block
    (1, 2, 1, 300, 900, 128, 64, 700),   # the sinks reach into the window
    (1, 8, 1, 333, 333, 256, 100, 4),
    (1, 4, 2, 200, 260, 72, 50, 3),
    (1, 2, 1, 190, 190, 96, 31, 9),
    (1, 2, 1, 140, 140, 8, 20, 1),
    (1, 2, 1, 70, 70, 33, 20, 1),
    (1, 2, 1, 70, 90, 200, 20, 1),
    (3, 2, 2, 40, 20, 64, 8, 2),         # more queries than keys: the first see nothing
    (1, 2, 1, 30, 0, 64, 8, 2),          # no key at all
    (1, 16, 2, 64, 640, 64, 256, 16),
])
def test_matches_the_oracle(b, h, hk, lq, lk, d, window, sinks, dtype):
    q, k, v = make(b, h, hk, lq, lk, d, dtype=dtype, seed=lq + d)
    out = bio.sliding_window_attention_batch_invariant(q, k, v, window, sinks)
    if lk == 0:
        assert torch.equal(out, torch.zeros_like(out))
        return
    check(out, q, k, v, window, sinks)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,dv", [(64, 128), (128, 64), (256, 64), (40, 256), (24, 17)])
def test_value_dim_of_its_own(d, dv, dtype):
    q, k, v = make(1, 4, 2, 150, 200, d, dv, dtype=dtype, seed=dv)
    check(bio.sliding_window_attention_batch_invariant(q, k, v, 64, 4), q, k, v, 64, 4)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", (64, 128, 256, 80))
@pytest.mark.parametrize("window,sinks", [(1, 0), (100, 0), (128, 4), (300, 140)])
def test_hidden_values_never_reach_a_row(window, sinks, d, dtype):
    """One key in the middle holds infinities and NaN: the rows that do not see
    it keep their exact bits, the others show it."""
    lk, bad = 700, 333
    q, k, v = make(1, 2, 1, lk, lk, d, dtype=dtype, seed=window)
    clean = bio.sliding_window_attention_batch_invariant(q, k, v, window, sinks)
    k, v = k.clone(), v.clone()
    k[:, :, bad, 0] = float("inf")
    v[:, :, bad, 1:] = float("nan")
    out = bio.sliding_window_attention_batch_invariant(q, k, v, window, sinks)
    i = torch.arange(lk, device="cuda")
    sees = (i >= bad) & ((i < bad + window) | (bad < sinks))
    hidden = ~sees
    err = (out[:, :, hidden].double() - clean[:, :, hidden].double()).abs().max().item()
    # finite, and the same values up to the order of the sums
    assert err <= 2 * bound_of(q, k, v)
    # a score of +inf shows up; one of -inf has weight 0 (and alone gives a zero row)
    shows = sees & (q[0, :, :, 0] > 0)
    assert torch.isnan(out[0][shows][:, 1:]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_extreme_scores(dtype):
    q, k, v = make(1, 4, 2, 300, 300, 64, dtype=dtype, seed=9, spread=100.0)
    q[:, 1] = 0
    check(bio.sliding_window_attention_batch_invariant(q, k, v, 90, 4), q, k, v, 90, 4)
    check(bio.sliding_window_attention_batch_invariant(q, k, v, 90, 4, scale=-0.02), q, k, v, 90, 4,
          -0.02)
    check(bio.sliding_window_attention_batch_invariant(q, k, v, 90, 4, scale=0.0), q, k, v, 90, 4,
          0.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", (64, 128, 256, 33))
def test_a_row_does_not_depend_on_the_batch(d, dtype):
    q, k, v = make(5, 4, 2, 300, 420, d, dtype=dtype, seed=d)
    full = bio.sliding_window_attention_batch_invariant(q, k, v, 130, 4)
    for b in range(5):
        alone = bio.sliding_window_attention_batch_invariant(q[b:b + 1], k[b:b + 1], v[b:b + 1],
                                                             130, 4)
        assert torch.equal(alone, full[b:b + 1])
    # heads are independent too
    pair = bio.sliding_window_attention_batch_invariant(q[:, 2:], k[:, 1:], v[:, 1:], 130, 4)
    assert torch.equal(pair, full[:, 2:])
    for _ in range(3):
        assert torch.equal(bio.sliding_window_attention_batch_invariant(q, k, v, 130, 4), full)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,h,hk,lq,lk,d,window,sinks", [
    (400, 2, 2, 3, 3, 64, 2, 0),         # one block each
    (260, 4, 2, 20, 150, 128, 130, 2),   # two
    (150, 8, 2, 70, 400, 64, 300, 40),   # three and four
    (40, 4, 1, 500, 500, 128, 200, 4),
    (160, 4, 2, 90, 200, 256, 100, 3),
    (3, 5, 1, 2500, 2500, 96, 700, 9),
])
def test_many_more_tiles_than_sms(b, h, hk, lq, lk, d, window, sinks, dtype):
    """Blocks that work through several tiles in a row: every sample has the bits
    that it has alone, and some are checked against the oracle."""
    q, k, v = make(b, h, hk, lq, lk, d, dtype=dtype, seed=b)
    full = bio.sliding_window_attention_batch_invariant(q, k, v, window, sinks)
    for i in sorted({0, 1, b // 2, b - 1}):
        alone = bio.sliding_window_attention_batch_invariant(
            q[i:i + 1], k[i:i + 1], v[i:i + 1], window, sinks)
        assert torch.equal(alone, full[i:i + 1])
    some = slice(b // 2, b // 2 + 1)
    rows = slice(max(0, lq - 300), lq)
    check(full[some][:, :, rows], q[some][:, :, rows], k[some], v[some], window, sinks)
    assert _lib.device_status() == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_leading_dims_strides_and_odd_offsets(dtype):
    q, k, v = make(6, 4, 2, 100, 100, 64, dtype=dtype)
    out = bio.sliding_window_attention_batch_invariant(q, k, v, 40, 4)
    lead = bio.sliding_window_attention_batch_invariant(
        q.reshape(2, 3, 4, 100, 64), k.reshape(2, 3, 2, 100, 64), v.reshape(2, 3, 2, 100, 64),
        40, 4)
    assert torch.equal(lead.reshape(6, 4, 100, 64), out)
    assert torch.equal(bio.sliding_window_attention_batch_invariant(
        q[0], k[0], v[0], 40, 4), out[0])
    fused = torch.zeros(6, 100, 8, 67, dtype=dtype, device="cuda")
    fused[:, :, :4, 3:] = q.transpose(1, 2)
    fused[:, :, 4:6, 3:] = k.transpose(1, 2)
    fused[:, :, 6:, 3:] = v.transpose(1, 2)
    f = fused[..., 3:].transpose(1, 2)
    assert torch.equal(bio.sliding_window_attention_batch_invariant(
        f[:, :4], f[:, 4:6], f[:, 6:], 40, 4), out)
    assert bio.sliding_window_attention_batch_invariant(q[:0], k[:0], v[:0], 4).shape == (
        0, 4, 100, 64)
    assert bio.sliding_window_attention_batch_invariant(q[:, :, :0], k, v, 4).shape == (
        6, 4, 0, 64)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", (64, 128, 256, 72))
@pytest.mark.parametrize("index", (torch.int32, torch.int64))
def test_packed_equals_dense(d, dtype, index):
    lens_q, lens_k = [1, 130, 0, 300, 5, 257, 20], [1, 130, 40, 500, 700, 257, 0]
    parts = [make(1, 4, 2, a, b, d, dtype=dtype, seed=a + b) for a, b in zip(lens_q, lens_k)]
    q, k, v = (torch.cat([p[i].transpose(1, 2) for p in parts], 1) for i in range(3))
    off = lambda x: torch.tensor([0, *x], device="cuda").cumsum(0).to(index)  # noqa: E731
    out = bio.varlen_sliding_window_attention_batch_invariant(q, k, v, off(lens_q), off(lens_k),
                                                              100, 4)
    for part, got in zip(parts, out.split(lens_q, 1)):
        if part[0].shape[2] == 0:
            continue
        want = bio.sliding_window_attention_batch_invariant(*part, 100, 4).transpose(1, 2)
        assert torch.equal(got, want)


def test_packed_neighbours_do_not_leak():
    """NaN in the next sequence's keys and values."""
    q, k, v = make(1, 2, 1, 300, 300, 64)
    q, k, v = (t.transpose(1, 2).contiguous() for t in (q, k, v))
    cu = torch.tensor([0, 100, 300], dtype=torch.int32, device="cuda")
    out = bio.varlen_sliding_window_attention_batch_invariant(q, k, v, cu, cu, 64, 2)
    k[:, 100:], v[:, 100:] = float("nan"), float("nan")
    got = bio.varlen_sliding_window_attention_batch_invariant(q, k, v, cu, cu, 64, 2)
    assert torch.equal(got[:, :100], out[:, :100])


def test_packed_bad_offsets_and_uncovered_tokens():
    q, k, v = (t.transpose(1, 2).contiguous() for t in make(1, 2, 1, 300, 300, 64))
    cu = torch.tensor([0, 100, 200], dtype=torch.int32, device="cuda")
    out = bio.varlen_sliding_window_attention_batch_invariant(q, k, v, cu, cu, 64, 2)
    assert torch.equal(out[:, 200:], torch.zeros_like(out[:, 200:]))
    assert _lib.device_status() == 0
    bad_k = torch.tensor([0, 100, 5000], dtype=torch.int32, device="cuda")
    got = bio.varlen_sliding_window_attention_batch_invariant(q, k, v, cu, bad_k, 64, 2)
    assert torch.equal(got[:, :100], out[:, :100])
    assert torch.equal(got[:, 100:], torch.zeros_like(got[:, 100:]))
    assert _lib.device_status() == _lib.BIO_DEV_INDEX
    _lib.clear_device_status()


def test_streams_and_graphs():
    q, k, v = make(2, 4, 2, 300, 300, 128)
    want = bio.sliding_window_attention_batch_invariant(q, k, v, 100, 4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = bio.sliding_window_attention_batch_invariant(q, k, v, 100, 4)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = bio.sliding_window_attention_batch_invariant(q, k, v, 100, 4)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held, want)


def one_token(d, heads, dtype, gen, step):
    """[1, heads, 1, d] whose batch and token strides are `heads * step`, off the
    16-byte borders that only a dimension of several elements has to keep."""
    x = torch.zeros(1, 1, heads, step, dtype=dtype, device="cuda")
    x[..., :d] = torch.randn(1, 1, heads, d, generator=gen, device="cuda").to(dtype)
    return x[..., :d].transpose(1, 2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", (1, 8, 33, 36, 64, 100, 250))
@pytest.mark.parametrize("h,step", [(1, 0), (3, 0), (1, 3), (1, 5)])
def test_one_token_of_any_stride(h, step, d, dtype):
    gen = torch.Generator(device="cuda").manual_seed(d + h)
    q, k, v = (one_token(d, n, dtype, gen, d + step) for n in (h, 1, 1))
    out = bio.sliding_window_attention_batch_invariant(q, k, v, 4)
    assert torch.equal(out, v.expand_as(out))  # one key: its value
    cu = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    packed = bio.varlen_sliding_window_attention_batch_invariant(
        *(t.transpose(1, 2) for t in (q, k, v)), cu, cu, 4)
    assert torch.equal(packed.transpose(1, 2), out)
    # the last token of a longer sequence, alone: strides of the whole
    q, k, v = make(1, h, 1, 9, 9, d, dtype=dtype, seed=d)
    whole = bio.sliding_window_attention_batch_invariant(q, k, v, 5, 1)
    last = bio.sliding_window_attention_batch_invariant(q[:, :, 8:], k, v, 5, 1)
    assert torch.equal(last, whole[:, :, 8:])
    first = bio.sliding_window_attention_batch_invariant(q[:, :, :1], k[:, :, :1], v[:, :, :1], 5, 1)
    assert torch.equal(first, whole[:, :, :1])
    assert _lib.device_status() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hk,d", [(1, 33), (2, 33), (2, 64), (4, 36)])
def test_no_key_with_any_stride(hk, d, dtype):
    q, k, v = make(2, 4, hk, 5, 0, d, dtype=dtype)
    for x in (k, k.contiguous()):
        out = bio.sliding_window_attention_batch_invariant(q, x, x, 4)
        assert torch.equal(out, torch.zeros_like(out))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", (64, 100, 256))
def test_keys_expanded_over_batch_and_heads(d, dtype):
    """One prefix under several prompts, or one head's keys under all of them: strides of 0."""
    q, _, _ = make(3, 4, 2, 70, 70, d, dtype=dtype)
    _, k, v = make(1, 4, 2, 70, 90, d, dtype=dtype, seed=1)
    want = bio.sliding_window_attention_batch_invariant(
        q, k.repeat(3, 1, 1, 1), v.repeat(3, 1, 1, 1), 40, 4)
    got = bio.sliding_window_attention_batch_invariant(
        q, k.expand(3, -1, -1, -1), v.expand(3, -1, -1, -1), 40, 4)
    assert torch.equal(got, want)
    k, v = k[:, :1], v[:, :1]
    want = bio.sliding_window_attention_batch_invariant(
        q[:1], k.repeat(1, 2, 1, 1), v.repeat(1, 2, 1, 1), 40, 4)
    got = bio.sliding_window_attention_batch_invariant(
        q[:1], k.expand(-1, 2, -1, -1), v.expand(-1, 2, -1, -1), 40, 4)
    assert torch.equal(got, want)
    same = q[:1, :, :1].expand(-1, -1, 70, -1)  # one query at every position
    got = bio.sliding_window_attention_batch_invariant(same, k, v, 40, 4)
    want = bio.sliding_window_attention_batch_invariant(same.contiguous(), k, v, 40, 4)
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", (64, 128, 256, 72))
@pytest.mark.parametrize("window,sinks", [(1, 0), (50, 4), (128, 0), (300, 140), (90, 700),
                                          (5000, 3)])
def test_chunks_equal_the_whole_prompt(d, window, sinks, dtype):
    """Chunks behind the tokens before them, cut anywhere, dense and packed."""
    n = 1000
    q, k, v = make(1, 6, 2, n, n, d, dtype=dtype, seed=window)
    whole = bio.sliding_window_attention_batch_invariant(q, k, v, window, sinks)
    cuts = [0, 1, 32, 97, 128, 129, 255, 500, 501, 777, n]
    for a, b in [*zip(cuts, cuts[1:]), (0, 501), (129, 777), (3, n)]:
        got = bio.sliding_window_attention_batch_invariant(
            q[:, :, a:b], k[:, :, :b], v[:, :, :b], window, sinks)
        assert torch.equal(got, whole[:, :, a:b]), (a, b)
    pairs = [(97, 255), (0, 33), (501, n)]
    cu_q, cu_k = ([0, *torch.tensor(x).cumsum(0).tolist()] for x in (
        [b - a for a, b in pairs], [b for _, b in pairs]))
    packed = bio.varlen_sliding_window_attention_batch_invariant(
        torch.cat([q[:, :, a:b] for a, b in pairs], 2).transpose(1, 2),
        torch.cat([k[:, :, :b] for _, b in pairs], 2).transpose(1, 2),
        torch.cat([v[:, :, :b] for _, b in pairs], 2).transpose(1, 2),
        torch.tensor(cu_q, dtype=torch.int32, device="cuda"),
        torch.tensor(cu_k, dtype=torch.int32, device="cuda"), window, sinks)
    for (a, b), got in zip(pairs, packed.split([b - a for a, b in pairs], 1)):
        assert torch.equal(got.transpose(1, 2), whole[:, :, a:b]), (a, b)


def test_rows_computed_again_hold_nobody_up():
    """Rows of 200000 visible keys that come out not finite take seconds to compute
    again: longer than the waits of a block's other warps, whose next sequences
    must not notice."""
    dtype, n = torch.bfloat16, 200000
    lens_q, lens_k = [32] + [2] * 400, [n] + [5] * 400
    gen = torch.Generator(device="cuda").manual_seed(4)
    q, k, v = (torch.randn(1, x, 1, 64, generator=gen, device="cuda").to(dtype)
               for x in (sum(lens_q), sum(lens_k), sum(lens_k)))
    off = lambda x: torch.tensor([0, *x], device="cuda").cumsum(0)  # noqa: E731
    cu = off(lens_q), off(lens_k)
    clean = bio.varlen_sliding_window_attention_batch_invariant(q, k, v, *cu, 2**31 - 1)
    v[:, 7, :, 3] = float("nan")
    out = bio.varlen_sliding_window_attention_batch_invariant(q, k, v, *cu, 2**31 - 1)
    assert _lib.device_status() == 0
    assert torch.equal(out[:, 32:], clean[:, 32:])
    assert torch.isnan(out[:, :32, :, 3]).all()
    rest = torch.arange(64, device="cuda") != 3
    # a mean of so many values is small beside them: within the weights' rounding of |v| <= 6
    err = (out[:, :32, :, rest].double() - clean[:, :32, :, rest].double()).abs().max().item()
    assert err <= 2 * 6 * (4 * UNIT[dtype] + 2.0**-24 * (2 * 64 * 50 + 2 * n + 8))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", (64, 128, 256, 72))
@pytest.mark.parametrize("window,sinks", [(1, 0), (100, 0), (128, 4), (300, 140), (5000, 0)])
@pytest.mark.parametrize("bads", [(333,), (0, 2, 128, 255, 256, 511), (699,),
                                  tuple(range(40, 60)) + tuple(range(300, 460))])
def test_hidden_values_do_not_change_a_bit(bads, window, sinks, d, dtype):
    """Keys with infinities and NaN: rows that see none of them have the bits that
    they have beside finite values, whole, in chunks and packed; rows that see one
    show it where the oracle does."""
    n = 700
    q, k, v = make(1, 6, 2, n, n, d, dtype=dtype, seed=window + d)
    clean = bio.sliding_window_attention_batch_invariant(q, k, v, window, sinks)
    k, v = k.clone(), v.clone()
    for x, bad in enumerate(bads):
        v[:, x % 2, bad, (5 * x) % d] = (float("nan"), float("inf"), -float("inf"))[x % 3]
        if x % 4 == 3:  # a NaN score, too
            k[:, x % 2, bad, 0] = float("nan")
    i, at = torch.arange(n, device="cuda")[:, None], torch.tensor(bads, device="cuda")
    sees = (i >= at) & ((i < at + window) | (at < sinks))
    head = torch.arange(len(bads), device="cuda") % 2
    out = bio.sliding_window_attention_batch_invariant(q, k, v, window, sinks)
    for hk in range(2):
        hidden = ~sees[:, head == hk].any(1)
        mine = slice(3 * hk, 3 * hk + 3)
        assert torch.equal(out[0, mine][:, hidden], clean[0, mine][:, hidden])
    ref = bio_oracle.window_attention(q, k, v, window, sinks)
    got = out.double().cpu()
    finite = torch.isfinite(ref)
    assert torch.equal(torch.isfinite(got), finite)
    assert torch.equal(got[~finite].nan_to_num(7.0), ref[~finite].nan_to_num(7.0))
    assert (got[finite] - ref[finite]).abs().max().item() <= bound_of(q, k, v)
    for a, b in [(0, 1), (1, 129), (129, 350), (350, n)]:
        part = bio.sliding_window_attention_batch_invariant(
            q[:, :, a:b], k[:, :, :b], v[:, :, :b], window, sinks)
        assert torch.equal(part.nan_to_num(7.0), out[:, :, a:b].nan_to_num(7.0)), (a, b)
    cu = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 60, 60 + n],
                                                                      [0, 60, 60 + n])]
    packed = bio.varlen_sliding_window_attention_batch_invariant(
        *(torch.cat([t[:, :, :60], t], 2).transpose(1, 2) for t in (q, k, v)), *cu, window, sinks)
    want = torch.cat([out[:, :, :60], out], 2).transpose(1, 2)
    assert torch.equal(packed.nan_to_num(7.0), want.nan_to_num(7.0))
    assert _lib.device_status() == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_hidden_values_beside_many_other_tiles(dtype):
    """Blocks that go through several tiles again, one of them with a NaN."""
    q, k, v = make(90, 4, 2, 300, 400, 128, dtype=dtype, seed=2)
    clean = bio.sliding_window_attention_batch_invariant(q, k, v, 130, 4)
    v = v.clone()
    v[7, 1, 350] = float("nan")
    v[50, 0, 9] = float("inf")
    out = bio.sliding_window_attention_batch_invariant(q, k, v, 130, 4)
    i = torch.arange(300, device="cuda") + 100
    keep = torch.ones(90, 4, 300, dtype=torch.bool, device="cuda")
    keep[7, 2:] = ~((i >= 350) & (i < 480))
    keep[50, :2] = ~((i >= 9) & (i < 139))
    assert torch.equal(out[keep], clean[keep])
    assert not torch.isfinite(out[~keep]).any()
    assert _lib.device_status() == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_small_weights_beside_a_large_one(dtype):
    """A sink that outweighs every other key by 2^25, and 300000 other keys that
    together weigh 0.6 % of it: none of them may be rounded away."""
    n, d = 300000, 64
    q, k, v = (torch.zeros(1, 1, x, d, dtype=dtype, device="cuda") for x in (3, n, n))
    q[..., 0], k[:, :, 0, 0], v[:, :, 1:] = 1, 17.75, 1
    out = bio.sliding_window_attention_batch_invariant(q, k, v, n, 0, scale=1.0)
    rest = torch.arange(n - 3, n, dtype=torch.float64)  # keys beside the sink
    ref = rest / (rest + torch.tensor(17.75, dtype=torch.float64).exp())
    # relative to their own sum: weights and output rounded (4 u), an fp16 weight of
    # 2^-18.6 kept to half of 2^-24 (2^-6), 18750 sums of 16 keys (2^-9)
    err = ((out.double().cpu() - ref[None, None, :, None]) / ref.max()).abs().max().item()
    assert err <= 4 * UNIT[dtype] + 2.0**-6 + 2.0**-9
