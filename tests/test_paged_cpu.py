"""CPU checks of the paged cache and the sliding-window attention: what they
refuse before anything is launched, the argument structs, the workspace sizes,
and the 64-bit oracle against the dense one.  No GPU is needed."""

from __future__ import annotations

import ctypes

import pytest
import torch

import batch_invariant_ops as bio
from batch_invariant_ops import _lib, paged
from oracle import bio_oracle

ADDED_NAMES = (
    "sliding_window_attention_batch_invariant", "varlen_sliding_window_attention_batch_invariant",
    "paged_attention_decode_batch_invariant", "PagedKVCache", "paged_kv_append", "paged_kv_extend",
    "paged_kv_fork", "paged_kv_free", "paged_kv_evict", "paged_kv_compact",
)


def test_names_are_exported():
    for name in ADDED_NAMES:
        assert hasattr(bio, name) and name in bio.__all__, name


def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def pool(*lead, pages=4, heads=2, page=8, d=16, dtype=torch.float32):
    return torch.zeros(*lead, pages, heads, page, d, dtype=dtype)


DECODE = dict(query=torch.zeros(3, 4, 16), key_pages=pool(), value_pages=pool(),
              page_table=i32(3, 2), seq_lens=i32(3))


@pytest.mark.parametrize("change,error", [
    (dict(query=torch.zeros(3, 64)), ValueError),
    (dict(query=torch.zeros(3, 3, 16)), ValueError),              # heads not a multiple
    (dict(query=torch.zeros(3, 4, 8)), ValueError),               # head dim
    (dict(query=torch.zeros(3, 4, 16, dtype=torch.float16)), ValueError),
    (dict(query=torch.zeros(2, 4, 16)), ValueError),              # rows of the table
    (dict(key_pages=pool()[0]), ValueError),
    (dict(value_pages=pool(pages=5)), ValueError),
    (dict(key_pages=pool(d=257), value_pages=pool(d=257), query=torch.zeros(3, 4, 257)),
     ValueError),
    (dict(key_pages=pool().double(), value_pages=pool().double(),
          query=torch.zeros(3, 4, 16).double()), ValueError),
    (dict(key_pages=pool(d=8, page=16).transpose(2, 3), value_pages=pool(page=8, d=16)),
     ValueError),                                                  # last dim not contiguous
    (dict(page_table=torch.zeros(3, 2, dtype=torch.int64)), ValueError),
    (dict(page_table=i32(2, 3).t()), ValueError),
    (dict(page_table=i32(1, 2).expand(3, 2)), ValueError),         # overlapping rows
    (dict(seq_lens=torch.zeros(3, dtype=torch.int64)), ValueError),
    (dict(seq_lens=i32(4)), ValueError),
    (dict(window=0), ValueError),
    (dict(window=4, sinks=-1), ValueError),
    (dict(rows=i32(2)), ValueError),
    (dict(rows=torch.zeros(3, dtype=torch.int64)), ValueError),
    (dict(), AssertionError),                                      # CPU tensors
])
def test_decode_refuses(change, error):
    args = {**DECODE, **change}
    keyword = {k: args.pop(k) for k in ("window", "sinks", "rows") if k in args}
    with pytest.raises(error):
        bio.paged_attention_decode_batch_invariant(*args.values(), **keyword)


APPEND = dict(key_pages=pool(), value_pages=pool(), key=torch.zeros(5, 2, 16),
              value=torch.zeros(5, 2, 16), page_table=i32(3, 2), rows=i32(5), positions=i32(5))


@pytest.mark.parametrize("change,error", [
    (dict(key=torch.zeros(5, 32)), ValueError),
    (dict(key=torch.zeros(5, 1, 16)), ValueError),
    (dict(value=torch.zeros(4, 2, 16)), ValueError),
    (dict(key=torch.zeros(5, 2, 16, dtype=torch.bfloat16)), ValueError),
    (dict(rows=i32(4)), ValueError),
    (dict(positions=torch.zeros(5, dtype=torch.int64)), ValueError),
    (dict(), AssertionError),
])
def test_append_refuses(change, error):
    with pytest.raises(error):
        bio.paged_kv_append(**{**APPEND, **change})


BOOK = dict(page_table=i32(3, 2), seq_lens=i32(3), ref_counts=i32(4))


@pytest.mark.parametrize("change,error", [
    (dict(rows=i32(2)), ValueError),                               # new_lens longer
    (dict(page_size=0), ValueError),
    (dict(ref_counts=torch.zeros(4)), ValueError),
    (dict(ref_counts=i32(2, 2)), ValueError),
    (dict(seq_lens=i32(6)[::2]), ValueError),                      # updated in place: no copies
    (dict(), AssertionError),
])
def test_extend_refuses(change, error):
    with pytest.raises(error):
        bio.paged_kv_extend(**{**BOOK, "rows": i32(3), "new_lens": i32(3), "page_size": 8,
                               **change})


@pytest.mark.parametrize("change,error", [
    (dict(window=0), ValueError), (dict(sinks=-1), ValueError), (dict(page_size=0), ValueError),
    (dict(rows=torch.zeros(2)), ValueError), (dict(), AssertionError),
])
def test_evict_refuses(change, error):
    with pytest.raises(error):
        bio.paged_kv_evict(**{**BOOK, "rows": i32(2), "window": 4, "sinks": 0, "page_size": 8,
                              **change})


def test_free_refuses():
    with pytest.raises(ValueError):
        bio.paged_kv_free(**BOOK, rows=torch.zeros(1))
    with pytest.raises(AssertionError):
        bio.paged_kv_free(**BOOK, rows=i32(1))


@pytest.mark.parametrize("change,error", [
    (dict(key_pages=pool()), ValueError),                          # needs the layer dimension
    (dict(ref_counts=i32(5)), ValueError),
    (dict(src=i32(2)), ValueError),
    (dict(), AssertionError),
])
def test_fork_refuses(change, error):
    with pytest.raises(error):
        bio.paged_kv_fork(**{**BOOK, "key_pages": pool(2), "value_pages": pool(2), "src": i32(1),
                             "dst": i32(1), **change})


@pytest.mark.parametrize("change,error", [
    (dict(out_key_pages=pool(3, pages=2)), ValueError),            # layers
    (dict(out_key_pages=pool(2, pages=2, page=4), out_value_pages=pool(2, pages=2, page=4)),
     ValueError),
    (dict(out_key_pages=pool(2, pages=2, dtype=torch.float16),
          out_value_pages=pool(2, pages=2, dtype=torch.float16)), ValueError),
    (dict(out_page_table=i32(3, 3)), ValueError),
    (dict(out_ref_counts=i32(4)), ValueError),
    (dict(), AssertionError),
])
def test_compact_refuses(change, error):
    with pytest.raises(error):
        bio.paged_kv_compact(**{
            "key_pages": pool(2), "value_pages": pool(2), "page_table": i32(3, 2),
            "ref_counts": i32(4), "out_key_pages": pool(2, pages=2),
            "out_value_pages": pool(2, pages=2), "out_page_table": i32(3, 2),
            "out_ref_counts": i32(2), **change})


def test_cache_refuses_empty_sizes():
    for bad in (dict(layers=0), dict(pages=0), dict(page_size=0), dict(rows=0)):
        with pytest.raises(ValueError):
            bio.PagedKVCache(**{"layers": 1, "pages": 1, "page_size": 1, "kv_heads": 1,
                                "head_dim": 8, "rows": 1, "max_tokens": 1, "device": "cpu", **bad})


QKV = dict(query=torch.zeros(2, 4, 5, 16), key=torch.zeros(2, 2, 9, 16),
           value=torch.zeros(2, 2, 9, 8), window=4)


@pytest.mark.parametrize("change,error", [
    (dict(query=torch.zeros(5, 16)), ValueError),
    (dict(query=torch.zeros(3, 4, 5, 16)), ValueError),
    (dict(query=torch.zeros(2, 3, 5, 16)), ValueError),
    (dict(key=torch.zeros(2, 2, 9, 8)), ValueError),
    (dict(value=torch.zeros(2, 2, 8, 8)), ValueError),
    (dict(value=torch.zeros(2, 2, 9, 8, dtype=torch.float16)), ValueError),
    (dict(value=torch.zeros(2, 2, 9, 300)), ValueError),
    (dict(window=0), ValueError),
    (dict(sinks=-1), ValueError),
    (dict(query=torch.zeros(2, 4, 5, 16).long(), key=torch.zeros(2, 2, 9, 16).long(),
          value=torch.zeros(2, 2, 9, 8).long()), ValueError),
    (dict(), AssertionError),
])
def test_window_refuses(change, error):
    with pytest.raises(error):
        bio.sliding_window_attention_batch_invariant(**{**QKV, **change})


PACKED = dict(query=torch.zeros(1, 7, 4, 16), key=torch.zeros(1, 9, 2, 16),
              value=torch.zeros(1, 9, 2, 8), cumulative_seqlen_q=i32(3),
              cumulative_seqlen_kv=i32(3), window=4)


@pytest.mark.parametrize("change,error", [
    (dict(query=torch.zeros(2, 7, 4, 16)), ValueError),
    (dict(cumulative_seqlen_q=i32(2)), ValueError),
    (dict(cumulative_seqlen_q=i32(3).float(), ), ValueError),
    (dict(cumulative_seqlen_q=i32(0), cumulative_seqlen_kv=i32(0)), ValueError),
    (dict(window=-3), ValueError),
    (dict(), AssertionError),
])
def test_packed_window_refuses(change, error):
    with pytest.raises(error):
        bio.varlen_sliding_window_attention_batch_invariant(**{**PACKED, **change})


def test_argument_structs_have_the_c_sizes():
    # bio_paged_attn_args: 2 int32, 4 pointers, 15 int64, pointer, 3 int64, 2 pointers, 2 int64,
    # 2 int32, float, int32
    assert paged._ATTN_ARGS.size == 8 * (1 + 4 + 15 + 1 + 3 + 2 + 2 + 2)
    # bio_kv_pool: 2 int32, 2 pointers, 14 int64; bio_kv_table: pointer, 3 int64, 2 pointers,
    # 2 int64, 2 int32
    assert paged._POOL.size == 8 * (1 + 2 + 14)
    assert paged._TABLE.size == 8 * (1 + 3 + 2 + 2 + 1)


def test_window_arguments_land_in_the_fields_of_the_c_struct():
    from batch_invariant_ops import _attn

    t = torch.zeros(2, 3, 4, 8)
    cu = torch.zeros(6, dtype=torch.int64)
    strides = tuple(range(11, 23))
    raw = _attn._window_args(t, t[:1], t[1:], t[1:, 1:], strides, 2, 6, 3, 4, 5, 8, 7, 0.25, cu,
                             cu[1:])
    a = _attn._AttnArgs.from_buffer_copy(raw)
    assert [getattr(a, n) for n in ("q", "k", "v", "o")] == [
        x.data_ptr() for x in (t, t[:1], t[1:], t[1:, 1:])]
    assert tuple(getattr(a, f"{n}_{s}") for n in "qkvo" for s in ("sb", "sh", "st")) == strides
    assert (a.dtype, a.batch, a.heads, a.kv_heads, a.lq, a.lk, a.d, a.dv, a.scale) == (
        0, 2, 6, 3, 4, 5, 8, 7, 0.25)
    assert (a.causal, a.mask_kind, a.mask, a.workspace) == (0, 0, None, None)
    assert (a.cu_q, a.cu_k, a.cu_is64, a.nseq) == (cu.data_ptr(), cu[1:].data_ptr(), 1, 5)


def attention_args(**change):
    a = dict(dtype=2, device=0, batch=4, heads=8, kv_heads=2, pages=64, page_size=16, rows=4,
             width=8, window=0, sinks=0, d=64, dv=64)
    a.update(change)
    return paged._ATTN_ARGS.pack(
        a["dtype"], a["device"], 0, 0, 0, 0, *([0] * 10), a["batch"], a["heads"], a["kv_heads"],
        a["pages"], a["page_size"], 0, a["width"], a["rows"], a["width"], 0, 0, a["window"],
        a["sinks"], a["d"], a["dv"], 1.0, 0)


def test_attention_workspace_is_a_function_of_the_sizes():
    need = _lib.load().bio_paged_attention_workspace
    assert need(attention_args(width=1)) == 0  # 16 tokens: one piece, nothing to join
    assert need(attention_args()) > 0          # 128 tokens
    more = need(attention_args(width=1024))
    assert more >= need(attention_args(width=512))  # longer rows have longer pieces
    # a window bounds what a row sees, whatever the table could hold
    assert need(attention_args(width=1024, window=40, sinks=4)) < need(attention_args(width=16))
    assert need(attention_args(batch=8)) == 2 * need(attention_args())


@pytest.mark.parametrize("change", [
    dict(heads=7), dict(kv_heads=0), dict(d=0), dict(d=257), dict(dv=257), dict(page_size=0),
    dict(window=-1), dict(sinks=-1), dict(batch=-1), dict(pages=-1), dict(width=1 << 40),
    dict(batch=1 << 40),
])
def test_c_entry_refuses(change):
    lib = _lib.load()
    assert lib.bio_paged_attention(attention_args(**change), None, 0, None) in (
        _lib.BIO_ERR_SHAPE, _lib.BIO_ERR_ARG)
    assert lib.bio_paged_attention_workspace(attention_args(**change)) == 0


def test_c_entries_refuse_null_structs():
    lib = _lib.load()
    assert lib.bio_paged_attention(None, None, 0, None) == _lib.BIO_ERR_ARG
    assert lib.bio_kv_append(None, None, None, 0, 0, None, 0, 0, None, None, 1, None) != 0
    assert lib.bio_kv_extend(None, None, None, 1, None, 0, None) == _lib.BIO_ERR_ARG
    assert lib.bio_kv_free(None, None, 1, None) == _lib.BIO_ERR_ARG
    assert lib.bio_kv_evict(None, None, 1, 4, 0, None) == _lib.BIO_ERR_ARG
    assert lib.bio_kv_fork(None, None, None, None, 1, None, 0, None) == _lib.BIO_ERR_ARG
    assert lib.bio_kv_compact(None, None, None, None, None, 0, None) == _lib.BIO_ERR_ARG
    assert lib.bio_attention_window(None, 4, 0, None) == _lib.BIO_ERR_ARG
    assert lib.bio_attention_window_varlen(None, 4, 0, None) == _lib.BIO_ERR_ARG
    assert lib.bio_kv_workspace(-1, 0) == 0


def test_window_entry_refuses_masks_and_bad_windows():
    from batch_invariant_ops._attn import _AttnArgs

    lib = _lib.load()
    for window, sinks, change in ((0, 0, {}), (1 << 40, 0, {}), (4, -1, {}), (4, 0, {"causal": 1}),
                                  (4, 0, {"mask_kind": 1}), (4, 0, {"d": 257}),
                                  (4, 0, {"heads": 3})):
        a = _AttnArgs()
        a.dtype, a.batch, a.heads, a.kv_heads, a.lq, a.lk, a.d, a.dv = 2, 1, 2, 2, 4, 4, 64, 64
        for key, value in change.items():
            setattr(a, key, value)
        assert lib.bio_attention_window(ctypes.byref(a), window, sinks, None) in (
            _lib.BIO_ERR_ARG, _lib.BIO_ERR_SHAPE)


@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (3, 2), (100, 1)])
def test_oracles_agree_with_dense_attention(window, sinks):
    gen = torch.Generator().manual_seed(3)
    lq, lk, d = 6, 11, 8
    q = torch.randn(2, 4, lq, d, generator=gen, dtype=torch.float64)
    k = torch.randn(2, 2, lk, d, generator=gen, dtype=torch.float64)
    v = torch.randn(2, 2, lk, d, generator=gen, dtype=torch.float64)
    i, j = torch.arange(lq)[:, None] + lk - lq, torch.arange(lk)
    keep = j <= i
    if window is not None:
        keep &= (j > i - window) | (j < sinks)
    want = torch.nn.functional.scaled_dot_product_attention(
        q, k.repeat_interleave(2, 1), v.repeat_interleave(2, 1), attn_mask=keep)
    if window is not None:
        got = bio_oracle.window_attention(q, k, v, window, sinks)
        assert torch.allclose(got, want, rtol=1e-12, atol=1e-12)
    # the last query, with the keys in pages of 3 tokens in reverse order
    page, pages = 3, 4
    table = torch.tensor([[3, 2, 1, 0], [7, 6, 5, 4]], dtype=torch.int32)
    kp, vp = torch.full((8, 2, page, d), float("nan")), torch.full((8, 2, page, d), float("nan"))
    kp, vp = kp.double(), vp.double()
    for b in range(2):
        for t in range(lk):
            kp[table[b, t // page], :, t % page] = k[b, :, t]
            vp[table[b, t // page], :, t % page] = v[b, :, t]
    got = bio_oracle.paged_attention(q[:, :, -1], kp, vp, table, torch.tensor([lk, lk]), window,
                                     sinks)
    assert torch.allclose(got, want[:, :, -1], rtol=1e-12, atol=1e-12)


def test_oracle_page_book():
    book = bio_oracle.PageBook(torch.full((3, 3), -1), torch.zeros(3, dtype=torch.int64),
                               torch.zeros(5, dtype=torch.int64), 4)
    book.extend([1, 0], [6, 3])
    assert book.table == [[2, -1, -1], [0, 1, -1], [-1, -1, -1]] and book.lens == [3, 6, 0]
    assert book.fork([1], [2]) == [(1, 3, 2)]
    assert book.table[2] == [0, 3, -1] and book.refs == [2, 1, 1, 1, 0]
    book.evict([2], 2, 0)
    assert book.table[2] == [-1, 3, -1] and book.refs == [1, 1, 1, 1, 0]
    book.free([0])
    assert book.compact(3) == [0, 1, 3] and book.refs == [1, 1, 1]
    assert book.table == [[-1, -1, -1], [0, 1, -1], [-1, 2, -1]]


def test_items_leave_room_for_a_step_past_the_last():
    """Pieces of all heads are walked in steps of some thousand with 32-bit numbers:
    2^31 of them, less one step, are refused."""
    need = _lib.load().bio_paged_attention_workspace
    sizes = dict(heads=1, kv_heads=1, width=64, d=4, dv=4)  # 1024 tokens: 32 pieces a row
    pieces = need(attention_args(batch=1, rows=1, **sizes)) // (4 * 4 + 8)
    assert pieces == 32
    most = (2**31 - 1) // pieces
    assert need(attention_args(batch=most - 4096, **sizes)) == (most - 4096) * pieces * 24
    for batch in (most - 10, most):
        assert need(attention_args(batch=batch, **sizes)) == 0
        assert _lib.load().bio_paged_attention(attention_args(batch=batch, **sizes), None, 0,
                                               None) == _lib.BIO_ERR_SHAPE
