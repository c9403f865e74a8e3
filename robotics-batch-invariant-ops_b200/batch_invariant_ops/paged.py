"""A paged key/value cache on the device and the operators that work on it.

Pages hold ``page_size`` tokens of every KV head: ``key_pages`` and
``value_pages`` are ``[pages, kv_heads, page_size, head_dim]`` for one layer,
with a leading layer dimension where one table serves every layer.  Token ``t``
of row ``r`` lives in page ``page_table[r, t // page_size]``, slot
``t % page_size``; the table is int32 with -1 for "no page", ``seq_lens`` int32
``[rows]`` and ``ref_counts`` int32 ``[pages]`` (how many table entries hold the
page, 0 = free).  All of it lives and changes on the device: no call here
synchronises with the host, so every one of them can be captured in a CUDA
graph.  Pages are handed out lowest number first, in the order of the request,
so the bookkeeping is a function of its inputs alone.

``PagedKVCache`` holds these tensors and calls the functions below.  The
reference keeps no cache between calls (its attention,
batch_invariant_ops.py:1148-1344, takes whole keys and values); these
operators are additions.

Errors: shapes, types and devices raise ``ValueError`` (CPU tensors
``AssertionError``) before anything is launched; rows, lengths and page numbers
are only known to the device, which skips what is out of range and sets
``BIO_DEV_INDEX`` in ``_lib.device_status()``; a pool without free pages sets
``BIO_DEV_PAGES``.
"""

from __future__ import annotations

import functools
import math
import struct
from typing import NamedTuple

import torch

from . import _lib, tracing
from ._attn import geometry as _geo

MAX_HEAD_DIM = 256

# Layouts of the C structs (native alignment), packed into bytes per call
_ATTN_ARGS = struct.Struct("@ii4P2q3q3q2q3q2qP3qPP2qiifi")  # bio_paged_attn_args
_POOL = struct.Struct("@iiPP4q4q4q2q")  # bio_kv_pool
_TABLE = struct.Struct("@PqqqPPqqii")  # bio_kv_table


# A call costs about as much on the host as its kernels take at the small end (a
# single token), so what follows from shapes, strides, types and devices alone --
# the checks and the integers of the C structs -- is worked out once per geometry.
# Nothing here depends on an address or on what a tensor holds.
_plan = functools.lru_cache(maxsize=1024)


class _Geometry(NamedTuple):
    shape: torch.Size
    stride: tuple
    dtype: torch.dtype
    device: int  # -1 for the CPU

    @property
    def ndim(self) -> int:
        return len(self.shape)

    def contiguous(self) -> bool:
        """For one dimension."""
        return self.shape[0] < 2 or self.stride[0] == 1


def _geometries(*geos) -> list:
    return [None if g is None else _Geometry(*g) for g in geos]


def _on_one_device(first: _Geometry, *others: _Geometry) -> None:
    assert first.device >= 0, "Input must be a CUDA tensor"
    for g in others:
        if g.device != first.device:
            raise ValueError("all tensors must be on the same CUDA device")


def _check_index(g: _Geometry, what: str) -> None:
    """A 1-D int32 tensor; ``_in_place`` makes it one the kernels can read."""
    if g.dtype != torch.int32 or g.ndim != 1:
        raise ValueError(f"{what} must be a 1-D int32 tensor")


def _in_place(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 else t.contiguous()


def _check_pages(key_pages: _Geometry, value_pages: _Geometry, ndim: int) -> None:
    if key_pages.ndim != ndim or value_pages.ndim != ndim:
        raise ValueError(f"key_pages and value_pages must have {ndim} dimensions")
    if key_pages.shape[:-1] != value_pages.shape[:-1]:
        raise ValueError("key_pages and value_pages must agree in all but the last dimension")
    if key_pages.dtype != value_pages.dtype or key_pages.dtype not in _lib.DTYPE_CODE:
        raise ValueError("key_pages and value_pages must share float32, float16 or bfloat16")
    if 0 in key_pages.shape[-3:] or value_pages.shape[-1] == 0:
        raise ValueError("pages need at least one head, one slot and one column")
    if key_pages.stride[-1] != 1 or value_pages.stride[-1] != 1:
        raise ValueError("pages must be contiguous in their last dimension")


def _check_table(page_table: _Geometry, seq_lens=None, ref_counts=None, pages=None) -> None:
    if page_table.ndim != 2 or page_table.dtype != torch.int32:
        raise ValueError("page_table must be a 2-D int32 tensor")
    if page_table.shape[1] > 1 and page_table.stride[1] != 1:
        raise ValueError("page_table must be contiguous in its last dimension")
    if page_table.shape[0] > 1 and page_table.stride[0] < page_table.shape[1]:
        raise ValueError("the rows of page_table must not overlap")
    if seq_lens is not None and (seq_lens.dtype != torch.int32
                                 or seq_lens.shape != page_table.shape[:1]
                                 or not seq_lens.contiguous()):
        raise ValueError("seq_lens must be a contiguous int32 tensor with one entry per table row")
    if ref_counts is not None and (ref_counts.dtype != torch.int32 or ref_counts.ndim != 1
                                   or not ref_counts.contiguous()
                                   or (pages is not None and ref_counts.shape[0] != pages)):
        raise ValueError("ref_counts must be a contiguous int32 tensor with one entry per page")


def _pool_ints(key_pages: _Geometry, value_pages: _Geometry) -> tuple:
    ks, vs, shape = tuple(key_pages.stride), tuple(value_pages.stride), tuple(key_pages.shape)
    if key_pages.ndim == 4:
        ks, vs, shape = (0, *ks), (0, *vs), (1, *shape)
    return ((_lib.DTYPE_CODE[key_pages.dtype], key_pages.device),
            (*shape[:4], *ks[:4], *vs[:4], shape[4], value_pages.shape[-1]))


def _pool_args(ints: tuple, key_pages: torch.Tensor, value_pages: torch.Tensor) -> bytes:
    return _POOL.pack(*ints[0], key_pages.data_ptr(), value_pages.data_ptr(), *ints[1])


def _table_ints(page_table: _Geometry, pages: int, page_size: int) -> tuple:
    return ((page_table.stride[0], *page_table.shape), (pages, page_size, page_table.device, 0))


def _table_args(ints: tuple, page_table: torch.Tensor, seq_lens=None, ref_counts=None) -> bytes:
    return _TABLE.pack(page_table.data_ptr(), *ints[0],
                       0 if seq_lens is None else seq_lens.data_ptr(),
                       0 if ref_counts is None else ref_counts.data_ptr(), *ints[1])


def _workspace(nbytes: int, device: torch.device) -> torch.Tensor:
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


@_plan
def _kv_workspace(n: int, pages: int) -> int:
    return _lib.load().bio_kv_workspace(n, pages)


def _call(name: str, note, *args) -> None:
    """One call of the library, recorded when launches are (``note()`` says as what)."""
    pushed = tracing.note(*note()) if note is not None and tracing.active() else False
    try:
        _lib.check(getattr(_lib.load(), name)(*args), name)
    finally:
        tracing.done(pushed)


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
@_plan
def _decode_plan(query, key_pages, value_pages, page_table, seq_lens, rows):
    query, key_pages, value_pages, page_table, seq_lens, rows = _geometries(
        query, key_pages, value_pages, page_table, seq_lens, rows)
    if query.ndim != 3:
        raise ValueError("query must be [batch, heads, head_dim]")
    _check_pages(key_pages, value_pages, 4)
    _check_table(page_table, seq_lens)
    batch, heads, d = query.shape
    pages, kv_heads, page_size, kd = key_pages.shape
    dv = value_pages.shape[3]
    if query.dtype != key_pages.dtype:
        raise ValueError("query and pages must have the same dtype")
    if d != kd:
        raise ValueError("query and key head dimensions must match")
    if d > MAX_HEAD_DIM or dv > MAX_HEAD_DIM:
        raise ValueError(f"head dimensions above {MAX_HEAD_DIM} are not supported (got {d}, {dv})")
    if heads == 0 or heads % kv_heads:
        raise ValueError("query heads must be divisible by key/value heads")
    if rows is not None:
        _check_index(rows, "rows")
        if rows.shape[0] != batch:
            raise ValueError("rows must have one entry per query")
    elif page_table.shape[0] != batch:
        raise ValueError("page_table must have one row per query (or give rows)")
    _on_one_device(query, key_pages, value_pages, page_table, seq_lens,
                   *([] if rows is None else [rows]))
    return ((_lib.DTYPE_CODE[query.dtype], query.device),
            (*key_pages.stride[:3], *value_pages.stride[:3], heads * dv, dv, batch, heads,
             kv_heads, pages, page_size), (page_table.stride[0], *page_table.shape),
            (d, dv), (batch, heads, dv), d ** -0.5)


def paged_attention_decode_batch_invariant(
    query: torch.Tensor,
    key_pages: torch.Tensor,
    value_pages: torch.Tensor,
    page_table: torch.Tensor,
    seq_lens: torch.Tensor,
    *,
    window: int | None = None,
    sinks: int = 0,
    scale: float | None = None,
    rows: torch.Tensor | None = None,
) -> torch.Tensor:
    """Attention of one new token per sequence over a paged cache.

    ``query [B, H, D]`` attends to the first ``seq_lens[r]`` tokens of table row
    ``r`` (its own key and value are already in the cache); query ``b`` belongs
    to row ``rows[b]``, or to row ``b`` without ``rows``.  With ``window``, only
    the last ``window`` tokens and the first ``sinks`` tokens are visible.
    Returns ``[B, H, Dv]``; rows of length 0 give zeros.  Slots beyond a row's
    length never reach the result, whatever they hold.

    A row's cache is cut into pieces whose size depends on its own length and
    the window alone, so its bits do not depend on the other rows of the call.
    """
    if window is not None and window < 1:
        raise ValueError("window must be at least 1")
    if sinks < 0:
        raise ValueError("sinks must not be negative")
    kind, shape, table, dims, out_shape, usual = _decode_plan(
        _geo(query), _geo(key_pages), _geo(value_pages), _geo(page_table), _geo(seq_lens),
        None if rows is None else _geo(rows))
    query = _in_place(query)
    out = query.new_empty(out_shape)
    if out_shape[0] == 0:
        return out
    if rows is not None:
        rows = _in_place(rows)
    qs = query.stride()
    args = _ATTN_ARGS.pack(
        *kind, query.data_ptr(), key_pages.data_ptr(), value_pages.data_ptr(), out.data_ptr(),
        qs[0], qs[1], *shape, page_table.data_ptr(), *table, seq_lens.data_ptr(),
        0 if rows is None else rows.data_ptr(),
        0 if window is None else min(window, 2147483647), min(sinks, 2147483647),
        *dims, usual if scale is None else scale, 0)
    nbytes = _lib.load().bio_paged_attention_workspace(args)
    workspace = _workspace(nbytes, out.device) if nbytes else None

    def note():
        batch, heads, dv = out_shape
        d, kv_heads, size = dims[0], shape[-3], query.element_size()
        most = table[2] * shape[-1]
        most = most if window is None else min(most, window + sinks)
        return ("paged_attention", f"bio_paged_attention [B={batch}, H={heads}/{kv_heads}, "
                f"tokens<={most}, D={d}/{dv}]", 2.0 * batch * heads * most * (d + dv),
                size * batch * (most * kv_heads * (d + dv) + heads * (d + dv)), size)

    _call("bio_paged_attention", note, args, workspace.data_ptr() if nbytes else None, nbytes,
          _lib.stream_of(out))
    return out


# ---------------------------------------------------------------------------
# pages
# ---------------------------------------------------------------------------
@_plan
def _append_plan(key_pages, value_pages, key, value, page_table, rows, positions):
    key_pages, value_pages, key, value, page_table, rows, positions = _geometries(
        key_pages, value_pages, key, value, page_table, rows, positions)
    _check_pages(key_pages, value_pages, 4)
    _check_table(page_table)
    if key.ndim != 3 or value.ndim != 3:
        raise ValueError("key and value must be [tokens, kv_heads, head_dim]")
    pages, kv_heads, page_size, d = key_pages.shape
    tokens = key.shape[0]
    if tuple(key.shape[1:]) != (kv_heads, d) or tuple(value.shape) != (
            tokens, kv_heads, value_pages.shape[3]):
        raise ValueError("key and value must match the heads and columns of the pages")
    if key.dtype != key_pages.dtype or value.dtype != key_pages.dtype:
        raise ValueError("key, value and pages must have the same dtype")
    _check_index(rows, "rows")
    _check_index(positions, "positions")
    if rows.shape[0] != tokens or positions.shape[0] != tokens:
        raise ValueError("rows and positions must have one entry per token")
    _on_one_device(key, value, key_pages, value_pages, page_table, rows, positions)
    return _pool_ints(key_pages, value_pages), _table_ints(page_table, pages, page_size)


def paged_kv_append(
    key_pages: torch.Tensor,
    value_pages: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    page_table: torch.Tensor,
    rows: torch.Tensor,
    positions: torch.Tensor,
) -> None:
    """Write new tokens into their pages (one layer, in place).

    Token ``t`` of ``key [T, kv_heads, D]`` and ``value [T, kv_heads, Dv]`` goes
    to position ``positions[t]`` of table row ``rows[t]`` (both int32); a negative
    position is skipped (padding).  Slices of a fused projection are read in
    place."""
    pool, table = _append_plan(_geo(key_pages), _geo(value_pages), _geo(key), _geo(value),
                               _geo(page_table), _geo(rows), _geo(positions))
    tokens = key.shape[0]
    if tokens == 0:
        return
    key, value, rows, positions = map(_in_place, (key, value, rows, positions))
    k_stride, v_stride = key.stride(), value.stride()
    _call("bio_kv_append",
          lambda: ("kv_append", f"bio_kv_append [T={tokens}, H={key.shape[1]}, D={key.shape[2]}]",
                   0, 2 * key.element_size() * (key.numel() + value.numel()), key.element_size()),
          _pool_args(pool, key_pages, value_pages), _table_args(table, page_table),
          key.data_ptr(), k_stride[0], k_stride[1], value.data_ptr(), v_stride[0], v_stride[1],
          rows.data_ptr(), positions.data_ptr(), tokens, _lib.stream_of(key))


@_plan
def _rows_plan(page_table, seq_lens, ref_counts, rows, new_lens, page_size):
    page_table, seq_lens, ref_counts, rows, new_lens = _geometries(
        page_table, seq_lens, ref_counts, rows, new_lens)
    _check_table(page_table, seq_lens, ref_counts)
    _check_index(rows, "rows")
    if new_lens is not None:
        _check_index(new_lens, "new_lens")
        if rows.shape[0] != new_lens.shape[0]:
            raise ValueError("rows and new_lens must have the same length")
    if page_size < 1:
        raise ValueError("page_size must be at least 1")
    _on_one_device(page_table, seq_lens, ref_counts, rows,
                   *([] if new_lens is None else [new_lens]))
    return _table_ints(page_table, ref_counts.shape[0], page_size)


def paged_kv_extend(
    page_table: torch.Tensor,
    seq_lens: torch.Tensor,
    ref_counts: torch.Tensor,
    rows: torch.Tensor,
    new_lens: torch.Tensor,
    page_size: int,
) -> None:
    """Grow row ``rows[i]`` to ``new_lens[i]`` tokens (int32, in place): the
    lowest free pages go to the rows in order.  A length that is not larger
    leaves its row as it is; when the pool runs out a row ends with the pages
    that it got (``BIO_DEV_PAGES``)."""
    table = _rows_plan(_geo(page_table), _geo(seq_lens), _geo(ref_counts), _geo(rows),
                       _geo(new_lens), int(page_size))
    rows, new_lens, n = _in_place(rows), _in_place(new_lens), rows.shape[0]
    nbytes = _kv_workspace(n, 0)
    workspace = _workspace(nbytes, page_table.device)
    _call("bio_kv_extend", None, _table_args(table, page_table, seq_lens, ref_counts),
          rows.data_ptr(), new_lens.data_ptr(), n, workspace.data_ptr(), nbytes,
          _lib.stream_of(page_table))


def paged_kv_free(
    page_table: torch.Tensor,
    seq_lens: torch.Tensor,
    ref_counts: torch.Tensor,
    rows: torch.Tensor,
) -> None:
    """Release every page of ``rows`` (int32, in place) and set their lengths to 0."""
    table = _rows_plan(_geo(page_table), _geo(seq_lens), _geo(ref_counts), _geo(rows), None, 1)
    rows = _in_place(rows)
    _call("bio_kv_free", None, _table_args(table, page_table, seq_lens, ref_counts),
          rows.data_ptr(), rows.shape[0], _lib.stream_of(page_table))


def paged_kv_evict(
    page_table: torch.Tensor,
    seq_lens: torch.Tensor,
    ref_counts: torch.Tensor,
    rows: torch.Tensor,
    window: int,
    sinks: int,
    page_size: int,
) -> None:
    """Release the pages of ``rows`` that no token within ``window`` or ``sinks``
    of the newest one lies in (int32, in place).  Lengths stay; attention with
    this window and these sinks gives the same bits before and after."""
    if window < 1:
        raise ValueError("window must be at least 1")
    if sinks < 0:
        raise ValueError("sinks must not be negative")
    table = _rows_plan(_geo(page_table), _geo(seq_lens), _geo(ref_counts), _geo(rows), None,
                       int(page_size))
    rows = _in_place(rows)
    _call("bio_kv_evict", None, _table_args(table, page_table, seq_lens, ref_counts),
          rows.data_ptr(), rows.shape[0], min(window, 2147483647), min(sinks, 2147483647),
          _lib.stream_of(page_table))



@_plan
def _fork_plan(key_pages, value_pages, page_table, seq_lens, ref_counts, src, dst):
    key_pages, value_pages, page_table, seq_lens, ref_counts, src, dst = _geometries(
        key_pages, value_pages, page_table, seq_lens, ref_counts, src, dst)
    _check_pages(key_pages, value_pages, 5)
    _, pages, _, page_size, _ = key_pages.shape
    _check_table(page_table, seq_lens, ref_counts, pages)
    _check_index(src, "src")
    _check_index(dst, "dst")
    if src.shape[0] != dst.shape[0]:
        raise ValueError("src and dst must have the same length")
    _on_one_device(key_pages, value_pages, page_table, seq_lens, ref_counts, src, dst)
    return _pool_ints(key_pages, value_pages), _table_ints(page_table, pages, page_size)


def paged_kv_fork(
    key_pages: torch.Tensor,
    value_pages: torch.Tensor,
    page_table: torch.Tensor,
    seq_lens: torch.Tensor,
    ref_counts: torch.Tensor,
    src: torch.Tensor,
    dst: torch.Tensor,
) -> None:
    """Branch row ``dst[i]`` off row ``src[i]`` (int32, in place, every layer of
    ``[layers, pages, kv_heads, page_size, D]``): what ``dst[i]`` held is
    released, whole pages are shared, the tokens of a last partial page are
    copied into the lowest free page, and the length is taken over.  No row may
    appear twice in ``dst`` or in both lists (``BIO_DEV_INDEX``, skipped)."""
    pool, table = _fork_plan(_geo(key_pages), _geo(value_pages), _geo(page_table), _geo(seq_lens),
                             _geo(ref_counts), _geo(src), _geo(dst))
    src, dst, n = _in_place(src), _in_place(dst), src.shape[0]
    nbytes = _kv_workspace(n, 0)
    workspace = _workspace(nbytes, key_pages.device)
    _call("bio_kv_fork",
          lambda: ("kv_fork", f"bio_kv_fork [n={n}, layers={key_pages.shape[0]}]", 0, 0,
                   key_pages.element_size()),
          _pool_args(pool, key_pages, value_pages),
          _table_args(table, page_table, seq_lens, ref_counts), src.data_ptr(), dst.data_ptr(), n,
          workspace.data_ptr(), nbytes, _lib.stream_of(key_pages))


@_plan
def _compact_plan(key_pages, value_pages, page_table, ref_counts, out_key_pages, out_value_pages,
                  out_page_table, out_ref_counts):
    (key_pages, value_pages, page_table, ref_counts, out_key_pages, out_value_pages,
     out_page_table, out_ref_counts) = _geometries(
         key_pages, value_pages, page_table, ref_counts, out_key_pages, out_value_pages,
         out_page_table, out_ref_counts)
    _check_pages(key_pages, value_pages, 5)
    _check_pages(out_key_pages, out_value_pages, 5)
    pages, out_pages = key_pages.shape[1], out_key_pages.shape[1]
    page_size = key_pages.shape[3]
    _check_table(page_table, None, ref_counts, pages)
    _check_table(out_page_table, None, out_ref_counts, out_pages)
    if key_pages.dtype != out_key_pages.dtype:
        raise ValueError("both pools must have the same dtype")
    for a, b in ((key_pages, out_key_pages), (value_pages, out_value_pages)):
        if (a.shape[0], *a.shape[2:]) != (b.shape[0], *b.shape[2:]):
            raise ValueError("the pools must agree in all but their number of pages")
    if page_table.shape != out_page_table.shape:
        raise ValueError("the page tables must have the same shape")
    _on_one_device(key_pages, value_pages, page_table, ref_counts, out_key_pages, out_value_pages,
                   out_page_table, out_ref_counts)
    return (_pool_ints(key_pages, value_pages), _table_ints(page_table, pages, page_size),
            _pool_ints(out_key_pages, out_value_pages),
            _table_ints(out_page_table, out_pages, page_size))


def paged_kv_compact(
    key_pages: torch.Tensor,
    value_pages: torch.Tensor,
    page_table: torch.Tensor,
    ref_counts: torch.Tensor,
    out_key_pages: torch.Tensor,
    out_value_pages: torch.Tensor,
    out_page_table: torch.Tensor,
    out_ref_counts: torch.Tensor,
) -> None:
    """Copy the pages in use to the front of another pool, in the order of
    their numbers, for every layer of ``[layers, pages, kv_heads, page_size,
    D]``, and write the table and the counts that go with them.  The pools may
    differ in their number of pages and must not overlap; pages that the other
    pool has no room for are dropped (``BIO_DEV_PAGES``)."""
    pool, table, out_pool, out_table = _compact_plan(
        _geo(key_pages), _geo(value_pages), _geo(page_table), _geo(ref_counts),
        _geo(out_key_pages), _geo(out_value_pages), _geo(out_page_table), _geo(out_ref_counts))
    nbytes = _kv_workspace(0, key_pages.shape[1])
    workspace = _workspace(nbytes, key_pages.device)
    _call("bio_kv_compact",
          lambda: ("kv_compact",
                   f"bio_kv_compact [pages={key_pages.shape[1]}, out={out_key_pages.shape[1]}]", 0,
                   2 * key_pages.element_size() * (out_key_pages.numel()
                                                   + out_value_pages.numel()),
                   key_pages.element_size()),
          _pool_args(pool, key_pages, value_pages),
          _table_args(table, page_table, None, ref_counts),
          _pool_args(out_pool, out_key_pages, out_value_pages),
          _table_args(out_table, out_page_table, None, out_ref_counts), workspace.data_ptr(),
          nbytes, _lib.stream_of(key_pages))


class PagedKVCache:
    """Key/value pages of ``layers`` layers under one page table.

    ``rows`` sequences of up to ``max_tokens`` tokens share ``pages`` pages.  A
    step of a served model: ``extend`` the rows by their new tokens once, then
    per layer ``append`` the new keys and values and ``attend`` with the new
    queries.  ``fork`` branches sequences (sampling, beams), ``evict`` drops what
    a sliding window has passed, ``free`` ends them, ``compact`` moves the pages
    in use into a pool of another size.  Row, length and position arguments are
    int32 tensors on the cache's device.
    """

    def __init__(self, layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int, *,
                 rows: int, max_tokens: int, value_dim: int | None = None,
                 dtype: torch.dtype = torch.bfloat16, device: torch.device | str = "cuda"):
        if min(layers, pages, page_size, kv_heads, head_dim, rows, max_tokens) < 1:
            raise ValueError("a cache needs at least one of everything")
        self.page_size = page_size
        shape = (layers, pages, kv_heads, page_size)
        self.key_pages = torch.empty(*shape, head_dim, dtype=dtype, device=device)
        self.value_pages = torch.empty(*shape, value_dim or head_dim, dtype=dtype, device=device)
        width = math.ceil(max_tokens / page_size)
        self.page_table = torch.full((rows, width), -1, dtype=torch.int32, device=device)
        self.seq_lens = torch.zeros(rows, dtype=torch.int32, device=device)
        self.ref_counts = torch.zeros(pages, dtype=torch.int32, device=device)

    def extend(self, rows: torch.Tensor, new_lens: torch.Tensor) -> None:
        paged_kv_extend(self.page_table, self.seq_lens, self.ref_counts, rows, new_lens,
                        self.page_size)

    def append(self, layer: int, key: torch.Tensor, value: torch.Tensor, rows: torch.Tensor,
               positions: torch.Tensor) -> None:
        paged_kv_append(self.key_pages[layer], self.value_pages[layer], key, value,
                        self.page_table, rows, positions)

    def attend(self, layer: int, query: torch.Tensor, *, rows: torch.Tensor | None = None,
               window: int | None = None, sinks: int = 0,
               scale: float | None = None) -> torch.Tensor:
        return paged_attention_decode_batch_invariant(
            query, self.key_pages[layer], self.value_pages[layer], self.page_table, self.seq_lens,
            window=window, sinks=sinks, scale=scale, rows=rows)

    def fork(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        paged_kv_fork(self.key_pages, self.value_pages, self.page_table, self.seq_lens,
                      self.ref_counts, src, dst)

    def free(self, rows: torch.Tensor) -> None:
        paged_kv_free(self.page_table, self.seq_lens, self.ref_counts, rows)

    def evict(self, rows: torch.Tensor, window: int, sinks: int = 0) -> None:
        paged_kv_evict(self.page_table, self.seq_lens, self.ref_counts, rows, window, sinks,
                       self.page_size)

    def compact(self, pages: int) -> "PagedKVCache":
        """A cache with a pool of ``pages`` pages that holds the same sequences."""
        if pages < 1:
            raise ValueError("a cache needs at least one page")
        layers, _, kv_heads, page_size, head_dim = self.key_pages.shape
        other = PagedKVCache.__new__(PagedKVCache)
        other.page_size = page_size
        other.key_pages = self.key_pages.new_empty(layers, pages, kv_heads, page_size, head_dim)
        other.value_pages = self.value_pages.new_empty(layers, pages, kv_heads, page_size,
                                                       self.value_pages.shape[4])
        other.page_table = torch.empty_like(self.page_table)
        other.seq_lens = self.seq_lens.clone()
        other.ref_counts = self.ref_counts.new_empty(pages)
        paged_kv_compact(self.key_pages, self.value_pages, self.page_table, self.ref_counts,
                         other.key_pages, other.value_pages, other.page_table, other.ref_counts)
        return other
