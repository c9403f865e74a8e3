"""Measured cases of the paged key/value cache and the attention operators that serve from it.

Five operators, each in its plain form (``own = False``: elementary torch
operations in 32 bits, rounded once) and as the calls of ``batch_invariant_ops``
(``own = True``):

``decode``   one new token per sequence against a paged cache
             (``paged_attention_decode_batch_invariant``);
``window``   prefill with a sliding window and sink tokens
             (``sliding_window_attention_batch_invariant``);
``append``   new keys and values into their pages (``paged_kv_append``);
``fork``     sequences that branch off others: whole pages shared, the last
             partial page copied (``paged_kv_fork``);
``compact``  the pages in use moved to the front of another pool
             (``paged_kv_compact``).

Pages are ``[pages, kv_heads, page_size, head_dim]`` (with a leading layer
dimension where one table serves every layer), the page table is int32
``[rows, width]`` with -1 for "no page", lengths are int32 ``[rows]``.
"""

import math
import os
import random
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}
_package = None


def _bio():
    """The framework's package, imported on the first call that needs it."""
    global _package
    if _package is None:
        root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                            "robotics-batch-invariant-ops_b200")
        if root not in sys.path:
            sys.path.insert(0, root)
        import batch_invariant_ops

        _package = batch_invariant_ops
    return _package


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # A control policy's next token: one robot, multi-query heads of 256, a
        # context of 304 prefix and 50 action tokens.  Latency counts.
        dict(name="decode one short", op="decode", dtype="bf16", batch=1, heads=8, kv_heads=1,
             dim=256, page=16, short=354, long=354, window=0, sinks=0),
        # A server's decode step: 128 requests of very different lengths.
        dict(name="decode ragged batch", op="decode", dtype="bf16", batch=128, heads=32,
             kv_heads=8, dim=128, page=16, short=1, long=8192, window=0, sinks=0),
        # Two long contexts: few rows, the work lies along the cache.
        dict(name="decode two long", op="decode", dtype="f16", batch=2, heads=32, kv_heads=8,
             dim=128, page=64, short=98305, long=131072, window=0, sinks=0),
        # A prompt of odd length in a small multi-query model.
        dict(name="window prompt", op="window", dtype="bf16", batch=1, heads=8, kv_heads=1,
             dim=256, queries=777, keys=777, window=256, sinks=4),
        # A chunk of a long prompt, behind 4096 tokens that are already cached.
        dict(name="window chunk", op="window", dtype="f16", batch=4, heads=32, kv_heads=8,
             dim=64, queries=512, keys=4608, window=2048, sinks=16),
        # A whole long prompt.
        dict(name="window long prompt", op="window", dtype="bf16", batch=1, heads=32, kv_heads=8,
             dim=128, queries=32768, keys=32768, window=1024, sinks=4),
        # One token of each of 64 requests, one layer: launch latency.
        dict(name="append one each", op="append", dtype="bf16", rows=64, tokens=1, kv_heads=8,
             dim=128, heads=32, page=16, before=1999),
        # The prompts of 16 requests, one layer.
        dict(name="append prompts", op="append", dtype="bf16", rows=16, tokens=2047, kv_heads=8,
             dim=128, heads=32, page=16, before=0),
        # Beam search over one sequence: eight beams branch off one prefix.
        dict(name="fork beams", op="fork", dtype="bf16", layers=18, sources=1, copies=8,
             kv_heads=1, dim=256, page=16, short=354, long=354),
        # Sampling eight continuations for each of 16 prompts.
        dict(name="fork prompts", op="fork", dtype="bf16", layers=32, sources=16, copies=8,
             kv_heads=8, dim=128, page=16, short=500, long=4001),
        # A small pool after some sequences have left it.
        dict(name="compact small pool", op="compact", dtype="f32", layers=2, pages=300, live=77,
             kv_heads=2, dim=64, page=16, rows=9),
        # A server's pool, moved into a smaller one.
        dict(name="compact large pool", op="compact", dtype="bf16", layers=16, pages=4096,
             live=2500, kv_heads=8, dim=128, page=16, rows=100),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["decode", "decode", "window", "window", "append", "fork", "compact"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    kv_heads = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 7, 8, 16])
    dim = rng.choice([64, 72, 80, 96, 128, 128, 256])
    page = rng.choice([8, 16, 16, 32, 64, 100])
    if op == "decode":
        batch = _log(rng, 1, 256)
        row = 2 * kv_heads * dim * _BYTES[dtype]
        most = max(64, min(131072, int(2.0e9 / (row * batch))))
        long = _log(rng, 1, most)
        short = rng.choice([1, max(1, long // 2), long])
        window = rng.choice([0, 0, _log(rng, 16, 8192)])
        return dict(op=op, dtype=dtype, batch=batch, heads=kv_heads * group, kv_heads=kv_heads,
                    dim=dim, page=page, short=short, long=long, window=window,
                    sinks=rng.choice([0, 1, 4, 20]) if window else 0)
    if op == "window":
        batch, queries = _log(rng, 1, 8), _log(rng, 1, 32768)
        window, sinks = _log(rng, 16, 4096), rng.choice([0, 1, 4, 4, 64])
        dtype = rng.choice(["bf16", "bf16", "bf16", "f16", "f16", "f16", "f32"])
        keys = queries + rng.choice([0, 0, _log(rng, 1, 8192)])
        # fp32 stays small: its products run on the CUDA cores
        most = 5.0e11 / (50 if dtype == "f32" else 1)
        cost = 4.0 * dim * batch * queries * min(keys, window + sinks)
        heads = kv_heads * group
        while heads * cost > most and queries > 16:
            queries, cost = queries // 2 + 1, cost / 2
        return dict(op=op, dtype=dtype, batch=batch, heads=heads, kv_heads=kv_heads, dim=dim,
                    queries=queries, keys=max(keys, queries), window=window, sinks=sinks)
    if op == "append":
        rows = _log(rng, 1, 256)
        return dict(op=op, dtype=dtype, rows=rows, tokens=_log(rng, 1, max(1, 32768 // rows)),
                    kv_heads=kv_heads, dim=dim, heads=kv_heads * group, page=page,
                    before=rng.choice([0, _log(rng, 1, 2000)]))
    if op == "fork":
        layers, sources, copies = _log(rng, 1, 32), _log(rng, 1, 64), _log(rng, 1, 8)
        # the pool holds the sources and what is copied: 3 GB at most
        most, row = 0, 2 * kv_heads * dim * _BYTES[dtype]
        while most < page:
            most = int(3.0e9 / (row * layers * sources)) - (copies + 1) * page
            if most < page:
                layers, sources = (layers, sources // 2) if sources > 1 else (layers // 2, 1)
        long = _log(rng, 1, min(32768, most))
        return dict(op=op, dtype=dtype, layers=layers, sources=sources, copies=copies,
                    kv_heads=kv_heads, dim=dim, page=page, short=max(1, long // 3), long=long)
    layers = _log(rng, 1, 32)
    row = 2 * layers * kv_heads * dim * _BYTES[dtype] * page
    pages = _log(rng, 8, max(9, min(65536, int(2.5e9 / row))))
    live = max(1, min(pages - 1, int(1.3e9 / row), int(pages * rng.uniform(0.1, 0.95))))
    return dict(op="compact", dtype=dtype, layers=layers, pages=pages, live=live,
                kv_heads=kv_heads, dim=dim, page=page, rows=_log(rng, 1, min(live, 200)))


def _lengths(count, short, long):
    """`count` lengths spread evenly from `short` to `long`."""
    return [short + (long - short) * i // max(1, count - 1) for i in range(count)] if count > 1 else [long]


def _visible(length, window, sinks):
    """How many of `length` keys the last token sees."""
    if not window or window >= length:
        return length
    return window + min(sinks, length - window)


def work(case):
    c, op, e = case, case["op"], _BYTES[case["dtype"]]
    if op == "decode":
        seen = sum(_visible(n, c["window"], c["sinks"]) for n in _lengths(c["batch"], c["short"], c["long"]))
        return {"bytes": e * (2 * seen * c["kv_heads"] * c["dim"] + 2 * c["batch"] * c["heads"] * c["dim"])
                + 4 * (seen // c["page"] + 2 * c["batch"]),
                "flops": 4.0 * c["dim"] * c["heads"] * seen}
    if op == "window":
        first = c["keys"] - c["queries"] + 1
        seen = sum(_visible(n, c["window"], c["sinks"]) for n in range(first, c["keys"] + 1))
        used = min(c["keys"], c["queries"] + c["window"] - 1 + c["sinks"])  # keys that some query sees
        return {"bytes": e * c["dim"] * c["batch"] * 2 * (c["queries"] * c["heads"] + used * c["kv_heads"]),
                "flops": 4.0 * c["dim"] * c["heads"] * c["batch"] * seen}
    if op == "append":
        tokens = c["rows"] * c["tokens"]
        return {"bytes": tokens * (4 * c["kv_heads"] * c["dim"] * e + 12), "flops": 0.0}
    token = 2 * c["layers"] * c["kv_heads"] * c["dim"] * e if op == "fork" else 0
    if op == "fork":
        lens = _lengths(c["sources"], c["short"], c["long"])
        part = sum(n % c["page"] for n in lens) * c["copies"]
        entries = sum(-(-n // c["page"]) for n in lens) * (c["copies"] + 1)
        return {"bytes": 2 * part * token + 12 * entries, "flops": 0.0}
    page = 2 * c["layers"] * c["kv_heads"] * c["dim"] * c["page"] * e
    return {"bytes": 2 * c["live"] * page + 8 * (c["live"] + c["pages"]), "flops": 0.0}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _normal(gen, dtype, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _pool(gen, dtype, *shape):
    """A pool of pages: normal values, made a slice at a time to keep the fp32 draft small."""
    out = torch.empty(shape, dtype=dtype, device="cuda")
    flat = out.view(-1)
    piece = 1 << 27
    for at in range(0, flat.numel(), piece):
        n = min(piece, flat.numel() - at)
        flat[at:at + n] = torch.randn(n, generator=gen, device="cuda")
    return out


def _table(gen, lens, page, pages, width=None):
    """A page table for rows of the given lengths: pages scattered over the pool, -1 elsewhere."""
    need = [-(-n // page) for n in lens]
    width = width or max(max(need), 1)
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    need_t = torch.tensor(need, device="cuda")
    start = torch.cumsum(need_t, 0) - need_t
    col = torch.arange(width, device="cuda")
    at = (start[:, None] + col).clamp(max=pages - 1)
    return torch.where(col < need_t[:, None], order[at], torch.full_like(order[at], -1)), sum(need)


def prepare(case, seed):
    c, op = case, case["op"]
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    mix = random.Random(int(seed))
    dtype = _DTYPES[c["dtype"]]
    s = {"case": dict(c)}
    if op == "window":
        # as a projection leaves them: heads of one token beside each other
        h, hk, d = c["heads"], c["kv_heads"], c["dim"]
        s["q"] = _normal(gen, dtype, c["batch"], c["queries"], h, d).transpose(1, 2)
        s["k"] = _normal(gen, dtype, c["batch"], c["keys"], hk, d).transpose(1, 2)
        s["v"] = _normal(gen, dtype, c["batch"], c["keys"], hk, d).transpose(1, 2)
        return s
    hk, d, page = c["kv_heads"], c["dim"], c["page"]
    if op == "decode":
        lens = _lengths(c["batch"], c["short"], c["long"])
        mix.shuffle(lens)
        pages = sum(-(-n // page) for n in lens) + 3
        s["q"] = _normal(gen, dtype, c["batch"], c["heads"], d)
        s["k_pages"] = _pool(gen, dtype, pages, hk, page, d)
        s["v_pages"] = _pool(gen, dtype, pages, hk, page, d)
        s["table"], _ = _table(gen, lens, page, pages)
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        return s
    if op == "append":
        rows, tokens = c["rows"], c["tokens"]
        lens = [c["before"] + tokens] * rows
        pages = sum(-(-n // page) for n in lens) + 3
        # keys and values as slices of the layer's fused projection
        qkv = _normal(gen, dtype, rows * tokens, c["heads"] + 2 * hk, d)
        s["k"], s["v"] = qkv[:, c["heads"]:c["heads"] + hk], qkv[:, c["heads"] + hk:]
        s["k_pages"] = _pool(gen, dtype, pages, hk, page, d)
        s["v_pages"] = _pool(gen, dtype, pages, hk, page, d)
        s["table"], _ = _table(gen, lens, page, pages)
        s["rows"] = torch.arange(rows, dtype=torch.int32, device="cuda").repeat_interleave(tokens)
        s["positions"] = (c["before"] + torch.arange(tokens, dtype=torch.int32, device="cuda")).repeat(rows)
        return s
    if op == "fork":
        src_lens = _lengths(c["sources"], c["short"], c["long"])
        mix.shuffle(src_lens)
        forks = c["sources"] * c["copies"]
        pages = sum(-(-n // page) for n in src_lens) + forks + 5
        table, used = _table(gen, src_lens + [0] * forks, page, pages)
        refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
        refs[table[table >= 0].long()] = 1
        order = torch.randperm(forks, generator=gen, device="cuda").to(torch.int32)
        s["k_pages"] = _pool(gen, dtype, c["layers"], pages, hk, page, d)
        s["v_pages"] = _pool(gen, dtype, c["layers"], pages, hk, page, d)
        s["table"], s["refs"] = table, refs
        s["lens"] = torch.tensor(src_lens + [0] * forks, dtype=torch.int32, device="cuda")
        s["src"] = order // c["copies"]
        s["dst"] = c["sources"] + torch.arange(forks, dtype=torch.int32, device="cuda")
        return s
    # compact: `live` pages shared out over the rows, the rest of the pool free;
    # one more row has branched off row 0 and shares its pages
    pages, live, rows = c["pages"], c["live"], c["rows"]
    per = [live // rows + (1 if i < live % rows else 0) for i in range(rows)]
    table, _ = _table(gen, [n * page for n in per], page, pages)
    table = torch.cat([table, table[:1]])
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs.index_add_(0, table[table >= 0].long(), torch.ones_like(table[table >= 0]))
    s["k_pages"] = _pool(gen, dtype, c["layers"], pages, hk, page, d)
    s["v_pages"] = _pool(gen, dtype, c["layers"], pages, hk, page, d)
    s["table"], s["refs"] = table, refs
    s["k_out"] = torch.zeros(c["layers"], live, hk, page, d, dtype=dtype, device="cuda")
    s["v_out"] = torch.zeros_like(s["k_out"])
    s["table_out"] = torch.empty_like(table)
    s["refs_out"] = torch.empty(live, dtype=torch.int32, device="cuda")
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    s, c = state, state["case"]
    op = c["op"]
    if own:
        bio = _package or _bio()
        if op == "decode":
            return bio.paged_attention_decode_batch_invariant(
                s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"],
                window=c["window"] or None, sinks=c["sinks"])
        if op == "window":
            return bio.sliding_window_attention_batch_invariant(
                s["q"], s["k"], s["v"], c["window"], c["sinks"])
        if op == "append":
            bio.paged_kv_append(s["k_pages"], s["v_pages"], s["k"], s["v"], s["table"],
                                s["rows"], s["positions"])
        elif op == "fork":
            bio.paged_kv_fork(s["k_pages"], s["v_pages"], s["table"], s["lens"], s["refs"],
                              s["src"], s["dst"])
        else:
            bio.paged_kv_compact(s["k_pages"], s["v_pages"], s["table"], s["refs"],
                                 s["k_out"], s["v_out"], s["table_out"], s["refs_out"])
    elif op == "decode":
        return _plain_decode(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"],
                             c["window"], c["sinks"])
    elif op == "window":
        return _plain_window(s["q"], s["k"], s["v"], c["window"], c["sinks"])
    elif op == "append":
        _plain_append(s)
    elif op == "fork":
        _plain_fork(s)
    else:
        _plain_compact(s)
    if op == "append":
        return {"k": s["k_pages"], "v": s["v_pages"]}
    if op == "fork":
        return {"k": s["k_pages"], "v": s["v_pages"], "table": s["table"], "lens": s["lens"],
                "refs": s["refs"]}
    return {"k": s["k_out"], "v": s["v_out"], "table": s["table_out"], "refs": s["refs_out"]}


def _softmax_product(scores, visible, v):
    """softmax over the last dimension of the visible scores, times v; rows that see nothing give zeros."""
    scores = scores.masked_fill(~visible, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    return (p @ v) / torch.where(total == 0, torch.ones_like(total), total)


def _plain_decode(q, k_pages, v_pages, table, lens, window, sinks):
    b, h, d = q.shape
    hk, page = k_pages.shape[1], k_pages.shape[2]
    at = table.clamp(min=0).long()
    n = at.shape[1] * page
    k = k_pages[at].float().permute(0, 2, 1, 3, 4).reshape(b, hk, n, d)
    v = v_pages[at].float().permute(0, 2, 1, 3, 4).reshape(b, hk, n, d)
    j = torch.arange(n, device=q.device)
    visible = j < lens[:, None]
    if window:
        visible &= (j >= lens[:, None] - window) | (j < sinks)
    scores = (q.float().view(b, hk, h // hk, d) @ k.transpose(-1, -2)) / math.sqrt(d)
    out = _softmax_product(scores, visible[:, None, None], v)
    return out.view(b, h, d).to(q.dtype)


def _plain_window(q, k, v, window, sinks):
    b, h, lq, d = q.shape
    hk, lk = k.shape[1], k.shape[2]
    g = h // hk
    c = min(256, lq)  # queries per band
    bands = -(-lq // c)
    span = min(window, lk) + c - 1
    pos = torch.arange(bands * c, device=q.device).view(bands, c) + (lk - lq)
    key = pos[:, :1] - min(window, lk) + 1 + torch.arange(span, device=q.device)  # [bands, span]
    inside = (key >= 0) & (key < lk)
    at = key.clamp(0, lk - 1)
    visible = (inside[:, None] & (key[:, None] <= pos[:, :, None])
               & (key[:, None] > pos[:, :, None] - window))
    few = min(sinks, lk)
    first = torch.arange(few, device=q.device)
    visible = torch.cat([visible, ((first <= pos[:, :, None]) & (first <= pos[:, :, None] - window))
                         .expand(bands, c, few)], -1)
    kf, vf = k.float(), v.float()
    kb = torch.cat([kf[:, :, at], kf[:, :, None, :few].expand(b, hk, bands, few, d)], 3)
    vb = torch.cat([vf[:, :, at], vf[:, :, None, :few].expand(b, hk, bands, few, d)], 3)
    qf = torch.zeros(b, h, bands * c, d, device=q.device)
    qf[:, :, :lq] = q.float()
    qf = qf.view(b, hk, g, bands, c, d).transpose(2, 3).reshape(b, hk, bands, g * c, d)
    scores = (qf @ kb.transpose(-1, -2)) / math.sqrt(d)
    out = _softmax_product(scores, visible.repeat(1, g, 1), vb)
    out = out.view(b, hk, bands, g, c, d).transpose(2, 3).reshape(b, h, bands * c, d)
    return out[:, :, :lq].to(q.dtype)


def _plain_append(s):
    page = s["k_pages"].shape[2]
    rows, positions = s["rows"].long(), s["positions"].long()
    at, slot = s["table"][rows, positions // page].long(), positions % page
    s["k_pages"][at, :, slot] = s["k"]
    s["v_pages"][at, :, slot] = s["v"]


def _plain_fork(s):
    k, v, table, lens, refs = s["k_pages"], s["v_pages"], s["table"], s["lens"], s["refs"]
    src, dst = s["src"].long(), s["dst"].long()
    page = k.shape[3]
    n = lens[src].long()
    full, part = n // page, n % page
    old = table[dst]
    refs.index_add_(0, old[old >= 0].long(), torch.full_like(old[old >= 0], -1))
    col = torch.arange(table.shape[1], device=table.device)
    new = torch.where(col < full[:, None], table[src], torch.full_like(old, -1))
    refs.index_add_(0, new[new >= 0].long(), torch.ones_like(new[new >= 0]))
    # the lowest free pages, in the order of the requests
    free = torch.argsort((refs != 0).int(), stable=True)
    takes = part > 0
    fresh = free[(torch.cumsum(takes.long(), 0) - 1).clamp(min=0)]
    last = table[src, full.clamp(max=table.shape[1] - 1)].long()
    new = torch.where(takes[:, None] & (col == full[:, None]), fresh[:, None].to(torch.int32), new)
    refs[fresh[takes]] = 1
    table[dst] = new
    lens[dst] = lens[src]
    slot = torch.arange(page, device=table.device)
    keep = (takes[:, None] & (slot < part[:, None])).nonzero()
    frm, to, slot = last[keep[:, 0]], fresh[keep[:, 0]], keep[:, 1]
    k[:, to, :, slot] = k[:, frm, :, slot]
    v[:, to, :, slot] = v[:, frm, :, slot]


def _plain_compact(s):
    table, refs = s["table"], s["refs"]
    live = refs > 0
    new = (torch.cumsum(live, 0) - 1).to(torch.int32)
    pages = live.nonzero()[:, 0]
    s["table_out"].copy_(torch.where(table >= 0, new[table.clamp(min=0).long()], table))
    s["refs_out"].zero_()
    s["refs_out"][:pages.numel()] = refs[pages]
    s["k_out"][:, :pages.numel()] = s["k_pages"][:, pages]
    s["v_out"][:, :pages.numel()] = s["v_pages"][:, pages]


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    """Attention outputs from the definition, a sequence or a block of queries
    at a time; the cache operators move values and compute none."""
    if case["op"] == "decode":
        s = prepare(case, seed)
        q, lens, table = s["q"].double(), s["lens"].tolist(), s["table"].long()
        b, h, d = q.shape
        hk = case["kv_heads"]
        out = torch.zeros_like(q)
        for i in range(b):
            keys = torch.arange(lens[i], device="cuda")
            if case["window"]:
                keys = keys[(keys >= lens[i] - case["window"]) | (keys < case["sinks"])]
            if not keys.numel():
                continue
            at, slot = table[i, keys // case["page"]], keys % case["page"]
            k, v = s["k_pages"][at, :, slot].double(), s["v_pages"][at, :, slot].double()  # [n, hk, d]
            w = torch.einsum("gad,ngd->gan", q[i].view(hk, h // hk, d), k) * d ** -0.5
            out[i] = torch.einsum("gan,ngd->gad", torch.softmax(w, -1), v).reshape(h, d)
        return out
    if case["op"] == "window":
        s = prepare(case, seed)
        q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
        b, h, lq, d = q.shape
        hk, lk = k.shape[1], k.shape[2]
        k, v = k.repeat_interleave(h // hk, 1), v.repeat_interleave(h // hk, 1)
        out = torch.zeros_like(q)
        step = 1024
        for i in range(0, lq, step):
            p = torch.arange(i, min(lq, i + step), device="cuda") + (lk - lq)
            lo, hi = max(0, int(p[0]) - case["window"] + 1), int(p[-1]) + 1
            keys = torch.cat([torch.arange(min(case["sinks"], lo), device="cuda"),
                              torch.arange(lo, hi, device="cuda")])
            hide = (keys > p[:, None]) | ((keys <= p[:, None] - case["window"]) & (keys >= case["sinks"]))
            w = (q[:, :, i:i + step] @ k[:, :, keys].transpose(-1, -2)) * d ** -0.5
            w = w.masked_fill(hide, -math.inf).softmax(-1)
            out[:, :, i:i + step] = w @ v[:, :, keys]
        return out
    return None
