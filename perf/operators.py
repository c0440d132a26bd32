"""Workloads of the 8-bit paged KV cache: attention over it, appending to it and
reading it back, and the management of its pages.

A cache holds the keys and values of ``layers`` layers in pages of ``page`` tokens:
``k`` and ``v`` are ``(layers, pages, kv_heads, page, head_dim)`` codes of 8 bits
(e4m3 or int8), ``k_scale`` and ``v_scale`` ``(layers, pages, kv_heads)`` hold one
power of two for each block (a page of one head), and code * scale is the value.
``tables`` ``(sequences, pages_per_sequence)`` lists the pages of each sequence in
order (-1: none), ``lengths`` its tokens, ``refcounts`` how many tables list a page.

``run`` computes a pass in plain torch operations, or, with ``own`` true, through
``gemma4_fa4_kernels_b200.PagedKVCache8``.  Head layouts are the two layers of this
repository's model: global (32 query heads, 4 KV heads, head_dim 512) and local
(32, 16, 256, window 1024).
"""

import math
import random

import torch

own = False

GLOBAL = {"q_heads": 32, "kv_heads": 4, "head_dim": 512, "window": 0}
LOCAL = {"q_heads": 32, "kv_heads": 16, "head_dim": 256, "window": 1024}
DTYPES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
# exponent range of a block's scale; a block of zeros takes the smallest
MIN_EXP, MAX_EXP = -100, 120


# ------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------
def _attention(name, layer, dtype, page, batch, q_len, min_len, max_len, ragged=False, layout=1):
    return {"name": name, "op": "attention", **layer, "dtype": dtype, "page": page, "batch": batch,
            "q_len": q_len, "min_len": min_len, "max_len": max_len, "ragged": ragged,
            "layout": layout}


def _append(name, layer, dtype, page, batch, tokens, min_len, max_len, ragged=False, layout=1):
    return {"name": name, "op": "append", **layer, "dtype": dtype, "page": page, "batch": batch,
            "q_len": tokens, "min_len": min_len, "max_len": max_len, "ragged": ragged,
            "layout": layout}


def _pages(name, op, layer, layers, page, layout=1, **more):
    return {"name": name, "op": op, **layer, "dtype": "int8", "layers": layers, "page": page,
            "layout": layout, **more}


def listed():
    return [
        # one user's first answer tokens, a global layer: launch latency is all there is
        _attention("decode_short", GLOBAL, "e4m3", 64, 1, 1, 300, 300),
        # one user deep in a long document, a global layer: the cache's bytes
        _attention("decode_long", GLOBAL, "e4m3", 64, 1, 1, 131072, 131072),
        # a server's decode batch, contexts of every length, a global layer
        _attention("decode_ragged", GLOBAL, "int8", 32, 24, 1, 90, 32768),
        # the same on a sliding-window layer: many short ranges
        _attention("decode_window", LOCAL, "e4m3", 16, 96, 1, 100, 20000),
        # a few drafted tokens verified at once, not as many for every user
        _attention("verify", GLOBAL, "int8", 64, 6, 5, 700, 9001, ragged=True),
        # a chunk of a prompt against what is cached of it already
        _attention("chunk", GLOBAL, "e4m3", 64, 1, 1000, 17000, 17000),
        # the decode batch's new tokens written to a local layer, and read back
        _append("append_token", LOCAL, "e4m3", 64, 64, 1, 1, 8000),
        # two prompts written to a global layer, and read back
        _append("append_prompt", GLOBAL, "int8", 32, 2, 6001, 6001, 9000, ragged=True),
        # a shared prefix given to another owner, page by page, in ten global layers
        _pages("copy", "copy", GLOBAL, 10, 64, pairs=200),
        # a few continuations of few sequences dropped and drawn anew
        _pages("beams_small", "beams", GLOBAL, 1, 16, parents=2, children=4, min_len=40,
               max_len=500, counts=2),
        # wide sampling: 48 continuations of 6 prompts in ten global layers
        _pages("beams", "beams", GLOBAL, 10, 64, parents=6, children=48, min_len=500,
               max_len=9000, counts=3),
        # a third of the users leave, the pool is closed up for the next big prompt
        _pages("defrag", "defrag", GLOBAL, 4, 64, sequences=60, min_len=300, max_len=4000),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    layer = rng.choice([GLOBAL, LOCAL])
    dtype = rng.choice(["e4m3", "int8"])
    page = rng.choice([16, 32, 64, 128])
    layout = rng.randrange(1, 1 << 30)
    op = rng.choice(["decode", "decode", "decode", "verify", "chunk", "append", "append", "copy",
                     "beams", "defrag"])
    if op in ("decode", "verify"):
        q_len = 1 if op == "decode" else rng.randint(2, 12)
        # the batch's visible keys stay below the long single sequence's
        batch = _log(rng, 1, 96)
        if layer["window"]:
            max_len = _log(rng, q_len + 20, 20000)
        else:
            max_len = _log(rng, q_len + 20, min(131072, 260000 // batch))
        min_len = rng.randint(q_len, max_len)
        return _attention("", layer, dtype, page, batch, q_len, min_len, max_len,
                          ragged=q_len > 1, layout=layout)
    if op == "chunk":
        q_len = _log(rng, 13, 1000)
        max_len = _log(rng, q_len, 17000)
        batch = rng.randint(1, 2) if max_len < 8000 else 1
        return _attention("", layer, dtype, page, batch, q_len, rng.randint(q_len, max_len), max_len,
                          ragged=batch > 1, layout=layout)
    if op == "append":
        tokens = _log(rng, 1, 6000)
        batch = _log(rng, 1, max(1, min(96, 12000 // tokens)))
        max_len = tokens + _log(rng, 1, 3000)
        return _append("", layer, dtype, page, batch, tokens, rng.randint(tokens, max_len), max_len,
                       ragged=tokens > 1, layout=layout)
    layers = _log(rng, 1, 10) if page <= 64 else _log(rng, 1, 5)
    if op == "copy":
        return _pages("", op, layer, layers, page, layout, pairs=_log(rng, 1, 200))
    if op == "beams":
        parents = rng.randint(1, 6)
        return _pages("", op, layer, layers, page, layout, parents=parents,
                      children=parents * rng.randint(1, 8), min_len=_log(rng, 1, 400),
                      max_len=_log(rng, 401, 6000), counts=rng.randint(1, 2 * page))
    return _pages("", op, layer, min(layers, 4), page, layout, sequences=rng.randint(3, 60),
                  min_len=_log(rng, 1, 300), max_len=_log(rng, 301, 3000))


# ------------------------------------------------------------------------------------
# the layout of a case: lengths and tables, from the case alone
# ------------------------------------------------------------------------------------
def _spread(count, lo, hi, rng):
    """``count`` lengths from lo to hi, even over their logarithm, in shuffled order."""
    if count == 1:
        return [hi]
    out = [int(round(lo * (hi / lo) ** (i / (count - 1)))) for i in range(count)]
    rng.shuffle(out)
    return out


def _ceil(a, b):
    return -(-a // b)


def _spans(case):
    """(start, end) of every row's new tokens; ends are the sequence lengths."""
    rng = random.Random(case["layout"])
    ends = _spread(case["batch"], case["min_len"], case["max_len"], rng)
    new = [max(1, case["q_len"] - (b % 3 if case["ragged"] else 0)) for b in range(case["batch"])]
    return [(e - n, e) for e, n in zip(ends, new)]


def _deal(lens, page, extra, rng):
    """Pages of sequences of these lengths, dealt at random from a pool with ``extra``
    more; the tables as lists, and the pool's size."""
    need = [_ceil(n, page) for n in lens]
    pool = sum(need) + extra
    ids = list(range(pool))
    rng.shuffle(ids)
    tables, at = [], 0
    for n in need:
        tables.append(ids[at:at + n])
        at += n
    return tables, pool


def _beams_layout(case):
    rng = random.Random(case["layout"])
    page, children = case["page"], case["children"]
    lens = _spread(case["parents"], case["min_len"], case["max_len"], rng)
    tables, pool = _deal(lens, page, children * (2 + case["counts"] // page), rng)
    of = [c * case["parents"] // children for c in range(children)]
    return lens, tables, pool, of


def _defrag_layout(case):
    rng = random.Random(case["layout"])
    n = case["sequences"]
    lens = _spread(n, case["min_len"], case["max_len"], rng)
    tables, pool = _deal(lens, case["page"], sum(lens) // case["page"] // 8 + 1, rng)
    done = sorted(rng.sample(range(n), _ceil(n, 3)))
    live = {p for s in range(n) if s not in done for p in tables[s]}
    moves = sum(p >= len(live) for p in live)
    return lens, tables, pool, done, moves


def _pairs(q_start, end, window):
    """Visible (query, key) pairs and distinct visible keys of one row and head."""
    pairs = sum(min(p + 1, window) if window else p + 1 for p in range(q_start, end))
    first = max(0, q_start - window + 1) if window else 0
    return pairs, end - first


def work(case):
    hq, hkv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    page = case["page"]
    if case["op"] == "attention":
        nbytes = flops = 0
        for start, end in _spans(case):
            pairs, keys = _pairs(start, end, case["window"])
            n = end - start
            nbytes += hkv * (2 * keys * d + 2 * 4 * _ceil(keys, page)) + 4 * _ceil(keys, page)
            nbytes += hq * n * (2 * 2 * d + 4)
            flops += 4 * hq * d * pairs
        return {"bytes": nbytes, "flops": flops}
    if case["op"] == "append":
        tokens = sum(e - s for s, e in _spans(case))
        blocks = sum(_ceil(e, page) - s // page for s, e in _spans(case))
        # written in 8 bits from 16, then read from 8 into 16; scales written and read
        return {"bytes": 2 * hkv * (tokens * d * (2 + 1 + 1 + 2) + blocks * 2 * 4),
                "flops": 4 * hkv * d * tokens}
    page_bytes = case["layers"] * hkv * 2 * (page * d + 4)
    if case["op"] == "copy":
        return {"bytes": 2 * case["pairs"] * (page_bytes + 4), "flops": 0}
    if case["op"] == "beams":
        lens, tables, _, of = _beams_layout(case)
        copies = sum(lens[p] % page != 0 for p in of)
        entries = sum(len(tables[p]) for p in of)
        # tables read and written, counters down and up again, the last pages copied
        return {"bytes": 2 * copies * page_bytes + 4 * entries * 6, "flops": 0}
    lens, tables, pool, _, moves = _defrag_layout(case)
    entries = sum(len(t) for t in tables)
    return {"bytes": 2 * moves * page_bytes + 4 * (2 * pool + 2 * entries), "flops": 0}


# ------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------
def _rms(x):
    return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-6)


def _random_rows(gen, *shape):
    """Rows as the norms before attention leave them: unit RMS."""
    return _rms(torch.randn(*shape, generator=gen, device="cuda"))


def _codes_of(x, dtype, exp):
    y = x * torch.exp2(-exp.float())
    return y.to(torch.float8_e4m3fn) if dtype == "e4m3" else torch.round(y).to(torch.int8)


def _fill(k, scale, dtype, gen):
    """Every block of the cache filled with quantised rows (recycled pages hold old ones)."""
    layers, pages, heads, page, d = k.shape
    step = max(1, (1 << 27) // (heads * page * d))
    for layer in range(layers):
        for p in range(0, pages, step):
            n = min(step, pages - p)
            x = _random_rows(gen, n, heads, page, d)
            exp = _need(x.abs().amax((-1, -2)), dtype)
            scale[layer, p:p + n] = torch.exp2(exp.float())
            k[layer, p:p + n] = _codes_of(x, dtype, exp[..., None, None])


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _cache(case, layers, tables, lens, pool, gen, sequences, row_pages):
    hkv, page, d = case["kv_heads"], case["page"], case["head_dim"]
    shape = (layers, pool, hkv, page, d)
    st = {"k": torch.empty(shape, dtype=DTYPES[case["dtype"]], device="cuda"),
          "v": torch.empty(shape, dtype=DTYPES[case["dtype"]], device="cuda"),
          "k_scale": torch.empty(shape[:3], device="cuda"),
          "v_scale": torch.empty(shape[:3], device="cuda")}
    _fill(st["k"], st["k_scale"], case["dtype"], gen)
    _fill(st["v"], st["v_scale"], case["dtype"], gen)
    refs = [0] * pool
    for t in tables:
        for p in t:
            refs[p] += 1
    rows = [t + [-1] * (row_pages - len(t)) for t in tables]
    rows += [[-1] * row_pages] * (sequences - len(rows))
    st["tables"] = _ints(rows)
    st["lengths"] = _ints(list(lens) + [0] * (sequences - len(lens)))
    st["refcounts"] = _ints(refs)
    return st


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, page = case["op"], case["page"]
    rng = random.Random(case["layout"] + 1)
    if op in ("attention", "append"):
        spans = _spans(case)
        lens = [e for _, e in spans]
        tables, pool = _deal(lens, page, 3, rng)
        st = _cache(case, 1, tables, lens, pool, gen, case["batch"], _ceil(max(lens), page))
        st["slots"] = _ints(list(range(case["batch"])))
        st["starts"], st["ends"] = _ints([s for s, _ in spans]), _ints(lens)
        st["spans"] = spans
        b, n, d = case["batch"], case["q_len"], case["head_dim"]
        if op == "attention":
            # scores spread by a few units, as the learned query scales leave them
            q = 0.25 * _random_rows(gen, b, n, case["q_heads"], d)
            st["q"] = q.to(torch.bfloat16)
        else:
            st["new_k"] = _random_rows(gen, b, n, case["kv_heads"], d).to(torch.bfloat16)
            st["new_v"] = _random_rows(gen, b, n, case["kv_heads"], d).to(torch.bfloat16)
            # read back from the start of the page that the first new token falls in
            st["first"] = _ints([s // page * page for s, _ in spans])
            st["most"] = max(e - s // page * page for s, e in spans)
    elif op == "copy":
        n = case["pairs"]
        ids = list(range(2 * n + 3))
        rng.shuffle(ids)
        st = _cache(case, case["layers"], [ids[:n]], [n * page], 2 * n + 3, gen, 2, 2 * n + 3)
        st["src"], st["dst"] = _ints(ids[:n]), _ints(ids[n:2 * n])
    elif op == "beams":
        lens, tables, pool, of = _beams_layout(case)
        children = case["children"]
        st = _cache(case, case["layers"], tables, lens, pool, gen, len(lens) + children,
                    _ceil(max(lens) + case["counts"], page))
        st["parents"] = _ints(of)
        st["children"] = _ints(list(range(len(lens), len(lens) + children)))
        st["counts"] = torch.full_like(st["children"], case["counts"])
    else:
        lens, tables, pool, done, _ = _defrag_layout(case)
        st = _cache(case, case["layers"], tables, lens, pool, gen, len(lens),
                    _ceil(max(lens), page))
        st["done"] = _ints(done)
        st["saved"] = [st[x].clone() for x in ("tables", "lengths", "refcounts")]
    st["case"] = case
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    if own:
        from gemma4_fa4_kernels_b200 import PagedKVCache8
        st["cache"] = PagedKVCache8.from_tensors(
            st["k"], st["v"], st["k_scale"], st["v_scale"], st["tables"], st["lengths"],
            st["refcounts"])
    return st


# ------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------
def _need(amax, dtype):
    """Least exponent e with amax <= largest * 2^e (largest: 448 = 0.875 * 2^9 for e4m3,
    127 = 0.9921875 * 2^7 for int8)."""
    m, x = torch.frexp(amax)
    if dtype == "e4m3":
        e = x - 9 + (m > 0.875).int()
    else:
        e = x - 7 + (m > 0.9921875).int()
    e = torch.where(amax > 0, e, torch.full_like(e, MIN_EXP))
    return e.clamp(MIN_EXP, MAX_EXP)


def _rows(st, pages, scale):
    """Values of these pages (n, heads, page, d) -> (heads, n * page, d), in 32 bits."""
    x = pages.float() * scale[..., None, None]
    n, h, page, d = x.shape
    return x.transpose(0, 1).reshape(h, n * page, d)


def _plain_attention(st):
    case = st["case"]
    q = st["q"]
    b, sq, hq, d = q.shape
    hkv, page, window = case["kv_heads"], case["page"], case["window"]
    group = hq // hkv
    out = torch.zeros_like(q)
    lse = torch.full((b, hq, sq), float("-inf"), device=q.device)
    for i, (start, end) in enumerate(st["spans"]):
        first = max(0, start - window + 1) // page if window else 0
        ids = st["tables"][i, first:_ceil(end, page)].long()
        n, lo = end - start, first * page
        k = _rows(st, st["k"][0][ids], st["k_scale"][0][ids])[:, :end - lo]
        v = _rows(st, st["v"][0][ids], st["v_scale"][0][ids])[:, :end - lo]
        q_pos = torch.arange(start, end, device=q.device)[:, None]
        k_pos = torch.arange(lo, end, device=q.device)[None]
        seen = k_pos <= q_pos
        if window:
            seen = seen & (k_pos > q_pos - window)
        qh = q[i, :n].float().view(n, hkv, group, d).permute(1, 2, 0, 3)
        s = (qh.reshape(hkv, group * n, d) @ k.transpose(1, 2)).view(hkv, group, n, -1)
        s.masked_fill_(~seen, float("-inf"))
        top = s.amax(-1, keepdim=True)
        p = s.sub_(top).exp_()
        total = p.sum(-1, keepdim=True)
        o = (p.view(hkv, group * n, -1) @ v).view(hkv, group, n, d) / total
        out[i, :n] = o.permute(2, 0, 1, 3).reshape(n, hq, d).to(q.dtype)
        lse[i, :, :n] = (top + total.log()).view(hq, n)
    return out, lse


def _plain_write(st, codes, scales, new):
    case = st["case"]
    page, dtype = case["page"], case["dtype"]
    for i, (start, end) in enumerate(st["spans"]):
        p0, p1 = start // page, _ceil(end, page)
        ids = st["tables"][i, p0:p1].long()
        pos = torch.arange(p0 * page, p1 * page, device=codes.device)
        fresh = (pos >= start) & (pos < end)
        x = torch.zeros((p1 - p0) * page, *new.shape[2:], device=codes.device)
        x[start - p0 * page:end - p0 * page] = new[i, :end - start].float()
        x = x.view(p1 - p0, page, *new.shape[2:]).transpose(1, 2)  # (pages, heads, page, d)
        exp = _need(x.abs().amax((-1, -2)), dtype)
        before = scales[ids]
        if start % page:  # the page holds earlier tokens: its scale only grows
            old = torch.frexp(before[0])[1] - 1
            exp[0] = torch.maximum(exp[0], old)
        e = exp[..., None, None]
        held = codes[ids]
        kept = _codes_of(held.float() * before[..., None, None], dtype, e)
        put = _codes_of(x, dtype, e)
        fresh = fresh.view(p1 - p0, 1, page, 1)
        earlier = (pos < start).view(p1 - p0, 1, page, 1)
        # through bytes: torch selects no 8-bit floats
        merged = torch.where(fresh, put.view(torch.uint8), torch.where(
            earlier, kept.view(torch.uint8), held.view(torch.uint8)))
        codes[ids] = merged.view(codes.dtype)
        scales[ids] = torch.exp2(exp.float())


def _plain_read(st, codes, scales):
    case = st["case"]
    page = case["page"]
    out = torch.zeros(case["batch"], st["most"], case["kv_heads"], case["head_dim"],
                      dtype=torch.bfloat16, device=codes.device)
    for i, (start, end) in enumerate(st["spans"]):
        p0 = start // page
        ids = st["tables"][i, p0:_ceil(end, page)].long()
        n = end - p0 * page
        x = _rows(st, codes[ids], scales[ids])[:, :n]
        out[i, :n] = x.transpose(0, 1).to(torch.bfloat16)
    return out


def _plain_copy(st, src, dst):
    for x in ("k", "v", "k_scale", "v_scale"):
        st[x][:, dst.long()] = st[x][:, src.long()]


def _count(st, ids):
    """How often each page is listed in ``ids`` (-1: none)."""
    pool = st["refcounts"].shape[0]
    flat = torch.where(ids >= 0, ids, pool).flatten().long()
    return torch.zeros(pool + 1, dtype=torch.int32, device=ids.device).scatter_add_(
        0, flat, torch.ones_like(flat, dtype=torch.int32))[:pool]


def _plain_free(st, slots):
    slots = slots.long()
    st["refcounts"] -= _count(st, st["tables"][slots])
    st["tables"][slots] = -1
    st["lengths"][slots] = 0


def _free_pages(st):
    """Page ids, the free ones first, ascending."""
    return torch.sort((st["refcounts"] > 0).int(), stable=True)[1]


def _plain_fork(st):
    page = st["case"]["page"]
    parents, children = st["parents"].long(), st["children"].long()
    lens = st["lengths"][parents]
    whole, part = lens // page, lens % page > 0
    rows = st["tables"][parents]
    col = torch.arange(rows.shape[1], device=rows.device)[None]
    rank = part.int().cumsum(0) - 1
    new = _free_pages(st)[rank.clamp(min=0).long()].int()
    at_part = (col == whole[:, None]) & part[:, None]
    kept = torch.where(col < whole[:, None], rows, -1)
    st["refcounts"] += _count(st, kept)
    st["tables"][children] = torch.where(at_part, new[:, None], kept)
    st["refcounts"] += _count(st, torch.where(part, new, -1))
    st["lengths"][children] = lens
    here = part.nonzero()[:, 0]
    _plain_copy(st, rows[here, whole[here].long()], new[here])


def _plain_extend(st):
    page, slots = st["case"]["page"], st["children"].long()
    starts = st["lengths"][slots]
    ends = starts + st["counts"]
    have, want = (starts + page - 1) // page, (ends + page - 1) // page
    need = want - have
    first = need.cumsum(0) - need
    free = _free_pages(st)
    for j in range(_ceil(st["case"]["counts"], page)):
        here = j < need
        page_id = torch.where(here, free[(first + j).long().clamp(max=free.shape[0] - 1)], -1).int()
        at = (have + j).clamp(max=st["tables"].shape[1] - 1).long()
        st["tables"][slots, at] = torch.where(here, page_id, st["tables"][slots, at])
        st["refcounts"] += _count(st, page_id)
    st["lengths"][slots] = ends
    return starts, ends


def _plain_compact(st):
    refs = st["refcounts"]
    live = refs > 0
    n_live = live.sum()
    ids = torch.arange(refs.shape[0], device=refs.device)
    holes = (~live & (ids < n_live)).nonzero()[:, 0]
    movers = (live & (ids >= n_live)).nonzero()[:, 0]
    moved = ids.clone()
    moved[movers] = holes
    t = st["tables"]
    t.copy_(torch.where(t >= 0, moved[t.clamp(min=0).long()].int(), t))
    refs[holes] = refs[movers]
    refs[movers] = 0
    _plain_copy(st, movers, holes)


# ------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------
def _state(st):
    return [st[x] for x in ("tables", "lengths", "refcounts", "k", "v", "k_scale", "v_scale")]


def run(state):
    st, case = state, state["case"]
    op = case["op"]
    cache = st["cache"] if own else None
    if op == "attention":
        if own:
            return cache.attention(0, st["q"], st["slots"], st["starts"], st["ends"],
                                   window=case["window"], max_seqlen_k=case["max_len"])
        return _plain_attention(st)
    if op == "append":
        if own:
            cache.append(0, st["new_k"], st["new_v"], st["slots"], st["starts"], st["ends"])
            k, v = cache.read(0, st["slots"], st["first"], st["ends"], max_tokens=st["most"])
        else:
            _plain_write(st, st["k"][0], st["k_scale"][0], st["new_k"])
            _plain_write(st, st["v"][0], st["v_scale"][0], st["new_v"])
            k = _plain_read(st, st["k"][0], st["k_scale"][0])
            v = _plain_read(st, st["v"][0], st["v_scale"][0])
        return k, v, st["k_scale"], st["v_scale"]
    if op == "copy":
        if own:
            cache.copy_pages(st["src"], st["dst"])
        else:
            _plain_copy(st, st["src"], st["dst"])
        return _state(st)
    if op == "beams":
        if own:
            cache.free(st["children"])
            cache.fork(st["parents"], st["children"])
            starts, ends = cache.extend(st["children"], st["counts"])
        else:
            _plain_free(st, st["children"])
            _plain_fork(st)
            starts, ends = _plain_extend(st)
        return [starts, ends] + _state(st)
    # the scheduler's tables are put back first, so that each pass finds the same holes
    for x, saved in zip(("tables", "lengths", "refcounts"), st["saved"]):
        st[x].copy_(saved)
    if own:
        cache.free(st["done"])
        cache.compact()
    else:
        _plain_free(st, st["done"])
        _plain_compact(st)
    return _state(st)


# ------------------------------------------------------------------------------------
# from the definitions, in 64 bits
# ------------------------------------------------------------------------------------
def _exact_attention(case, st):
    q = st["q"].double()
    b, sq, hq, d = q.shape
    hkv, page, window = case["kv_heads"], case["page"], case["window"]
    group = hq // hkv
    out = torch.zeros(b, sq, hq, d, dtype=torch.float64, device=q.device)
    lse = torch.full((b, hq, sq), -math.inf, dtype=torch.float64, device=q.device)
    for i, (start, end) in enumerate(_spans(case)):
        lo = max(0, start - window + 1) if window else 0
        pos = torch.arange(lo, end, device=q.device)
        ids = st["tables"][i].long()[pos // page]
        for h in range(hkv):
            k = st["k"][0, ids, h, pos % page].double() * st["k_scale"][0, ids, h, None].double()
            v = st["v"][0, ids, h, pos % page].double() * st["v_scale"][0, ids, h, None].double()
            step = max(1, (1 << 28) // (group * (end - lo)))  # queries at once
            for t in range(0, end - start, step):
                n = min(step, end - start - t)
                at = torch.arange(start + t, start + t + n, device=q.device)
                s = torch.einsum("ngd,kd->ngk", q[i, t:t + n, h * group:(h + 1) * group], k)
                hidden = pos[None] > at[:, None]
                if window:
                    hidden = hidden | (at[:, None] - pos[None] >= window)
                s = s.masked_fill(hidden[:, None], -math.inf)
                norm = torch.logsumexp(s, -1)
                w = torch.exp(s - norm[..., None])
                out[i, t:t + n, h * group:(h + 1) * group] = torch.einsum("ngk,kd->ngd", w, v)
                lse[i, h * group:(h + 1) * group, t:t + n] = norm.T
    return out, lse


def _exact_grid(x, dtype):
    """Nearest code value, ties to even, in 64 bits."""
    if dtype == "int8":
        return torch.round(x)
    size = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -9)))
    step = torch.exp2(size.clamp(min=-6) - 3)
    return torch.round(x / step) * step


def _exact_append(case, st, codes, scales, new):
    page, dtype = case["page"], case["dtype"]
    top = 448.0 if dtype == "e4m3" else 127.0
    powers = torch.exp2(torch.arange(MIN_EXP, MAX_EXP + 1, dtype=torch.float64, device=codes.device))
    out = torch.zeros(case["batch"], st["most"], case["kv_heads"], case["head_dim"],
                      dtype=torch.float64, device=codes.device)
    scales = scales.double().clone()
    for i, (start, end) in enumerate(_spans(case)):
        for p in range(start // page, _ceil(end, page)):
            a, z = max(start, p * page), min(end, (p + 1) * page)
            page_id = int(st["tables"][i, p])
            x = new[i, a - start:z - start].double()  # (tokens, heads, d)
            largest = x.abs().amax(dim=(0, 2))
            scale = powers[(largest[:, None] > top * powers).sum(1).clamp(max=len(powers) - 1)]
            at = p * page - start // page * page
            if a > p * page:
                scale = torch.maximum(scale, scales[page_id])
                old = codes[page_id, :, :a - p * page].double() * scales[page_id][:, None, None]
                old = _exact_grid(old / scale[:, None, None], dtype) * scale[:, None, None]
                out[i, at:at + a - p * page] = old.transpose(0, 1)
            x = _exact_grid(x / scale[:, None], dtype) * scale[:, None]
            out[i, at + a - p * page:at + z - p * page] = x
            scales[page_id] = scale
    return out, scales[None]


def exact(case, seed):
    if case["op"] not in ("attention", "append"):
        return None  # whole numbers and bytes moved: nothing is computed
    st = _inputs(case, seed)
    if case["op"] == "attention":
        return _exact_attention(case, st)
    k, k_scale = _exact_append(case, st, st["k"][0], st["k_scale"][0], st["new_k"])
    v, v_scale = _exact_append(case, st, st["v"][0], st["v_scale"][0], st["new_v"])
    return k, v, k_scale, v_scale
