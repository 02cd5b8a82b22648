"""The operators of a paged poly KV cache, as cases that can be timed.

A server keeps the cached positions of its rows (users' conversations) in pages of one pool: row b's
position p lies in page ``pages[b, p // page_size]``, so that rows grow, share what they have in common
and end without anything being moved.  A step brings each row a chunk of new tokens -- a prompt's, or
one token of a row that is being continued -- padded to the longest chunk, or packed one row behind the
other.  Four kinds of case:

* ``append`` -- the query/key norms and the rotary embedding of a layer's new tokens, and the writes of
  their keys and deepest values into the rows' pages;
* ``attend`` -- every level of the poly attention for the new tokens, over the row's cached positions
  and the chunk's own up to each token.  Level t (0 the deepest) scores ``keys[t]`` with the queries
  ``keys[t + 1]`` (the last level's are given) plus ``lses[t - 1]`` and averages ``values[t]``; its
  average, times the next middle level's projected values, is that level's ``values[t + 1]``, held in
  the cache's type like every other cached value;
* ``fork`` -- rows become the beginnings of other rows, sharing their pages, and all of them grow: the
  pages that are needed are found, and a page that is shared and about to be written is copied first;
* ``compact`` -- the pages in use move to the front of the pool.
"""

import math
import os
import random
import sys
import types

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_ES = {"bf16": 2, "f16": 2, "f32": 4}


def _package():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    path = os.path.join(root, "poly-attention_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import poly_attention

    return poly_attention


# ---------------------------------------------------------------------------------------
# cases.  n: cached positions of the longest row, t: new tokens of the longest chunk.  chunks: "all"
# rows bring t tokens, "mixed" one row t and the others one, "ragged" anything from none to t.


def _attend(order, rows, n, t, heads, kv_heads, d, dtype="bf16", page=64, chunks="all",
            packed=False, ragged=True, softclamp=0.0):
    return {"kind": "attend", "order": order, "rows": rows, "n": n, "t": t, "heads": heads,
            "kv_heads": kv_heads, "d": d, "dtype": dtype, "page": page, "chunks": chunks,
            "packed": packed, "ragged": ragged, "softclamp": softclamp}


def _append(order, rows, t, heads, kv_heads, d, rot, dtype="bf16", page=64, chunks="all",
            packed=False):
    return {"kind": "append", "order": order, "rows": rows, "n": 8192, "t": t, "heads": heads,
            "kv_heads": kv_heads, "d": d, "rot": rot, "dtype": dtype, "page": page,
            "chunks": chunks, "packed": packed, "ragged": True}


def _fork(layers, order, rows, prompts, n, t, kv_heads, d, dtype="bf16", page=64):
    return {"kind": "fork", "layers": layers, "order": order, "rows": rows, "prompts": prompts,
            "n": n, "t": t, "kv_heads": kv_heads, "d": d, "dtype": dtype, "page": page}


def _compact(layers, order, rows, n, kv_heads, d, dtype="bf16", page=64):
    return {"kind": "compact", "layers": layers, "order": order, "rows": rows, "n": n,
            "kv_heads": kv_heads, "d": d, "dtype": dtype, "page": page}


def listed():
    cases = {
        # one user's next token in a short conversation: latency
        "attend_one_user": _attend(2, 1, 300, 1, 8, 8, 64),
        # the grouped-query layer over long rows (bench.py's config 5), a token each
        "attend_tokens": _attend(2, 32, 8192, 1, 32, 8, 128),
        # a long prompt's next piece, behind as much that is cached already
        "attend_prompt": _attend(2, 1, 4096, 4096, 32, 8, 128, ragged=False),
        # an order-3 layer (bench.py's config 4) with a prompt beside rows that go on, packed, small pages
        "attend_mixed": _attend(3, 16, 2048, 512, 16, 16, 64, page=16, chunks="mixed", packed=True),
        # several short chunks of uneven lengths, f16, soft-clamped scores, large pages
        "attend_chunks": _attend(2, 6, 5003, 61, 12, 4, 128, dtype="f16", page=256,
                                 chunks="ragged", softclamp=50.0),
        # full precision, a head dim between the usual ones
        "attend_f32": _attend(2, 3, 1111, 130, 8, 2, 96, dtype="f32", page=32, chunks="ragged",
                              packed=True),
        # the norms and rotary of a prompt's piece of the grouped-query layer
        "append_prompt": _append(2, 1, 4096, 32, 8, 128, 128),
        # a token each of a few rows of a small order-3 layer, half of each head rotated: latency
        "append_tokens": _append(3, 5, 1, 8, 8, 64, 32, dtype="f16", page=16),
        # eight prompts of an eight-layer model tried in four ways each
        "fork_beams": _fork(8, 2, 32, 8, 1500, 1, 8, 128),
        # one user's conversation continued twice: latency
        "fork_one_user": _fork(2, 2, 2, 1, 301, 1, 8, 64, page=16),
        # a server's pool (order-3 layers of bench.py's config 4) after half of its rows have ended
        "compact_pool": _compact(6, 3, 64, 700, 16, 64),
        # a small pool with large pages
        "compact_small": _compact(1, 2, 9, 333, 4, 96, dtype="f32", page=128),
    }
    return [dict(c, name=k) for k, c in cases.items()]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "attend", "append", "fork", "compact"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    page = rng.choice([16, 32, 64, 64, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8, 16])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 8])
    d = rng.choice([64, 64, 128, 128, 32, 96, 40])
    es = _ES[dtype]
    if kind == "attend":
        order = rng.choice([2, 2, 2, 3, 4])
        rows = _log_int(rng, 1, 48)
        t = rng.choice([1, _log_int(rng, 2, 64), _log_int(rng, 2, 1500)])
        chunks = rng.choice(["all", "all", "mixed", "ragged"])
        tokens = t + rows if chunks == "mixed" else rows * t
        # at most about a quarter of the largest listed cases' bytes and products, and of the plain
        # form's scores
        most = 5e8 / (rows * kv_heads * d * es * 2 * order)
        most = min(most, (4e10 if dtype == "f32" else 1.5e11) / (4.0 * tokens * d * (heads + (order - 1) * kv_heads)))
        most = min(most, 4e8 / (rows * t * heads))
        while most < 2 and t > 1:
            t, most = t // 2, 4 * most
        n = _log_int(rng, 1, max(2, min(32768, int(most))))
        return _attend(order, rows, n, t, heads, kv_heads, d, dtype=dtype, page=page, chunks=chunks,
                       packed=rng.random() < 0.5, ragged=rng.random() < 0.7,
                       softclamp=rng.choice([0.0, 0.0, 30.0]))
    if kind == "append":
        rows = _log_int(rng, 1, 48)
        t = rng.choice([1, _log_int(rng, 2, 1000)])
        t = max(1, min(t, 8192 // rows))
        return _append(rng.choice([2, 3]), rows, t, heads, kv_heads, d,
                       rng.choice([0, d, d, d // 2]), dtype=dtype, page=page,
                       chunks=rng.choice(["all", "mixed", "ragged"]), packed=rng.random() < 0.5)
    layers, order = rng.choice([1, 2, 5]), rng.choice([2, 3])
    rows = _log_int(rng, 2, 40)
    n = _log_int(rng, 1, 2000)
    while layers * rows * kv_heads * (n + page) * d * es * 2 * order > 4e8:
        if layers > 1:
            layers -= 1
        elif n > 1:
            n = n // 2
        else:
            rows = max(2, rows // 2)
    if kind == "fork":
        return _fork(layers, order, rows, _log_int(rng, 1, rows), n, rng.choice([1, 1, _log_int(rng, 2, 40)]),
                     kv_heads, d, dtype=dtype, page=page)
    return _compact(layers, order, rows, n, kv_heads, d, dtype=dtype, page=page)


# ---------------------------------------------------------------------------------------
# inputs, made from the seed alone


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _rng(seed):
    return random.Random(int(seed) * 7919 + 13)


def _lengths(c):
    """(cached positions, new tokens) of every row: the case's, whatever the seed, since shapes follow
    from them."""
    n, t, rows, rng = c["n"], c["t"], c["rows"], random.Random(29)
    lens = [n] * rows
    if c["ragged"]:
        lens = [n] + [max(0, min(n, int(n * rng.random() ** 0.7))) for _ in range(rows - 1)]
        rng.shuffle(lens)
    if c["chunks"] == "mixed":
        new = [1] * rows
        new[rng.randrange(rows)] = t
    elif c["chunks"] == "ragged":
        new = [t] + [rng.randrange(0, t + 1) for _ in range(rows - 1)]
        rng.shuffle(new)
    else:
        new = [t] * rows
    return lens, new


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _table(c, pages, capacity):
    """What names the rows' pages: this package's PageTable, or the same tensors alone."""
    rows, ps = c["rows"], c["page"]
    if own:
        return _package().PageTable(rows, pages=pages, page_size=ps, capacity=capacity, device="cuda")
    most = -(-capacity // ps)

    def i32(*shape):
        return torch.zeros(*shape, dtype=torch.int32, device="cuda")

    return types.SimpleNamespace(page_size=ps, pages=i32(rows, most).sub_(1), counts=i32(rows),
                                 refs=i32(pages), new=i32(rows), starts=i32(rows + 1))


def _cache(c, table):
    """A layer's pages: this package's PagedCache, or the same tensors alone."""
    order, hk, d, ps, dt = c["order"], c["kv_heads"], c["d"], c["page"], _DT[c["dtype"]]
    if own:
        return _package().PagedCache(table, order=order, kv_heads=hk, dim_head=d, dtype=dt)
    pool = table.refs.numel()
    keys, values = ([torch.empty(pool, hk, ps, d, dtype=dt, device="cuda") for _ in range(order)]
                    for _ in range(2))
    lses = [torch.empty(pool, hk, ps, device="cuda") for _ in range(order - 1)]
    return types.SimpleNamespace(keys=keys, values=values, lses=lses)


def _fill(c, cache, g):
    """Keys as a norm leaves them, values, each level's averages (smaller) and logsumexps (about the log
    of the number of positions attended)."""
    for t in range(c["order"]):
        cache.keys[t].normal_(0.0, 1.0, generator=g)
        cache.values[t].normal_(0.0, 0.2 if t else 1.0, generator=g)
    for t, x in enumerate(cache.lses):
        x.normal_(0.0, 0.2, generator=g).add_((t + 1) * (math.log(c["n"] + 1) + 0.5) * 0.9)


def _deal(rows_of_pages, pool, seed):
    """Lists of a row's number of pages -> pages [row] from all over a pool, no two the same."""
    order = random.Random(seed).sample(range(pool), sum(rows_of_pages))
    out, at = [], 0
    for k in rows_of_pages:
        out.append(order[at:at + k])
        at += k
    return out


def _set_table(table, lists, counts, new=None):
    """The state of a table whose row b has the pages lists[b] and counts[b] positions."""
    most = table.pages.shape[1]
    table.pages.copy_(_i32([x + [-1] * (most - len(x)) for x in lists]))
    table.counts.copy_(_i32(counts))
    refs = [0] * table.refs.numel()
    for x in lists:
        for p in x:
            if p >= 0:
                refs[p] += 1
    table.refs.copy_(_i32(refs))
    if new is not None:
        starts = [0]
        for m in new:
            starts.append(starts[-1] + m)
        table.new.copy_(_i32(new))
        table.starts.copy_(_i32(starts))


def _tokens(c, g, new, heads):
    """[rows, heads, t, d], or packed [1, heads, sum of new, d], as a projection's output seen per head."""
    shape = (1, sum(new)) if c["packed"] else (c["rows"], max(new))
    x = torch.randn(*shape, heads, c["d"], generator=g, device="cuda")
    return x.to(_DT[c["dtype"]]).permute(0, 2, 1, 3)


def prepare(case, seed):
    c = case
    g, rng = _gen(seed), _rng(seed)
    ps = c["page"]
    state = {"case": c}
    if c["kind"] in ("attend", "append"):
        lens, new = _lengths(c)
        total = [n + m for n, m in zip(lens, new)]
        need = [-(-x // ps) for x in total]
        if c["kind"] == "append":  # nothing of the cached positions is read: their pages are one
            need = [k - n // ps for k, n in zip(need, lens)]
        pool = sum(need) + 3
        lists = _deal(need, pool - 1, seed)
        if c["kind"] == "append":
            lists = [[pool - 1] * (n // ps) + x for n, x in zip(lens, lists)]
        table = _table(c, pool, max(total))
        _set_table(table, lists, total, new)
        cache = _cache(c, table)
        _fill(c, cache, g)
        state.update(table=table, cache=cache, lens=lens, tokens=new)
        hk, order = c["kv_heads"], c["order"]
        if c["kind"] == "attend":
            state["q1"] = _tokens(c, g, new, c["heads"])
            state["vs"] = [_tokens(c, g, new, hk) for _ in range(order - 2)]
            return state
        state.update(
            eps=1e-6, v=_tokens(c, g, new, hk),
            qs=[_tokens(c, g, new, c["heads"])] + [_tokens(c, g, new, hk) for _ in range(order)],
            weights=[(1.0 + 0.1 * torch.randn(c["d"], generator=g, device="cuda")).to(_DT[c["dtype"]])
                     for _ in range(order + 1)], angles=None)
        if c["rot"]:
            freqs = 10000.0 ** -(torch.arange(0, c["rot"], 2, device="cuda").float() / c["rot"])
            if c["packed"]:
                pos = [[n + i for n, m in zip(lens, new) for i in range(m)]]
            else:
                pos = [[n + i for i in range(max(new))] for n in lens]
            pos = torch.tensor(pos, dtype=torch.float32, device="cuda")
            state["angles"] = (pos[..., None] * freqs).repeat_interleave(2, dim=-1)
        return state
    rows, fixed = c["rows"], random.Random(29)
    if c["kind"] == "fork":
        k = c["prompts"]
        lens = [c["n"] - fixed.randrange(0, max(1, c["n"] // 4)) if b < k else 0 for b in range(rows)]
        index = [b % k if b < k or rng.random() < 0.95 else -1 for b in range(rows)]
        pool = sum(-(-n // ps) for n in lens) + rows * (1 + -(-c["t"] // ps))
        capacity = c["n"] + c["t"]
    else:
        lens = [max(1, int(c["n"] * fixed.random() ** 0.5)) for _ in range(rows)]
        index, pool, capacity = None, sum(-(-n // ps) for n in lens), c["n"]
    lists = _deal([-(-n // ps) for n in lens], pool, seed)
    if c["kind"] == "compact":  # half of the rows have ended
        ended = set(rng.sample(range(rows), rows // 2))
        lists = [[] if b in ended else x for b, x in enumerate(lists)]
        lens = [0 if b in ended else n for b, n in enumerate(lens)]
    table = _table(c, pool, capacity)
    _set_table(table, lists, lens)
    state.update(table=table, caches=[_cache(c, table) for _ in range(c["layers"])],
                 saved=[x.clone() for x in (table.pages, table.counts, table.refs)])
    for cache in state["caches"]:
        _fill(c, cache, g)
    if index is not None:
        state.update(index=_i32(index), more=_i32([c["t"] if i >= 0 else 0 for i in index]))
    return state


# ---------------------------------------------------------------------------------------
# one pass


def run(state):
    c = state["case"]
    kind = c["kind"]
    if not own:
        with torch.no_grad():
            return _PLAIN[kind](state)
    if kind == "attend":
        cache = state["cache"]
        out = cache.attend(state["q1"], state["vs"], scale=c["d"] ** -0.5,
                           softclamp=c["softclamp"] or None)
        return {"out": out, "values": list(cache.values[1:]), "lses": list(cache.lses)}
    if kind == "append":
        cache = state["cache"]
        q1 = cache.append(state["qs"], state["v"], state["weights"], eps=state["eps"],
                          angles=state["angles"])
        return {"q1": q1, "keys": list(cache.keys), "value": cache.values[0]}
    table = state["table"]
    _restore(state)  # every pass begins where the first one began
    if kind == "fork":
        table.select(state["index"])
        table.extend(state["more"])
    else:
        table.compact()
    return _pool_outputs(state)


def _restore(state):
    table = state["table"]
    for to, x in zip((table.pages, table.counts, table.refs), state["saved"]):
        to.copy_(x)


def _pool_outputs(state):
    table = state["table"]
    out = {"pages": table.pages, "counts": table.counts, "refs": table.refs,
           "caches": [[*x.keys, *x.values, *x.lses] for x in state["caches"]]}
    if state["case"]["kind"] == "fork":
        out.update(new=table.new, starts=table.starts)
    return out


def _plain_places(state):
    """Of the padded chunks [rows, t]: the tokens' places in the (padded or packed) inputs, whether
    they are there, and their positions."""
    c, table = state["case"], state["table"]
    rows, t = c["rows"], max(state["tokens"])
    i = torch.arange(t, device="cuda")
    here = i < table.new[:, None]
    pos = (table.counts - table.new)[:, None] + i
    if c["packed"]:
        at = (table.starts[:-1, None] + i).clamp(max=sum(state["tokens"]) - 1)
        batch = torch.zeros_like(at)
    else:
        at = i.expand(rows, t)
        batch = torch.arange(rows, device="cuda")[:, None].expand(rows, t)
    return batch, at, here, pos


def _plain_slots(state, here, pos):
    """(rows, tokens, pages, places inside them) of the tokens that are there."""
    table, ps = state["table"], state["case"]["page"]
    b, i = torch.nonzero(here, as_tuple=True)
    p = pos[b, i].long()
    return b, i, table.pages[b, p // ps].long(), p % ps


def _plain_gather(table, x, most, ps):
    """Positions [rows, heads, most, ...] of an array of pages."""
    ix = table.pages[:, :-(-most // ps)].long().clamp(min=0)
    y = x[ix].transpose(1, 2)
    return y.reshape(*y.shape[:2], -1, *y.shape[4:])[:, :, :most].float()


def _plain_attend(state):
    c, table, x = state["case"], state["table"], state["cache"]
    rows, ps, order, hk, d = c["rows"], c["page"], c["order"], c["kv_heads"], c["d"]
    dt = _DT[c["dtype"]]
    rep = c["heads"] // hk
    t = max(state["tokens"])
    most = max(n + m for n, m in zip(state["lens"], state["tokens"]))
    batch, at, here, pos = _plain_places(state)
    b, i, page, slot = _plain_slots(state, here, pos)
    j = torch.arange(most, device="cuda")
    sees = (j <= pos[..., None]) & here[..., None]                      # [rows, t, most]
    there = (j < table.counts[:, None])[:, None, :, None]
    out = torch.zeros_like(state["q1"])
    for lvl in range(order):
        last = lvl == order - 1
        if last:
            q = state["q1"][batch, :, at].float()                       # [rows, t, heads, d]
            q = q.view(rows, t, hk, rep, d).permute(0, 2, 3, 1, 4)
        else:
            q = _plain_gather(table, x.keys[lvl + 1], most, ps)
            q = q.gather(2, pos.long().clamp(0, most - 1)[:, None, :, None].expand(rows, hk, t, d))[:, :, None]
        k = _plain_gather(table, x.keys[lvl], most, ps)
        v = _plain_gather(table, x.values[lvl], most, ps).masked_fill(~there, 0.0)
        s = torch.matmul(q.reshape(rows, hk, -1, d), k.transpose(2, 3)).mul_(d ** -0.5)
        if c["softclamp"]:
            s = s.div_(c["softclamp"]).tanh_().mul_(c["softclamp"])
        if lvl:
            s += _plain_gather(table, x.lses[lvl - 1], most, ps)[:, :, None]
        s = s.view(rows, hk, -1, t, most).masked_fill_(~sees[:, None, None], -math.inf)
        top = s.amax(-1, keepdim=True).clamp(min=-3e38)
        e = torch.exp(s.sub_(top))
        z = e.sum(-1, keepdim=True)
        o = torch.matmul(e.view(rows, hk, -1, most), v).view(rows, hk, -1, t, d) / z
        if last:
            o = o.permute(0, 3, 1, 2, 4).reshape(rows, t, hk * rep, d)
            out[batch[b, i], :, at[b, i]] = o[b, i].to(dt)
            break
        o = o[:, :, 0].transpose(1, 2)[b, i]                            # [tokens, hk, d]
        if lvl + 1 < order - 1:
            o = o * state["vs"][order - 3 - lvl][batch[b, i], :, at[b, i]].float()
        x.values[lvl + 1][page, :, slot] = o.to(dt)
        x.lses[lvl][page, :, slot] = (top + torch.log(z))[:, :, 0, :, 0].transpose(1, 2)[b, i]
    return {"out": out, "values": list(x.values[1:]), "lses": list(x.lses)}


def _plain_append(state):
    c, x, angles = state["case"], state["cache"], state["angles"]
    dt = _DT[c["dtype"]]
    batch, at, here, pos = _plain_places(state)
    b, i, page, slot = _plain_slots(state, here, pos)
    src = (batch[b, i], slice(None), at[b, i])

    def norm(q, w):
        q = q[src].float()                                              # [tokens, heads, d]
        y = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + state["eps"]) * w.float()
        if angles is None:
            return y.to(dt)
        a = angles[batch[b, i], at[b, i]][:, None]
        z = y[..., :a.shape[-1]]
        turned = torch.stack([-z[..., 1::2], z[..., 0::2]], -1).flatten(-2)
        return torch.cat([z * a.cos() + turned * a.sin(), y[..., a.shape[-1]:]], -1).to(dt)

    ys = [norm(q, w) for q, w in zip(state["qs"], state["weights"])]
    q1 = torch.zeros_like(state["qs"][0])
    q1[src] = ys[0]
    for to, y in zip((*reversed(x.keys), x.values[0]), (*ys[1:], state["v"][src])):
        to[page, :, slot] = y
    return {"q1": q1, "keys": list(x.keys), "value": x.values[0]}


def _plain_select(table, index):
    """Row b becomes what row index[b] was, with its pages; -1: nothing."""
    ps = table.page_size
    old, pool = table.pages.long(), table.refs.numel()
    src = index.long().clamp(min=0)
    counts = torch.where(index >= 0, table.counts[src], 0)
    place = torch.arange(old.shape[1], device=old.device)
    new = torch.where(place < ((counts + ps - 1) // ps)[:, None], old[src], -1)
    more = torch.bincount((new + 1).view(-1), minlength=pool + 1) - torch.bincount((old + 1).view(-1), minlength=pool + 1)
    table.refs += more[1:].to(torch.int32)
    table.pages.copy_(new)
    table.counts.copy_(counts)


def _plain_extend(table, caches, more):
    """Every row gets more[b] further positions: pages for them, the lowest free ones in the order of
    the rows, and a copy of a page that is shared and about to be written.  A row whose pages are not
    to be had gets none."""
    ps, pool = table.page_size, table.refs.numel()
    rows, most = table.pages.shape
    pages, counts = table.pages.long(), table.counts.long()
    m = more.long()
    m = torch.where(counts + m <= most * ps, m, 0)
    place = torch.arange(most, device=pages.device)
    have, want = (counts + ps - 1) // ps, (counts + m + ps - 1) // ps
    part = counts % ps
    tail = pages.gather(1, (counts // ps).clamp(max=most - 1)[:, None])[:, 0]
    writes = (m > 0) & (part > 0)
    # the rows before this one that write the same page: all but the last row that shares it copy it
    row = torch.arange(rows, device=pages.device)
    before = ((tail[:, None] == tail) & writes & (row < row[:, None])).sum(1)
    copies = writes & (table.refs[tail.clamp(min=0)] - before > 1)
    need = (want - have) * (m > 0) + copies
    upto = torch.cumsum(need, 0)
    free = table.refs == 0
    # a page that an earlier row has to leave first waits for that row's own pages
    ok = (m > 0) & ((upto <= free.sum()) | ((need == 0) & ~(writes & (before > 0))))
    found = torch.sort((~free).to(torch.int8), stable=True).indices  # the free pages, lowest first
    first = upto - need                                              # of a row, in the list of free pages
    start = torch.where(copies, counts // ps, have)
    fresh = ok[:, None] & (place >= start[:, None]) & (place < want[:, None])
    ix = (first[:, None] + place - start[:, None]).clamp(0, pool - 1)
    table.pages.copy_(torch.where(fresh, found[ix], pages))
    b = torch.nonzero(ok & copies)[:, 0]
    src, dst = tail[b], found[first[b]]
    table.refs.index_add_(0, src, torch.full_like(src, -1, dtype=torch.int32))
    table.refs[found[ix[fresh]]] = 1
    kept = (torch.arange(ps, device=pages.device) < part[b, None])[:, None]
    for cache in caches:
        for x in (*cache.keys, *cache.values, *cache.lses):
            k = kept[..., None] if x.dim() == 4 else kept
            x[dst] = torch.where(k, x[src], x[dst])
    m = torch.where(ok, m, 0)
    table.counts.copy_(counts + m)
    table.new.copy_(m)
    table.starts[1:] = torch.cumsum(more, 0)
    table.starts[0] = 0


def _plain_fork(state):
    table = state["table"]
    _restore(state)
    _plain_select(table, state["index"])
    _plain_extend(table, state["caches"], state["more"])
    return _pool_outputs(state)


def _plain_compact(state):
    table = state["table"]
    _restore(state)
    used = table.refs > 0
    number = used.sum()
    at = torch.arange(table.refs.numel(), device="cuda")
    src = torch.nonzero(used & (at >= number))[:, 0]
    dst = torch.nonzero(~used & (at < number))[:, 0]
    for cache in state["caches"]:
        for x in (*cache.keys, *cache.values, *cache.lses):
            x[dst] = x[src]
    to = at.clone()
    to[src] = dst
    pages = table.pages.long()
    table.pages.copy_(torch.where(pages >= 0, to[pages.clamp(min=0)], pages))
    table.refs[dst] = table.refs[src]
    table.refs[src] = 0
    return _pool_outputs(state)


_PLAIN = {"attend": _plain_attend, "append": _plain_append, "fork": _plain_fork,
          "compact": _plain_compact}


# ---------------------------------------------------------------------------------------
# what a pass cannot do without


def work(case):
    c = case
    d, es, hk, order = c["d"], _ES[c["dtype"]], c["kv_heads"], c["order"]
    position = hk * (2 * order * d * es + (order - 1) * 4)  # of all levels
    if c["kind"] == "attend":
        lens, new = _lengths(c)
        pairs = sum(m * n + m * (m + 1) // 2 for n, m in zip(lens, new))
        h, tokens = c["heads"], sum(new)
        # every cached key, value and logsumexp, the chunks' own, the queries and outputs, and what the
        # levels leave for the next ones
        total = sum(n + m for n, m in zip(lens, new) if m)
        size = total * position + 2 * tokens * h * d * es
        size += tokens * hk * ((order - 1) * (d * es + 4) + (order - 2) * d * es)
        return {"bytes": size, "flops": 4 * d * pairs * (h + (order - 1) * hk)}
    if c["kind"] == "append":
        _, new = _lengths(c)
        elems = sum(new) * d * (c["heads"] + (order + 1) * hk)
        return {"bytes": 2 * elems * es + sum(new) * c["rot"] * 4 + (order + 1) * d * es,
                "flops": 8 * elems}
    ps, rows = c["page"], c["rows"]
    if c["kind"] == "fork":
        # the pages that are shared and written are copied (about half of each is held), the table twice
        most = -(-(c["n"] + c["t"]) // ps)
        copies = max(1, rows - c["prompts"])
        return {"bytes": 2 * c["layers"] * copies * position * (ps // 2) + 4 * rows * most * 4,
                "flops": rows}
    # about a quarter of the pool's pages are in use behind the ones that are free
    used = sum(max(1, int(c["n"] * 0.67)) for _ in range(rows)) / 2
    return {"bytes": int(2 * c["layers"] * position * used / 2), "flops": rows}


# ---------------------------------------------------------------------------------------
# the definitions in 64 bits


def exact(case, seed):
    global own
    if case["kind"] in ("fork", "compact"):
        return None  # values moved, none computed
    was, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = was
    with torch.no_grad():
        return _exact_append(state) if case["kind"] == "append" else _exact_attend(state)


def _exact_rows(state):
    """(row, its new tokens' places in the inputs, all its pages and places of positions 0 .. total)."""
    c, table = state["case"], state["table"]
    pages, at = table.pages.tolist(), 0
    for b, (n, m) in enumerate(zip(state["lens"], state["tokens"])):
        if m == 0:
            continue
        p = torch.arange(n + m, device="cuda")
        page = torch.tensor(pages[b], device="cuda")[p // c["page"]]
        where = (0, slice(at, at + m)) if c["packed"] else (b, slice(0, m))
        at += m
        yield n, m, where, page, p % c["page"]


def _exact_append(state):
    x = state["cache"]
    q1 = torch.zeros_like(state["qs"][0], dtype=torch.float64)
    keys = [k.double() for k in x.keys]
    value = x.values[0].double()
    for n, m, (b, new), page, slot in _exact_rows(state):
        ys = []
        for q, w in zip(state["qs"], state["weights"]):
            y = q[b, :, new].double()
            y = y / torch.sqrt(y.square().sum(-1, keepdim=True) / y.shape[-1] + state["eps"]) * w.double()
            if state["angles"] is not None:
                a = state["angles"][b, new].double()
                z = y.clone()
                for i in range(0, a.shape[-1], 2):
                    y0, y1 = y[..., i], y[..., i + 1]
                    z[..., i] = y0 * torch.cos(a[..., i]) - y1 * torch.sin(a[..., i])
                    z[..., i + 1] = y1 * torch.cos(a[..., i + 1]) + y0 * torch.sin(a[..., i + 1])
                y = z
            ys.append(y)
        q1[b, :, new] = ys[0]
        for to, y in zip((*keys[::-1], value), (*ys[1:], state["v"][b, :, new].double())):
            to[page[n:], :, slot[n:]] = y.transpose(0, 1)
    return {"q1": q1, "keys": keys, "value": value}


def _exact_attend(state):
    """Row by row and head by head: weight(i, j) = exp(score) over the positions up to token i, the
    average weighted with them and the logsumexp the log of their sum.  What the cache holds has the
    cache's type: the next level reads each stored average rounded to it."""
    c, x = state["case"], state["cache"]
    hk, d, order, dt = c["kv_heads"], c["d"], c["order"], _DT[c["dtype"]]
    rep = c["heads"] // hk
    out = torch.zeros_like(state["q1"], dtype=torch.float64)
    values = [v.double() for v in x.values]
    lses = [z.double() for z in x.lses]
    for n, m, (b, new), page, slot in _exact_rows(state):
        hidden = torch.arange(n + m, device="cuda") > torch.arange(n, n + m, device="cuda")[:, None]
        for h in range(hk):
            def row(t):
                return t[page, h, slot].double()

            bias = below = None
            for lvl in range(order):
                last = lvl == order - 1
                k = row(x.keys[lvl])
                v = row(x.values[lvl])
                if lvl:  # this step's, as the cache holds them
                    v[n:] = below
                for r in range(rep if last else 1):
                    q = state["q1"][b, h * rep + r, new].double() if last else row(x.keys[lvl + 1])[n:]
                    s = q @ k.t() / math.sqrt(d)
                    if c["softclamp"]:
                        s = c["softclamp"] * torch.tanh(s / c["softclamp"])
                    if lvl:
                        s = s + bias
                    s[hidden] = -math.inf
                    z = torch.logsumexp(s, -1)
                    o = torch.exp(s - z[:, None]) @ v
                    if last:
                        out[b, h * rep + r, new] = o
                if not last:
                    if lvl + 1 < order - 1:
                        o = o * state["vs"][order - 3 - lvl][b, h, new].double()
                    values[lvl + 1][page[n:], h, slot[n:]] = o
                    lses[lvl][page[n:], h, slot[n:]] = z
                    below = o.to(dt).double()
                    bias = lses[lvl][page, h, slot]
    return {"out": out, "values": values[1:], "lses": lses}
