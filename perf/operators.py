"""The operators of a drafted decoding step, as cases that can be timed.

A serving loop drafts a few tokens for every row of a batch, has the model look at all of them in one
step, keeps the ones that the model would have produced itself and goes on behind them.  The drafted
tokens of a row form a tree: ``parents[b, t]`` is the node that node t follows (lower than t), -1 a
node that follows the cached positions, anything else no node at all.  Four kinds of case:

* ``append`` -- the query/key norms, the rotary embedding at each node's position and the writes
  into the cache's draft slots, for one layer;
* ``attend`` -- every level of the poly attention for all nodes: a node attends to its row's
  cached positions, to its ancestors and to itself;
* ``verify`` -- the walk down the tree against the target's probabilities, from given random
  numbers, and the token that follows the last node kept;
* ``commit`` -- the kept nodes of every layer move behind the cached positions and the rows'
  position counts advance.
"""

import math
import os
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
# cases


def _attend(order, b, n, t, heads, kv_heads, d, dtype="bf16", tree="tree", ragged=True,
            softclamp=0.0):
    return {"kind": "attend", "order": order, "b": b, "n": n, "t": t, "heads": heads,
            "kv_heads": kv_heads, "d": d, "dtype": dtype, "tree": tree, "ragged": ragged,
            "softclamp": softclamp}


def _append(order, b, t, heads, kv_heads, d, rot, dtype="bf16", tree="tree"):
    return {"kind": "append", "order": order, "b": b, "n": 8192, "t": t, "heads": heads,
            "kv_heads": kv_heads, "d": d, "rot": rot, "dtype": dtype, "tree": tree,
            "ragged": True}


def _verify(b, t, vocab, dtype="bf16", tree="tree", probs=False, greedy="none"):
    return {"kind": "verify", "b": b, "t": t, "vocab": vocab, "dtype": dtype, "tree": tree,
            "probs": probs, "greedy": greedy}


def _commit(layers, order, b, n, t, kv_heads, d, dtype="bf16"):
    return {"kind": "commit", "layers": layers, "order": order, "b": b, "n": n, "t": t,
            "kv_heads": kv_heads, "d": d, "dtype": dtype, "tree": "tree"}


def listed():
    cases = {
        # one user's short conversation, a handful of drafted tokens: latency
        "attend_one_user": _attend(2, 1, 300, 5, 8, 8, 64),
        # the grouped-query layer over a long cache (bench.py's config 5), eight drafts in a row
        "attend_gqa_long": _attend(2, 32, 8192, 8, 32, 8, 128, tree="chain"),
        # an order-3 layer (bench.py's config 4) with a tree of sixteen drafts, ragged rows
        "attend_order3_tree": _attend(3, 8, 2048, 16, 16, 16, 64),
        # no drafts at all: one token a row, rows of very different lengths, f16
        "attend_token_ragged": _attend(2, 7, 21333, 1, 16, 4, 128, dtype="f16"),
        # full precision, a wide tree, soft-clamped scores, a head dim between the usual ones
        "attend_f32_wide": _attend(2, 3, 1111, 33, 8, 2, 96, dtype="f32", softclamp=50.0),
        # the norms and rotary of the grouped-query layer's drafts
        "append_gqa": _append(2, 32, 8, 32, 8, 128, 128),
        # the same of a small order-3 layer for one user, half of each head rotated: latency
        "append_one_user": _append(3, 1, 5, 8, 8, 64, 32, dtype="f16"),
        # bytes as tokens (the reference's own training script), one user, greedy: latency
        "verify_bytes": _verify(1, 5, 256, dtype="f32", greedy="all"),
        # a batch of trees of drafts a small model ranked first, sampled and greedy rows
        "verify_trees": _verify(32, 16, 32000, greedy="some"),
        # drafts sampled from a draft model's own distribution over a large vocabulary
        "verify_sampled": _verify(8, 6, 128256, dtype="f32", tree="chain", probs=True),
        # the caches of six order-3 layers (of bench.py's config 4) after a step of sixteen drafts
        "commit_model": _commit(6, 3, 8, 150, 16, 16, 64),
        # one grouped-query layer, one user: latency
        "commit_one_user": _commit(1, 2, 1, 301, 5, 8, 64),
    }
    return [dict(c, name=k) for k, c in cases.items()]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "append", "verify", "verify", "commit"])
    tree = rng.choice(["tree", "tree", "chain", "sparse"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    t = rng.choice([1, _log_int(rng, 2, 64), _log_int(rng, 2, 24)])
    kv_heads = rng.choice([1, 2, 4, 8, 16])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 8])
    d = rng.choice([64, 64, 128, 128, 32, 96, 40])
    if kind == "attend":
        order = rng.choice([2, 2, 2, 3, 4])
        b = _log_int(rng, 1, 48)
        # at most about a quarter of the largest listed case's bytes and products
        most = 5e8 / (b * kv_heads * d * _ES[dtype] * (3 * order - 2))
        most = min(most, 4e10 / (4.0 * b * t * d * (heads + (order - 1) * kv_heads)))
        if dtype == "f32":
            most /= 4
        n = _log_int(rng, 1, max(2, min(32768, int(most))))
        return _attend(order, b, n, t, heads, kv_heads, d, dtype=dtype, tree=tree,
                       ragged=rng.random() < 0.7, softclamp=rng.choice([0.0, 0.0, 30.0]))
    if kind == "append":
        return _append(rng.choice([2, 3]), _log_int(rng, 1, 64), min(t, 32), heads, kv_heads, d,
                       rng.choice([0, d, d, d // 2]), dtype=dtype, tree=tree)
    if kind == "verify":
        b = _log_int(rng, 1, 32)
        vocab = rng.choice([256, 1009, _log_int(rng, 256, 150000), 32000])
        t = max(1, min(t, int(3e7 / (b * vocab))))
        return _verify(b, t, vocab, dtype=dtype, tree=tree, probs=rng.random() < 0.4,
                       greedy=rng.choice(["none", "none", "some", "all"]))
    d = min(d, 128)
    b = _log_int(rng, 1, 16)
    t = min(t, 32)
    layers = rng.choice([1, 2, 5])
    order = rng.choice([2, 3])
    n = _log_int(rng, 1, 400)
    while layers * b * kv_heads * (n + t) * d * _ES[dtype] * (3 * order - 2) > 1.2e8:
        if layers > 1:
            layers -= 1
        elif b > 1:
            b -= 1
        else:
            n = max(1, n // 2)
    return _commit(layers, order, b, n, t, kv_heads, d, dtype=dtype)


# ---------------------------------------------------------------------------------------
# inputs, made from the seed alone


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _rng(seed):
    import random

    return random.Random(int(seed) * 7919 + 13)


def _make_tree(c, rng):
    """parents [b][t] as a drafter makes them: a chain; a tree whose nodes follow the level before
    them; ``sparse`` trees of fewer nodes than there is room for, some rows without any."""
    rows = []
    for _ in range(c["b"]):
        t, p = c["t"], [-1]
        for i in range(1, t):
            if c["tree"] == "chain":
                p.append(i - 1)
            else:
                p.append(rng.randrange(max(0, (i - 1) // 2 - 1), max(1, min(i, (i + 1) // 2 + 1))))
        if c["tree"] == "sparse":
            keep = rng.randrange(0, t + 1)
            p = [x if i < keep else -2 for i, x in enumerate(p)]
        rows.append(p)
    return rows


def _make_lengths(c, rng):
    n = c["n"]
    if not c.get("ragged"):
        return [n] * c["b"]
    # the longest row is full, the others anything down to a prompt of a few tokens
    lens = [n] + [max(0, min(n, int(n * rng.random() ** 0.7))) for _ in range(c["b"] - 1)]
    rng.shuffle(lens)
    return lens


def _depths(parents):
    out = []
    for p in parents:
        d = []
        for i, x in enumerate(p):
            d.append(d[x] + 1 if 0 <= x < i else 0)
        out.append(d)
    return out


def _i32(rows):
    return torch.tensor(rows, dtype=torch.int32, device="cuda")


def _cache(c, capacity, counts):
    """The buffers of one layer's cache: this package's DraftCache, or the same tensors alone."""
    order, b, hk, d, t = c["order"], c["b"], c["kv_heads"], c["d"], c["t"]
    if own:
        return _package().DraftCache.empty(order=order, batch=b, kv_heads=hk, dim_head=d,
                                           capacity=capacity, max_drafts=t, dtype=_DT[c["dtype"]],
                                           device="cuda", counts=counts)
    dt = _DT[c["dtype"]]

    def rows(m, count):
        return [torch.empty(b, hk, m, d, dtype=dt, device="cuda") for _ in range(count)]

    def lses(m):
        return [torch.empty(b, hk, m, device="cuda") for _ in range(order - 1)]

    return types.SimpleNamespace(
        qs=rows(capacity, order), vs=rows(capacity, order - 1), msgs=rows(capacity, order - 1),
        lses=lses(capacity), draft_qs=rows(t, order), draft_vs=rows(t, order - 1),
        draft_msgs=rows(t, order - 1), draft_lses=lses(t), counts=counts)


def _fill(cache, g):
    """Keys as a norm leaves them, values, each level's outputs (averages of values, so smaller) and
    logsumexps (about the log of the number of positions attended)."""
    for ts, std in ((cache.qs, 1.0), (cache.vs, 1.0), (cache.msgs, 0.2), (cache.draft_qs, 1.0),
                    (cache.draft_vs, 1.0), (cache.draft_msgs, 0.2)):
        for x in ts:
            x.normal_(0.0, std, generator=g)
    for ts in (cache.lses, cache.draft_lses):
        for lvl, x in enumerate(ts):
            rise = torch.log(torch.arange(1, x.shape[2] + 1, device="cuda").float())
            x.normal_(0.0, 0.2, generator=g).add_((lvl + 1) * (rise + 0.5))


def _heads_view(g, c, heads):
    """[b, heads, t, d] as a projection's output seen per head."""
    x = torch.randn(c["b"], c["t"], heads, c["d"], generator=g, device="cuda")
    return x.to(_DT[c["dtype"]]).permute(0, 2, 1, 3)


def prepare(case, seed):
    c = case
    g, rng = _gen(seed), _rng(seed)
    parents = _make_tree(c, rng)
    state = {"case": c, "parents": _i32(parents)}
    if c["kind"] == "attend":
        lens = _make_lengths(c, rng)
        cache = _cache(c, c["n"] + c["t"], _i32(lens))
        _fill(cache, g)
        q1 = _heads_view(g, c, c["heads"])
        state.update(cache=cache, q1=q1, lens=lens)
    elif c["kind"] == "append":
        lens = _make_lengths(c, rng)
        cache = _cache(c, 8, _i32([0] * c["b"]))  # nothing of the cached positions is read here
        hk, order = c["kv_heads"], c["order"]
        state.update(
            cache=cache, eps=1e-6,
            qs=[_heads_view(g, c, c["heads"])] + [_heads_view(g, c, hk) for _ in range(order)],
            vs=[_heads_view(g, c, hk) for _ in range(order - 1)],
            weights=[(1.0 + 0.1 * torch.randn(c["d"], generator=g, device="cuda")).to(_DT[c["dtype"]])
                     for _ in range(order + 1)], angles=None)
        if c["rot"]:
            pos = torch.tensor([[n + x for x in row] for n, row in zip(lens, _depths(parents))],
                               device="cuda", dtype=torch.float32)
            freqs = 10000.0 ** -(torch.arange(0, c["rot"], 2, device="cuda").float() / c["rot"])
            state["angles"] = (pos[..., None] * freqs).repeat_interleave(2, dim=-1)
    elif c["kind"] == "verify":
        state.update(_verify_inputs(c, g, rng, parents))
    else:
        lens = [rng.randrange(0, c["n"] + 1) for _ in range(c["b"])]
        counts = _i32(lens)
        caches = []
        for _ in range(c["layers"]):
            cache = _cache(c, c["n"] + c["t"], counts)  # one position count for all layers
            _fill(cache, g)
            caches.append(cache)
        path, kept = [], []
        for p in parents:
            # some way down the tree
            node, row = 0, [0]
            while rng.random() < 0.75:
                below = [i for i, x in enumerate(p) if x == node]
                if not below:
                    break
                node = rng.choice(below)
                row.append(node)
            kept.append(len(row))
            path.append(row + [-1] * (c["t"] - len(row)))
        state.update(caches=caches, start=counts.clone(), path=_i32(path), kept=_i32(kept))
    return state


def _verify_inputs(c, g, rng, parents):
    b, t, v = c["b"], c["t"], c["vocab"]
    logits = 2.0 * torch.randn(b, t, v, generator=g, device="cuda")
    temp = torch.ones(b, device="cuda")
    if c["greedy"] == "all":
        temp.zero_()
    else:
        temp.copy_(torch.tensor([rng.choice([0.7, 1.0, 1.3]) for _ in range(b)]))
        if c["greedy"] == "some":
            temp[::3] = 0.0
    par = torch.tensor(parents, device="cuda").clamp(min=0)
    # distinct tokens in a row
    first, step = ([rng.randrange(1, m) for _ in range(b)] for m in (v, v // t))
    slot = torch.arange(t, device="cuda")
    tokens = (torch.tensor(first, device="cuda")[:, None]
              + torch.tensor(step, device="cuda")[:, None] * slot) % v
    probs = None
    if c["probs"]:
        # the draft model agrees with the target for the most part; its tokens are drawn from it
        probs = torch.randn(b, t, v, generator=g, device="cuda").mul_(0.7).add_(logits)
        probs = torch.softmax(probs.mul_(1.5), dim=-1)
        drawn = torch.multinomial(probs.view(b * t, v), t, replacement=True, generator=g)
        drawn = drawn.view(b, t, t)
        tokens = drawn[torch.arange(b, device="cuda")[:, None], par, slot[None, :]]
    else:
        # the drafter ranked these tokens first, and the target finds them likely too
        lse = torch.logsumexp(logits, dim=-1)
        share = torch.tensor([[0.15 + 0.8 * rng.random() for _ in range(t)] for _ in range(b)],
                             device="cuda")
        up = lse.gather(1, par) + torch.log(share / (1.0 - share))
        rows = torch.arange(b, device="cuda")[:, None].expand(b, t)
        logits[rows, par, tokens] = up
    u = torch.rand(b, t, generator=g, device="cuda")
    noise = torch.empty(b, v, device="cuda").exponential_(generator=g).clamp_(min=1e-20)
    return {"logits": logits.to(_DT[c["dtype"]]), "tokens": tokens, "uniforms": u, "noise": noise,
            "temperature": temp, "draft_probs": probs}


# ---------------------------------------------------------------------------------------
# one pass


def run(state):
    c = state["case"]
    if not own:
        with torch.no_grad():
            return _PLAIN[c["kind"]](state)
    kind = c["kind"]
    if kind == "attend":
        cache, t = state["cache"], c["t"]
        out = cache.attend(state["q1"], parents=state["parents"], scale=c["d"] ** -0.5,
                           softclamp=c["softclamp"] or None)
        return {"out": out, "msgs": list(cache.draft_msgs), "lses": list(cache.draft_lses)}
    if kind == "append":
        cache = state["cache"]
        q1 = cache.append(state["qs"], state["vs"], state["weights"], eps=state["eps"],
                          parents=state["parents"], angles=state["angles"])
        return {"q1": q1, "qs": list(cache.draft_qs), "vs": list(cache.draft_vs)}
    pa = _package()
    if kind == "verify":
        path, kept, token = pa.verify_drafts(
            state["logits"], state["tokens"], state["parents"], uniforms=state["uniforms"],
            noise=state["noise"], temperature=state["temperature"],
            draft_probs=state["draft_probs"])
        return {"path": path, "kept": kept, "token": token}
    caches = state["caches"]
    caches[0].counts.copy_(state["start"])  # every pass begins where the step began
    pa.commit_drafts(caches, state["path"], state["kept"])
    return _commit_outputs(caches)


def _commit_outputs(caches):
    return {"counts": caches[0].counts,
            "caches": [[*x.qs, *x.vs, *x.lses, *x.msgs] for x in caches]}


def _plain_tree(parents):
    """live [b, t], anc [b, t, t] (node, ancestor or itself) of a [b, t] tensor of parents."""
    b, t = parents.shape
    slot = torch.arange(t, device=parents.device)
    inner = (parents >= 0) & (parents < slot)
    live, anc = [], []
    for i in range(t):
        p = parents[:, i].clamp(0, t - 1).long()
        row = torch.zeros(b, t, dtype=torch.bool, device=parents.device)
        ok = parents[:, i] == -1
        if i:
            sel = torch.stack(anc, 1).gather(1, p.clamp(max=i - 1)[:, None, None].expand(b, 1, t))
            row = sel[:, 0] & inner[:, i, None]
            ok = ok | (inner[:, i] & torch.stack(live, 1).gather(1, p.clamp(max=i - 1)[:, None])[:, 0])
        live.append(ok)
        anc.append((row | (slot == i)) & ok[:, None])
    return torch.stack(live, 1), torch.stack(anc, 1)


def _plain_attend(state):
    c, x, q1 = state["case"], state["cache"], state["q1"]
    t, order, hk = c["t"], c["order"], c["kv_heads"]
    rep, scale, dt = c["heads"] // hk, c["d"] ** -0.5, q1.dtype
    live, anc = _plain_tree(state["parents"])
    out = torch.empty_like(q1)
    for b, n in enumerate(state["lens"]):
        ok = live[b][None, :, None]
        msg = lse = None
        for lvl in range(order - 1, -1, -1):
            src = order - 2 - lvl  # the msg / lse of the level below, deepest first
            q = q1[b] if lvl == 0 else x.draft_qs[lvl - 1][b]
            group = rep if lvl == 0 else 1
            q = q.float().reshape(hk, group * t, -1)
            k = torch.cat([x.qs[lvl][b, :, :n], x.draft_qs[lvl][b]], 1).float()
            s = torch.matmul(q, k.transpose(1, 2)) * scale
            if c["softclamp"]:
                s = c["softclamp"] * torch.tanh(s / c["softclamp"])
            if lvl < order - 1:
                s = s + torch.cat([x.lses[src][b, :, :n], lse], 1)[:, None]
            s = s.view(hk, group, t, n + t)
            s[..., n:] = s[..., n:].masked_fill(~anc[b], -math.inf)
            if lvl == order - 1:
                v = torch.cat([x.vs[-1][b, :, :n], x.draft_vs[-1][b]], 1).float()
            else:
                v = torch.cat([x.msgs[src][b, :, :n].float(), msg], 1)
                if lvl:
                    v = v * torch.cat([x.vs[lvl - 1][b, :, :n], x.draft_vs[lvl - 1][b]], 1).float()
            top = s.amax(-1, keepdim=True).clamp(min=-3e38)
            e = torch.exp(s - top)
            z = e.sum(-1, keepdim=True)
            o = torch.matmul((e / z).view(hk, group * t, n + t), v)
            o = o.view(hk, group, t, -1)
            if lvl == 0:
                out[b] = torch.where(ok, o.reshape(hk * group, t, -1), 0.0).to(dt)
            else:
                msg = torch.where(ok, o[:, 0], 0.0)
                lse = torch.where(ok[..., 0], (top + torch.log(z))[:, 0, :, 0], 0.0)
                x.draft_msgs[src + 1][b] = msg.to(dt)
                x.draft_lses[src + 1][b] = lse
    return {"out": out, "msgs": list(x.draft_msgs), "lses": list(x.draft_lses)}


def _plain_append(state):
    x, angles = state["cache"], state["angles"]

    def norm(q, w):
        q = q.float()
        y = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + state["eps"]) * w.float()
        if angles is None:
            return y
        r = angles.shape[-1]
        a = angles[:, None]
        z = y[..., :r]
        turned = torch.stack([-z[..., 1::2], z[..., 0::2]], -1).flatten(-2)
        return torch.cat([z * a.cos() + turned * a.sin(), y[..., r:]], -1)

    dt = state["qs"][0].dtype
    ys = [norm(q, w).to(dt) for q, w in zip(state["qs"], state["weights"])]
    for to, y in zip((*x.draft_qs, *x.draft_vs), (*ys[1:], *state["vs"])):
        to.copy_(y)
    return {"q1": ys[0], "qs": list(x.draft_qs), "vs": list(x.draft_vs)}


def _plain_verify(state):
    """In 64 bits: a test against a random number is next to its border now and then."""
    c = state["case"]
    b, t, v = c["b"], c["t"], c["vocab"]
    parents, tokens, u, q = state["parents"], state["tokens"], state["uniforms"], state["draft_probs"]
    x, temp = state["logits"].double(), state["temperature"].double()
    ids = torch.arange(v, device=x.device)
    rows = torch.arange(b, device=x.device)
    greedy = temp == 0
    live, _ = _plain_tree(parents)

    def target(node):
        """The target's distribution behind node [b]: softmax(logits / temperature), and where the
        temperature is 0 all of it on the first of the largest logits."""
        y = x[rows, node]
        top = y.amax(-1, keepdim=True)
        first = torch.where(y == top, ids, v).amin(-1, keepdim=True)
        e = torch.exp((y - top) / torch.where(greedy, 1.0, temp)[:, None])
        return torch.where(greedy[:, None], (ids == first).double(), e / e.sum(-1, keepdim=True))

    cur = torch.zeros(b, dtype=torch.long, device=x.device)
    kept = live[:, 0].to(torch.int32)
    path = torch.full((b, t), -1, dtype=torch.int32, device=x.device)
    path[:, 0] = torch.where(live[:, 0], 0, -1)
    p = target(cur)
    for i in range(1, t):
        child = live[:, i] & (parents[:, i] == cur) & live[:, 0]
        tok = tokens[:, i, None]
        px = p.gather(1, tok)[:, 0]
        qx = 1.0 if q is None else q[rows, cur].gather(1, tok)[:, 0].double()
        take = child & (u[:, i].double() * qx < px)
        if q is None:
            rest = p.masked_fill(ids == tok, 0.0)
        else:
            rest = (p - q[rows, cur].double()).clamp(min=0.0)
        z = rest.sum(-1, keepdim=True)
        rest = torch.where(z > 0, rest / z, p)
        cur = torch.where(take, i, cur)
        p = torch.where(take[:, None], target(cur), torch.where((child & ~take)[:, None], rest, p))
        path.scatter_(1, kept.long().clamp(max=t - 1)[:, None],
                      torch.where(take, i, path.gather(1, kept.long().clamp(max=t - 1)[:, None])[:, 0])
                      [:, None].to(torch.int32))
        kept = kept + take.to(torch.int32)
    key = torch.where(p > 0, p / state["noise"].double(), -1.0)
    token = torch.where(key == key.amax(-1, keepdim=True), ids, v).amin(-1)
    return {"path": path, "kept": kept, "token": torch.where(live[:, 0], token, -1)}


def _plain_commit(state):
    caches = state["caches"]
    counts = caches[0].counts
    counts.copy_(state["start"])
    path, kept = state["path"].long().clamp(min=0), state["kept"]
    t = path.shape[1]
    slot = torch.arange(t, device=path.device)
    move = slot[None] < kept[:, None]
    to = counts.long()[:, None] + slot[None]
    for x in caches:
        for dst, src in zip((*x.qs, *x.vs, *x.msgs, *x.lses),
                            (*x.draft_qs, *x.draft_vs, *x.draft_msgs, *x.draft_lses)):
            shape = (*src.shape[:2], t, *src.shape[3:])
            tail = (1,) * (src.dim() - 3)

            def ix(m):
                return m.view(m.shape[0], 1, t, *tail).expand(shape)

            dst.scatter_(2, ix(to), torch.where(ix(move), src.gather(2, ix(path)),
                                                dst.gather(2, ix(to))))
    counts.add_(kept)
    return _commit_outputs(caches)


_PLAIN = {"attend": _plain_attend, "append": _plain_append, "verify": _plain_verify,
          "commit": _plain_commit}


# ---------------------------------------------------------------------------------------
# what a pass cannot do without


def work(case):
    c = case
    b, t, d, es = c["b"], c["t"], c.get("d", 0), _ES[c["dtype"]]
    if c["kind"] == "attend":
        order, h, hk = c["order"], c["heads"], c["kv_heads"]
        total = sum(_make_lengths(c, _counted(c)))
        # every cached key, value, level output and logsumexp of the rows' lengths, the drafts', and
        # the queries and outputs
        rows = total + b * t
        size = rows * hk * ((3 * order - 2) * d * es + (order - 1) * 4)
        size += 2 * b * h * t * d * es + b * t * hk * (order - 1) * (d * es + 4)
        return {"bytes": size, "flops": 4 * d * t * (total + b * t) * (h + (order - 1) * hk)}
    if c["kind"] == "append":
        order, h, hk = c["order"], c["heads"], c["kv_heads"]
        elems = b * t * d * (h + (2 * order - 1) * hk)
        size = 2 * elems * es + b * t * c["rot"] * 4 + (order + 1) * d * es
        return {"bytes": size, "flops": 8 * elems}
    if c["kind"] == "verify":
        v = c["vocab"]
        size = b * t * v * es + b * v * 4 + (b * v * 4 if c["probs"] else 0) + b * t * 16
        return {"bytes": size, "flops": 4 * b * t * v}
    order, hk = c["order"], c["kv_heads"]
    # about half the nodes a way down the tree passes are kept
    kept = b * min(t, 3)
    size = 2 * c["layers"] * kept * hk * ((3 * order - 2) * d * es + (order - 1) * 4)
    return {"bytes": size, "flops": kept}


def _counted(c):
    """The generator of a case's lengths for its work: those of seed 0."""
    rng = _rng(0)
    _make_tree(c, rng)
    return rng


# ---------------------------------------------------------------------------------------
# the definitions in 64 bits


def exact(case, seed):
    global own
    c = case
    if c["kind"] == "verify":
        return None  # tokens and tree nodes: no computed numbers
    if c["kind"] == "commit":
        return None  # values moved, none computed
    was, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = was
    with torch.no_grad():
        return _exact_append(state) if c["kind"] == "append" else _exact_attend(state)


def _exact_append(state):
    x = state["cache"]
    ys = []
    for q, w in zip(state["qs"], state["weights"]):
        y = q.double()
        y = y / torch.sqrt(y.square().sum(-1, keepdim=True) / y.shape[-1] + state["eps"]) * w.double()
        if state["angles"] is not None:
            a = state["angles"].double().unsqueeze(1)
            z = y.clone()
            for i in range(0, a.shape[-1], 2):
                y0, y1 = y[..., i], y[..., i + 1]
                z[..., i] = y0 * torch.cos(a[..., i]) - y1 * torch.sin(a[..., i])
                z[..., i + 1] = y1 * torch.cos(a[..., i + 1]) + y0 * torch.sin(a[..., i + 1])
            y = z
        ys.append(y)
    return {"q1": ys[0], "qs": ys[1:], "vs": [v.double() for v in state["vs"]]}


def _exact_attend(state):
    """Level by level over the whole row: weight(i, j) = exp(score) over the positions that node i
    sees, the output their weighted mean and the logsumexp the log of their sum."""
    c, x = state["case"], state["cache"]
    b, t, h, hk, d, order = c["b"], c["t"], c["heads"], c["kv_heads"], c["d"], c["order"]
    parents = state["parents"].tolist()
    out = torch.zeros(b, h, t, d, dtype=torch.float64, device="cuda")
    msgs = [torch.zeros(b, hk, t, d, dtype=torch.float64, device="cuda") for _ in range(order - 1)]
    lses = [torch.zeros(b, hk, t, dtype=torch.float64, device="cuda") for _ in range(order - 1)]
    for r in range(b):
        n = state["lens"][r]
        sees = torch.zeros(t, n + t, dtype=torch.bool)
        known = []
        for i, p in enumerate(parents[r]):
            known.append(p == -1 or (0 <= p < i and known[p]))
            if known[i]:
                if p >= 0:
                    sees[i] = sees[p]
                sees[i, :n] = True
                sees[i, n + i] = True
        sees = sees.cuda()
        nodes = torch.tensor(known, device="cuda")
        for step in range(order):  # deepest level first
            key = order - 1 - step
            for kv in range(hk):
                k = torch.cat([x.qs[key][r, kv, :n], x.draft_qs[key][r, kv]]).double()
                if step == 0:
                    val = torch.cat([x.vs[-1][r, kv, :n], x.draft_vs[-1][r, kv]]).double()
                else:
                    val = torch.cat([x.msgs[step - 1][r, kv, :n].double(), msgs[step - 1][r, kv]])
                    if key:
                        val = val * torch.cat([x.vs[key - 1][r, kv, :n],
                                               x.draft_vs[key - 1][r, kv]]).double()
                heads = range(kv * (h // hk), (kv + 1) * (h // hk)) if key == 0 else [kv]
                for hh in heads:
                    q = state["q1"][r, hh] if key == 0 else x.draft_qs[key - 1][r, hh]
                    s = q.double() @ k.t() / math.sqrt(d)
                    if c["softclamp"]:
                        s = c["softclamp"] * torch.tanh(s / c["softclamp"])
                    if step:
                        s = s + torch.cat([x.lses[step - 1][r, kv, :n].double(),
                                           lses[step - 1][r, kv]])
                    s = torch.where(sees, s, -math.inf)
                    z = torch.logsumexp(s, -1)
                    o = torch.exp(s - z[:, None]) @ val
                    o = torch.where(nodes[:, None], o, 0.0)
                    if key == 0:
                        out[r, hh] = o
                    else:
                        msgs[step][r, hh] = o
                        lses[step][r, hh] = torch.where(nodes, z, 0.0)
    return {"out": out, "msgs": msgs, "lses": lses}
