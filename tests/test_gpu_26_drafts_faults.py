"""GPU: drafted tokens, cases that once went wrong or could have: each test says which."""

import pytest
import torch

import drafts_oracle as DO
from test_gpu_25_drafts import BUFS, DT, assert_within, dev, fill_cache, make_tree, random_caches

pytestmark = pytest.mark.gpu
param = pytest.mark.parametrize


def test_commit_many_buffers_at_one_count():
    """Every workgroup of a row moves to the count as it was before the call, however many draw their tickets
    before it (the count advances within the launch)."""
    from poly_attention import commit_drafts

    d = dev()
    g = torch.Generator().manual_seed(3)
    B, slots, cap = 5, 8, 200
    caches = random_caches(12, 3, B, 2, 64, cap, slots, [0, 3, 17, 150, 40], "bf16", d, g)  # 120 buffers: one launch
    bufs = [(dst, src) for c in caches for name in BUFS
            for dst, src in zip(getattr(c, name), getattr(c, "draft_" + name))]
    want = [dst.clone() for dst, _ in bufs]
    counts = caches[0].lengths()
    for step in range(12):
        path = torch.stack([torch.randperm(slots, generator=g) for _ in range(B)]).int()
        kept = torch.randint(0, 5, (B,), generator=g).int()
        commit_drafts(caches, path.to(d), kept.to(d))
        for b in range(B):
            for w, (_, src) in zip(want, bufs):
                w[b, :, counts[b]:counts[b] + kept[b]] = src[b][:, path[b, :kept[b]].tolist()]
            counts[b] += int(kept[b])
        assert caches[0].lengths() == counts
        for w, (dst, _) in zip(want, bufs):
            assert torch.equal(dst, w), step


# A weight of a cached position, and a middle level's v * msg, enter the products as two numbers of the type,
# the second of what the first leaves: bf16 is off by at most 2^-16 of the value (8 bits cut off, the rest below 2^-7
# rounded to 8), fp16 by 2^-21 (11, 2^-10 and 11) where it is not among the smallest numbers.  The oracle's bound takes one rounding to
# the type for each (2^-9, 2^-12); in its place, of a weight's value:
def pair(dtype, order):
    return 2.0 ** -15 if dtype == "bf16" or order > 2 else 2.0 ** -18


def attend_pairs(u, q1, host, lens, trees, scale, softclamp=None):
    """The oracle's results, with bounds that one rounding of a weight or of a product does not fit."""
    unit = DO.unit
    try:
        DO.unit = lambda dtype: u
        want, tol = DO.attend(q1, host, lens, trees, scale, softclamp)
    finally:
        DO.unit = unit
    sums = len(want) - len(host["lses"])  # the logsumexps are stored in fp32
    return want, [e + DO.stored(w, q1.dtype) if k < sums else e for k, (w, e) in enumerate(zip(want, tol))]


@param("dtype", ("bf16", "f16"))
@param("order,B,counts,T,H,hk,D,kind", [
    (2, 1, [700], 1, 2, 2, 64, "chain"),
    (2, 2, [300, 41], 5, 8, 2, 128, "tree"),      # 20 rows
    (3, 1, [500], 7, 4, 2, 64, "tree"),
    (4, 2, [129, 350], 3, 2, 1, 40, "forest"),
    (3, 1, [300], 40, 2, 2, 64, "tree"),          # four tiles of a middle level
    (3, 1, [257], 20, 2, 1, 256, "tree"),
    (2, 1, [400], 33, 4, 2, 64, "tree"),          # the blocks of many rows
    (3, 1, [310], 48, 3, 1, 128, "holes"),
])
def test_attend_holds_more_than_one_rounding(dtype, order, B, counts, T, H, hk, D, kind):
    """The outputs are those of fp32 weights and products, rounded once: with weights rounded to the type the
    error was 1.2 to 1.5 times that of the output's rounding alone."""
    from poly_attention import DraftCache

    d = dev()
    g = torch.Generator().manual_seed(order * 100 + T)
    cache = DraftCache.empty(order=order, batch=B, kv_heads=hk, dim_head=D, capacity=max(counts), max_drafts=T,
                             dtype=DT[dtype], device=d, counts=torch.tensor(counts, dtype=torch.int32, device=d))
    host = fill_cache(cache, g, d)
    trees = [make_tree(T, g, kind) for _ in range(B)]
    q1 = torch.randn(B, H, T, D, generator=g).to(DT[dtype])
    out = cache.attend(q1.to(d), parents=torch.tensor(trees, device=d))
    want, tol = attend_pairs(pair(dtype, order), q1, host, counts, trees, D ** -0.5)
    for k, (x, w, e) in enumerate(zip((out, *cache.draft_msgs, *cache.draft_lses), want, tol)):
        assert_within(x, w, e, f"output {k}")


@param("dtype", ("bf16", "f16"))
@param("T,H,D", [(1, 16, 64), (5, 8, 128), (1, 48, 128)])
def test_attend_weights_of_few_positions(dtype, T, H, D):
    """Queries of 0: the weights are those of the logsumexps alone, and the scores' own error hides nothing."""
    from poly_attention import DraftCache

    d = dev()
    g = torch.Generator().manual_seed(T)
    cache = DraftCache.empty(order=2, batch=4, kv_heads=1, dim_head=D, capacity=6, max_drafts=T, dtype=DT[dtype],
                             device=d, counts=torch.tensor([2, 3, 5, 6], dtype=torch.int32, device=d))
    host = fill_cache(cache, g, d)
    q1 = torch.zeros(4, H, T, D, dtype=DT[dtype])
    chain = [list(range(-1, T - 1))] * 4
    out = cache.attend(q1.to(d))
    want, tol = attend_pairs(pair(dtype, 2), q1, host, [2, 3, 5, 6], chain, D ** -0.5)
    assert_within(out, want[0], tol[0], "out")


@param("dtype", ("bf16", "f16", "f32"))
@param("T", (1, 20, 40))
def test_attend_small_weights_beside_a_large_one(dtype, T):
    """One position takes nearly all of the weight and has a value of 0: what is left are 4000 weights of 2^-25.6,
    below fp16's smallest number where the largest is 1.  So many key heads that one workgroup holds a row."""
    from poly_attention import DraftCache

    d = dev()
    g = torch.Generator().manual_seed(T)
    hk, n, D = 600, 4000, 8
    cache = DraftCache.empty(order=2, batch=1, kv_heads=hk, dim_head=D, capacity=n, max_drafts=T, dtype=DT[dtype],
                             device=d, counts=torch.tensor([n], dtype=torch.int32, device=d))
    host = fill_cache(cache, g, d)
    host["lses"][0].zero_()
    host["lses"][0][:, :, 100] = 25.6 * 0.6931471805599453
    host["msgs"][0].add_(1.0)
    host["msgs"][0][:, :, 100] = 0.0
    cache.lses[0].copy_(host["lses"][0])
    cache.msgs[0].copy_(host["msgs"][0])
    q1 = torch.zeros(1, hk, T, D, dtype=DT[dtype])
    out = cache.attend(q1.to(d))
    two = {k: [t[:, :2] for t in ts] for k, ts in host.items()}
    want, tol = attend_pairs(pair(dtype, 2), q1[:, :2], two, [n], [list(range(-1, T - 1))], D ** -0.5)
    # below 2^-14 fp16's steps stop shrinking: a weight is off by up to 2^-25, where the largest is at least 2^7
    floor = 2.0 ** -32 if dtype == "f16" else 0.0
    tol[0] += floor * host["msgs"][0][:, :2].double().abs().sum(2)[:, :, None]
    assert_within(out[:, :2], want[0], tol[0], "out")
def middle_case(dtype, T, H, D, g, d):
    """An order-3 cache of 64 positions a row, and one query tensor."""
    from poly_attention import DraftCache

    cache = DraftCache.empty(order=3, batch=2, kv_heads=1, dim_head=D, capacity=64, max_drafts=T, dtype=DT[dtype],
                             device=d, counts=torch.tensor([64, 50], dtype=torch.int32, device=d))
    host = fill_cache(cache, g, d)
    return cache, host, torch.randn(2, H, T, D, generator=g).to(DT[dtype])


MIDDLE = [(1, 2, 64), (9, 2, 128), (3, 1, 144), (13, 3, 64), (20, 4, 64), (12, 4, 128)]


@param("T,H,D", MIDDLE)
def test_attend_middle_products_beyond_fp16(T, H, D):
    """v * msg of a middle level passes fp16's largest and smallest numbers at some positions, their weighted mean
    mostly does not: the product is not rounded to the type.  One such position has weight 0."""
    d = dev()
    g = torch.Generator().manual_seed(T + D)
    cache, host, q1 = middle_case("f16", T, H, D, g, d)
    # chain level 1 scores q2 . q3 over v = vs[0], multiplied by the deepest level's outputs
    for at, v, m in ((7, 300.0, 1500.0), (11, -60000.0, 60.0), (40, 2.0 ** -14, 2.0 ** -10)):
        host["vs"][0][:, :, at, 3:6] = v
        host["msgs"][0][:, :, at, 3:6] = m
    host["lses"][0][:, :, 11] = -torch.finfo(torch.float32).max
    for name in ("vs", "msgs", "lses"):
        getattr(cache, name)[0].copy_(host[name][0])
    out = cache.attend(q1.to(d))
    host["lses"][0].clamp_(min=-1e30)  # the oracle's bounds stay finite; the weight is 0 as well
    want, tol = attend_pairs(pair("f16", 3), q1, host, [64, 50], [list(range(-1, T - 1))] * 2, D ** -0.5)
    assert all(bool(w.isfinite().all()) for w in want)
    for k, (x, w, e) in enumerate(zip((out, *cache.draft_msgs, *cache.draft_lses), want, tol)):
        x = x.double().cpu()
        past = w.abs() >= 65520.0  # a mean that rounds to fp16's infinity (the last of the cases: 116916)
        assert bool((x.isinf() == past).all()) and bool((x.sign() == w.sign())[past].all())
        assert_within(x.masked_fill(past, 0.0), w.masked_fill(past, 0.0), e.masked_fill(past, 0.0), f"output {k}")


@param("dtype", ("bf16", "f16", "f32"))
@param("T,H,D", MIDDLE)
def test_attend_infinite_values(dtype, T, H, D):
    """An infinite value or level output of a position with a weight gives an infinite output of its sign at
    its feature, no NaN, and leaves the other features' bits as they were."""
    d = dev()
    g = torch.Generator().manual_seed(T + D)
    cache, host, q1 = middle_case(dtype, T, H, D, g, d)
    q1 = q1.to(d)
    clean = [x.clone() for x in (cache.attend(q1), *cache.draft_msgs)]
    inf = float("inf")
    cache.vs[0][:, :, 5, 2], cache.msgs[0][:, :, 5, 2] = inf, -0.5     # the middle level: either factor,
    cache.vs[0][:, :, 17, 9], cache.msgs[0][:, :, 17, 9] = -2.0, -inf  # both
    cache.vs[0][:, :, 33, 12], cache.msgs[0][:, :, 33, 12] = inf, inf
    cache.vs[1][:, :, 5, 20] = -inf                                     # the deepest one's values
    cache.msgs[1][:, :, 8, 30] = inf                                    # and the final one's
    out = cache.attend(q1)
    signs = {2: -inf, 9: inf, 12: inf}
    deepest, middle, final = cache.draft_msgs[0], cache.draft_msgs[1], out
    same = [c for c in range(D) if c not in (2, 9, 12, 20, 30)]
    for x, y in ((deepest, clean[1]), (middle, clean[2]), (final, clean[0])):
        assert torch.equal(x[..., same], y[..., same])
    for c, s in signs.items():
        assert bool((middle[..., c] == s).all() and (final[..., c] == s).all()), c
    assert bool((deepest[..., 20] == -inf).all() and (final[..., 30] == inf).all())
    # the middle level's drafted values are v * -inf: of one sign up to the first v of the other, then inf - inf
    own = cache.draft_vs[0][..., 20].double().cumsum(-1) * 0 - cache.draft_vs[0][..., 20].double().sign() * inf
    one = (own.cummax(-1).values == own.cummin(-1).values)
    assert torch.equal(middle[..., 20].double().nan_to_num(0, 7, -7), own.masked_fill(~one, 0.0).nan_to_num(0, 7, -7))


def test_a_forked_cache_goes_its_own_way():
    """Two caches of one prompt, copied before a step and after one: steps and commits of one leave the other as it
    is, also when the other is gone."""
    import copy

    from poly_attention import commit_drafts

    d = dev()
    g = torch.Generator().manual_seed(8)
    caches = random_caches(2, 3, 2, 2, 64, 40, 4, [7, 3], "bf16", d, g)
    bufs = lambda cs: [t for c in cs for name in BUFS for t in getattr(c, name)]  # noqa: E731
    q1 = torch.randn(2, 4, 3, 64, generator=g).bfloat16().to(d)
    path = torch.tensor([[0, 2, 1], [1, 0, 2]], dtype=torch.int32, device=d)
    kept = torch.tensor([3, 1], dtype=torch.int32, device=d)

    def step(cs):
        outs = [c.attend(q1).clone() for c in cs]
        commit_drafts(cs, path, kept)
        return outs

    fork = copy.deepcopy(caches)
    before = [t.clone() for t in bufs(caches)]
    first = step(fork)
    assert fork[0].lengths() == [10, 4] and caches[0].lengths() == [7, 3]
    for a, b in zip(bufs(caches), before):
        assert torch.equal(a, b)
    for a, b in zip(step(caches), first):
        assert torch.equal(a, b)
    again = copy.deepcopy(caches)  # after a step
    del caches
    for a, b in zip(step(again), step(fork)):
        assert torch.equal(a, b)
    for a, b in zip(bufs(again), bufs(fork)):
        assert torch.equal(a, b)
    assert again[1].lengths() == fork[1].lengths() == [13, 5]


def test_overflow_shows_on_every_cache_of_a_commit():
    """Tokens past the capacity are dropped from all layers: each of their caches says so, a copy too, and still does
    after a commit with another cache first."""
    import copy

    from poly_attention import commit_drafts

    d = dev()
    a, b, c = random_caches(3, 2, 2, 1, 64, 8, 4, [7, 2], "bf16", d, torch.Generator().manual_seed(1))
    path = torch.tensor([[0, 1, 2, 3]] * 2, dtype=torch.int32, device=d)
    two = torch.tensor([2, 2], dtype=torch.int32, device=d)
    none = torch.zeros(2, dtype=torch.int32, device=d)
    commit_drafts([a, b], path, none)
    for x in (a, b, c):
        x.check_overflow()
    commit_drafts([a, b], path, two)
    assert a.lengths() == [8, 4]
    c.check_overflow()  # not of that commit
    commit_drafts([c, b, a], path, none)
    c.check_overflow()
    for x in (a, b, *copy.deepcopy([a, b])):
        with pytest.raises(RuntimeError, match="overflow"):
            x.check_overflow()
    commit_drafts([b, c], path, two)
    for x in (a, b, c):
        with pytest.raises(RuntimeError, match="overflow"):
            x.check_overflow()


# (children's tokens in order, vocabulary, gaps between the two logits that hold all of p)
COVERED = [((0, 1), 2), ((1, 0), 2), ((0, 1), 300), ((1, 0), 5000), ((0, 0, 1), 40000), ((1, 5, 0), 700)]


def covered_inputs(tokens, V):
    """Rows whose p is two tokens', 0 below 1 by a gap, both of them children of node 0, and the largest uniforms."""
    gaps = torch.linspace(0.0, 15.0, 121)
    B, T = len(gaps), 1 + len(tokens)
    logits = torch.full((B, T, V), -2000.0)  # 0 in fp32
    logits[:, :, 1] = 3.0
    logits[:, :, 0] = 3.0 - gaps[:, None]
    u = torch.full((B, T), 1.0 - 2.0 ** -24)
    g = torch.Generator().manual_seed(V)
    noise = -torch.log(torch.rand(B, V, generator=g).clamp(min=1e-30))
    return (logits, torch.tensor([[0, *tokens]] * B), [[-1] + [0] * len(tokens)] * B, u, noise, None, None)


@param("tokens,V", COVERED)
def test_verify_children_that_hold_all_of_p(tokens, V):
    """What is left after the first is rejected is the other's, so that is kept whatever its number (below 1); the row
    always has a token."""
    from test_gpu_25_drafts import run_verify

    path, kept, token = (t.cpu() for t in run_verify(covered_inputs(tokens, V), dev()))
    last = max(i for i, x in enumerate(tokens) if x == [y for y in tokens if y < 2][-1] and x not in tokens[:i]) + 1
    assert kept.tolist() == [2] * len(kept) and path[:, 1].tolist() == [last] * len(kept)
    assert bool(((token == 0) | (token == 1)).all())


SHARES = [(2 ** -k, s, V, order) for k in (4, 7, 11, 16) for s in (0.3, 0.8) for V in (3, 40, 6000)
          for order in ((0, 1), (0, 2, 1))]


def share_inputs(below):
    """Per case of SHARES a row of each of its vocabularies: token 0 has all but a small part of p, token 1 a share of
    that part.  The child with token 0 is rejected; that with token 1 gets a number 2^-14 below its share, or above."""
    rows = []
    for part, share, V, order in SHARES:
        p = torch.full((V,), part * (1 - share) / (V - 2), dtype=torch.float64)
        p[0], p[1] = 1 - part, part * share
        x = p.log().float()
        p = torch.softmax(x.double(), 0)
        out = [t for t in order if t != 1]
        now = p[1] / (p.sum() - p[out].sum())
        T = 1 + len(order)
        u = torch.full((1, T), 1.0 - 2.0 ** -24)
        u[0, T - 1] = float(now) * (1 - below * 2.0 ** -14)
        noise = -torch.log(torch.rand(1, V, generator=torch.Generator().manual_seed(T)).clamp(min=1e-30))
        rows.append((x.expand(1, T, V).contiguous(), torch.tensor([[0, *order]]), [[-1] + [0] * len(order)], u, noise, None,
                     None))
    return rows


@param("below", (1, -1))
def test_verify_share_of_a_small_remainder(below):
    """A child's probability after a rejection that leaves down to 2^-16 of p is exact to fp32's few last digits."""
    from test_gpu_25_drafts import assert_walk, run_verify

    for inputs in share_inputs(below):
        want, margin = DO.verify(*inputs)
        assert margin > 2.0 ** -17  # the kernel's probabilities are within 2^-20
        assert len(want[0][0]) == (2 if below > 0 else 1)
        assert_walk(run_verify(inputs, dev()), want)


@param("order", (2, 3))
@param("dtype", (torch.bfloat16, torch.float16))
@param("freqs_too", (True, False))
def test_module_rotary_of_a_layer_cast_whole(order, dtype, freqs_too):
    """A layer cast to 16 bits with its rotary frequencies rotates by angles of 16 bits, up to a radian off behind a few
    hundred positions: a drafted step's keys are turned by the same ones as the cached keys."""
    from parity import assert_parity
    from poly_attention import DraftCache, commit_drafts
    from poly_attention.rotary import RotaryEmbedding
    from test_gpu_25_drafts import make_module

    d = dev()
    torch.manual_seed(5)
    m, _, _ = make_module(order, 4, d, dtype, use_rotary_embed=True)
    if not freqs_too:
        m.rotary_emb.freqs.data = RotaryEmbedding(2 * m.rotary_emb.freqs.numel()).freqs.data.to(d)
    x = torch.randn(2, 404, 64, generator=torch.Generator().manual_seed(2)).to(d, dtype)
    with torch.no_grad():
        _, cache = m(x[:, :400], return_cache=True)
        dc = DraftCache(cache, capacity=410)
        got = m(x[:, 400:], cache=dc)
        commit_drafts([dc], torch.arange(4, dtype=torch.int32, device=d).expand(2, 4).contiguous(),
                      torch.full((2,), 4, dtype=torch.int32, device=d))
        want = []
        for i in range(400, 404):
            y, cache = m(x[:, i:i + 1], cache=cache, return_cache=True)
            want.append(y)
        assert_parity(got, torch.cat(want, 1), dtype, "a chain", roundings=3)
        # the tuple cache holds its keys unrotated.  Rounded on the module's way: the norm, cos, sin, both products and
        # their sum, and the draft's one: each half a step of the pair's values
        half = torch.finfo(dtype).eps / 2
        for q, raw in zip(dc.qs, cache[:2] if order == 2 else cache[0]):
            turned = m.rotary_emb.rotate_queries_or_keys(raw)
            pair = raw.float().abs().unflatten(-1, (-1, 2)).sum(-1, keepdim=True).expand(*raw.shape[:-1], -1, 2).flatten(-2)
            off = (q[:, :, :404].float() - turned.float()).abs()
            assert bool((off <= 7 * half * pair).all()), float((off / pair).max())


def test_rows_of_size_one_dimensions_of_any_stride():
    """One row, one token, one head: a stride that nothing follows is no reason to refuse."""
    from poly_attention import DraftCache

    d = dev()
    g = torch.Generator().manual_seed(6)
    cache = DraftCache.empty(order=2, batch=1, kv_heads=1, dim_head=64, capacity=9, max_drafts=2, device=d,
                             counts=torch.tensor([9], dtype=torch.int32, device=d))
    fill_cache(cache, g, d)
    rows = [torch.randn(64, generator=g).bfloat16().to(d) for _ in range(4)]
    plain = [r.view(1, 1, 1, 64) for r in rows]
    odd = [r.as_strided((1, 1, 1, 64), (3, 5, 7, 1)) for r in rows]
    results = []
    for qs in (plain, odd):
        q1 = cache.append(qs[:3], qs[3:], [None] * 3, eps=1e-6)
        results.append([q1.clone(), cache.attend(qs[0]).clone(), *[t.clone() for t in (*cache.draft_qs, *cache.draft_vs)]])
    for a, b in zip(*results):
        assert torch.equal(a, b)


@param("dtype", ("bf16", "f32"))
@param("order,T,H,D", [(8, 64, 1, 8), (8, 5, 3, 16), (6, 17, 2, 40), (5, 33, 4, 136 + 8)])
def test_attend_many_levels(dtype, order, T, H, D):
    from test_gpu_25_drafts import check_attend

    check_attend(order, 1, [37], T, H, 1, D, dtype, "tree")


def test_offsets_past_32_bits():
    """2.3e9 elements a buffer (4.6 GB): the last key head's positions, keys and records lie past 2^31 elements and 2^32
    bytes, the committed ones too."""
    from poly_attention import DraftCache, commit_drafts

    d = dev()
    hk, n, D, T = 17, 1 << 20, 128, 3
    cache = DraftCache.empty(order=2, batch=1, kv_heads=hk, dim_head=D, capacity=n + 2, max_drafts=T, device=d,
                             counts=torch.tensor([n], dtype=torch.int32, device=d))
    g = torch.Generator(device=d).manual_seed(0)
    for t in (*cache.qs, *cache.vs, *cache.msgs, *cache.draft_qs, *cache.draft_vs):
        t.normal_(generator=g)
    cache.lses[0].normal_(generator=g).add_(14.0)
    q1 = torch.randn(1, hk, T, D, generator=g, device=d).bfloat16()
    out = cache.attend(q1)
    for h in (0, hk - 1):
        def level(q, k, dk, v, dv, bias=None, dbias=None):
            s = torch.cat([q.double() @ k[:n].double().t(), q.double() @ dk.double().t()], 1) * D ** -0.5
            if bias is not None:
                s = s + torch.cat([bias[:n].double(), dbias])
            s[:, n:].masked_fill_(torch.ones(T, T, device=d).triu(1).bool(), -float("inf"))
            w = torch.softmax(s, -1)
            return w[:, :n] @ v[:n].double() + w[:, n:] @ dv.double(), torch.logsumexp(s, -1)

        msg, lse = level(cache.draft_qs[0][0, h], cache.qs[1][0, h], cache.draft_qs[1][0, h], cache.vs[0][0, h],
                         cache.draft_vs[0][0, h])
        want, _ = level(q1[0, h], cache.qs[0][0, h], cache.draft_qs[0][0, h], cache.msgs[0][0, h], msg, cache.lses[0][0, h], lse)
        # values of size 1 under 10^6 weights: outputs of 10^-3, and the sums' fp32 roundings of 2^-24 sqrt(n) n / n
        assert float((out[0, h].double() - want).abs().max()) <= 2.0 ** -8 * float(want.abs().max()) + 2.0 ** -14
        assert float((cache.draft_msgs[0][0, h].double() - msg).abs().max()) <= 2.0 ** -8 * float(msg.abs().max()) + 2.0 ** -14
        assert float((cache.draft_lses[0][0, h].double() - lse).abs().max()) <= 2.0 ** -14
    commit_drafts([cache], torch.tensor([[0, 2, 1]], dtype=torch.int32, device=d), torch.tensor([2], dtype=torch.int32, device=d))
    assert cache.lengths() == [n + 2]
    for name in BUFS:
        for dst, src in zip(getattr(cache, name), getattr(cache, "draft_" + name)):
            assert torch.equal(dst[0, :, n:], src[0][:, [0, 2]])


# (seed, B, T, V): every node a child of node 0, tokens that repeat, numbers near 1: many rejections in a row
STARS = [(1, 6, 64, 40), (2, 6, 64, 20000), (3, 8, 8, 30), (4, 8, 8, 500), (5, 4, 33, 4097), (6, 8, 5, 6)]


def star_inputs(case):
    seed, B, T, V = case
    g = torch.Generator().manual_seed(seed)
    logits = 3 * torch.randn(B, T, V, generator=g)
    likely = logits[:, 0].topk(min(V, 24)).indices
    tokens = likely.gather(1, torch.randint(0, likely.shape[1], (B, T), generator=g))
    tokens[:, 1::5] = torch.randint(0, V, tokens[:, 1::5].shape, generator=g)
    tokens[0, T // 2] = V
    u = 1 - 0.15 * torch.rand(B, T, generator=g) ** 2
    noise = -torch.log(torch.rand(B, V, generator=g).clamp(min=1e-30))
    temperature = 0.5 + torch.rand(B, generator=g)
    return logits, tokens, [[-1] + [0] * (T - 1)] * B, u, noise, temperature, None


@param("case", STARS)
def test_verify_many_children_of_one_node(case):
    from test_gpu_25_drafts import assert_walk, run_verify

    inputs = star_inputs(case)
    want, margin = DO.verify(*inputs)
    assert margin > 2.0 ** -17
    assert_walk(run_verify(inputs, dev()), want)
