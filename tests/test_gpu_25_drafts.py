"""GPU: drafted tokens -- DraftCache.append / attend, verify_drafts, commit_drafts -- against the 64-bit
oracle of drafts_oracle.py (whose docstring derives the bounds), and the modules' drafted steps against
the oracle's parallel forward."""

import pytest
import torch

import drafts_oracle as DO
import oracle.poly_oracle as O
from parity import assert_parity

pytestmark = pytest.mark.gpu
param = pytest.mark.parametrize

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda")


def make_tree(T, g, kind):
    p = [-1]
    for t in range(1, T):
        p.append(t - 1 if kind == "chain" else int(torch.randint(max(0, t // 2 - 1), t, (1,), generator=g)))
    if kind == "holes" and T > 2:
        p[T // 2] = -2          # absent, and so is what follows it
        p[T - 1] = T // 2
        if T > 6:
            p[3], p[4] = 3, 70  # its own parent, a later one
    if kind == "forest":
        p[T // 2] = -1
    return p


def fill_cache(cache, g, d, stale=float("nan")):
    """Random contents; everything behind a row's count is ``stale``."""
    host = {}
    n = cache.lengths()
    for name in ("qs", "vs", "msgs", "lses", "draft_qs", "draft_vs", "draft_msgs", "draft_lses"):
        std = 0.3 if "msgs" in name else 1.0
        host[name] = []
        for lvl, t in enumerate(getattr(cache, name)):
            x = torch.randn(t.shape, generator=g) * std
            if "lses" in name:
                x += 2.0 * (lvl + 1)
            if not name.startswith("draft"):
                for b in range(t.shape[0]):
                    x[b, :, n[b]:] = stale
            x = x.to(t.dtype)
            t.copy_(x)
            host[name].append(x)
    return host


def assert_within(got, want, tol, what):
    diff = (got.double().cpu() - want).abs()
    over = diff - tol
    assert bool((over <= 0).all()), (f"{what}: off by {diff.max().item():.3e}, over the bound by "
                                     f"{over.max().item():.3e} at {(over == over.max()).nonzero()[0].tolist()}")


def check_attend(order, B, counts, T, H, hk, D, dtype, kind, softclamp=None, scale=None, capacity=None,
                 one_tree=False, stale=float("nan"), max_drafts=None, parents_dtype=torch.int32):
    from poly_attention import DraftCache

    d = dev()
    g = torch.Generator().manual_seed(order * 1000 + B * 100 + T)
    cap = capacity or max(1, max(counts))
    cache = DraftCache.empty(order=order, batch=B, kv_heads=hk, dim_head=D, capacity=cap,
                             max_drafts=max_drafts or T, dtype=DT[dtype], device=d,
                             counts=torch.tensor(counts, dtype=torch.int32, device=d))
    host = fill_cache(cache, g, d, stale)
    trees = [make_tree(T, g, kind) for _ in range(1 if one_tree else B)]
    # absent nodes' slots may hold anything
    if kind == "holes":
        for b in range(B):
            for t, x in enumerate(DO.walk_tree(trees[0 if one_tree else b])):
                if x is None:
                    for name in ("draft_vs", "draft_qs"):
                        for buf in getattr(cache, name):
                            buf[b, :, t] = float("nan")
    q1 = torch.randn(B, T, H, D, generator=g).to(DT[dtype]).permute(0, 2, 1, 3)
    par = torch.tensor(trees, dtype=parents_dtype)
    before = [t.clone() for t in (*cache.qs, *cache.vs, *cache.msgs, *cache.lses)]
    slots = [t.clone() for t in (*cache.draft_msgs, *cache.draft_lses)]
    out = cache.attend(q1.to(d), parents=None if kind == "chain" else (par[0] if one_tree else par).to(d),
                       scale=scale, softclamp=softclamp)
    torch.cuda.synchronize()
    lens = [min(max(n, 0), cap) for n in counts]
    want, tol = DO.attend(q1, host, lens, trees * B if one_tree else trees,
                          D ** -0.5 if scale is None else scale, softclamp)
    got = [out, *[t[:, :, :T] for t in cache.draft_msgs], *[t[:, :, :T] for t in cache.draft_lses]]
    for k, (x, w, e) in enumerate(zip(got, want, tol)):
        assert_within(x, w, e, f"output {k}")
    # the cached positions and the slots behind the last token are as they were
    for a, b in zip(before, (*cache.qs, *cache.vs, *cache.msgs, *cache.lses)):
        assert torch.equal(a.nan_to_num(9.0), b.nan_to_num(9.0))
    for a, b in zip(slots, (*cache.draft_msgs, *cache.draft_lses)):
        assert torch.equal(a[:, :, T:], b[:, :, T:])
    return cache, q1, out


@param("dtype", ("bf16", "f16", "f32"))
@param("order,B,counts,T,H,hk,D,kind", [
    (2, 1, [0], 1, 1, 1, 64, "chain"),            # nothing cached, nothing drafted
    (2, 1, [1], 1, 2, 1, 64, "tree"),
    (2, 2, [127, 128], 5, 4, 2, 64, "tree"),      # around one unit of positions
    (2, 3, [129, 0, 300], 16, 2, 2, 128, "holes"),
    (3, 2, [40, 513], 17, 4, 2, 64, "tree"),      # a middle level; a second tile of rows
    (4, 1, [33], 3, 2, 1, 32, "forest"),
    (2, 2, [31, 65], 33, 3, 1, 96, "tree"),       # head dims between the usual ones
    (2, 2, [17, 50], 7, 6, 2, 40, "holes"),
    (2, 1, [260], 64, 8, 1, 64, "tree"),          # several blocks of rows
    (3, 1, [70], 9, 2, 2, 256, "tree"),
    (2, 1, [20], 20, 4, 2, 144, "tree"),
    (2, 1, [90], 40, 2, 1, 8, "holes"),
])
def test_attend(dtype, order, B, counts, T, H, hk, D, kind):
    check_attend(order, B, counts, T, H, hk, D, dtype, kind)


@param("dtype", ("bf16", "f16"))
@param("order,B,counts,T,H,hk,D,kind", [
    (2, 2, [0, 1], 64, 8, 4, 64, "tree"),         # blocks of more than 64 rows: nothing cached, one position
    (2, 2, [127, 1000], 33, 4, 2, 128, "holes"),  # 66 rows: 32, 32, 2 and none per wave
    (2, 3, [33, 64, 2500], 13, 8, 1, 96, "forest"),
    (3, 2, [600, 5], 40, 8, 2, 64, "tree"),       # a middle level of fewer rows than a block holds
    (4, 1, [300], 64, 8, 1, 128, "tree"),         # several blocks
    (3, 1, [1500], 64, 5, 1, 40, "chain"),        # 320 rows of 64 padded columns
    (2, 70, [7 * b % 90 for b in range(70)], 17, 4, 1, 8, "holes"),
])
def test_attend_wide_blocks(dtype, order, B, counts, T, H, hk, D, kind):
    check_attend(order, B, counts, T, H, hk, D, dtype, kind)


def test_attend_wide_blocks_softclamp():
    check_attend(3, 2, [100, 3], 24, 6, 2, 128, "bf16", "tree", softclamp=5.0)


@param("dtype,softclamp,scale", [("bf16", 5.0, None), ("f32", 30.0, 0.05), ("f16", 0.5, 1.0), ("f32", None, 0.0)])
def test_attend_softclamp_and_scale(dtype, softclamp, scale):
    check_attend(3, 2, [100, 3], 6, 4, 2, 64, dtype, "tree", softclamp=softclamp, scale=scale)


def test_attend_many_rows():
    """More rows than a wave has lanes, of very different lengths."""
    counts = [(37 * b) % 150 if b % 5 else 0 for b in range(70)]
    check_attend(2, 70, counts, 3, 2, 1, 32, "bf16", "tree", one_tree=True, parents_dtype=torch.int64)


def test_attend_long_row_among_short():
    check_attend(2, 3, [3, 4100, 0], 4, 4, 2, 64, "bf16", "tree", capacity=5000)


def test_attend_counts_out_of_range_are_clamped():
    check_attend(2, 3, [-5, 1000, 2 ** 31 - 1], 4, 2, 2, 64, "bf16", "tree", capacity=150)


def test_attend_slots_beyond_the_tokens():
    check_attend(2, 2, [10, 20], 3, 4, 2, 64, "bf16", "chain", max_drafts=16)


@param("dtype", ("bf16", "f32"))
def test_attend_masked_rows_of_the_prompt(dtype):
    """A cached position whose own level saw nothing (logsumexp the lowest value, or -inf) weighs
    nothing, in the middle of a row and where every cached position is one."""
    from poly_attention import DraftCache

    d = dev()
    g = torch.Generator().manual_seed(5)
    cache = DraftCache.empty(order=2, batch=2, kv_heads=1, dim_head=64, capacity=300, max_drafts=4,
                             dtype=DT[dtype], device=d, counts=torch.tensor([300, 200], dtype=torch.int32, device=d))
    host = fill_cache(cache, g, d)
    host["lses"][0][0, :, ::2] = -torch.finfo(torch.float32).max
    host["lses"][0][0, :, 5] = -float("inf")
    host["lses"][0][1] = -torch.finfo(torch.float32).max
    cache.lses[0].copy_(host["lses"][0])
    q1 = torch.randn(2, 2, 4, 64, generator=g).to(DT[dtype])
    out = cache.attend(q1.to(d))
    for h in host["lses"]:
        h.clamp_(min=-1e30)  # the oracle's bounds stay finite; the weights are 0 as well
    want, tol = DO.attend(q1, host, [300, 200], [[-1, 0, 1, 2]] * 2, 64 ** -0.5, None)
    assert_within(out, want[0], tol[0], "out")


def test_attend_is_deterministic_and_follows_its_stream():
    cache, q1, out = check_attend(2, 2, [700, 90], 8, 4, 2, 64, "bf16", "chain")
    q = q1.to(dev())
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        outs = [cache.attend(q) for _ in range(5)]
    s.synchronize()
    for o in outs:
        assert torch.equal(o, out)


def test_two_caches_at_once_on_two_streams():
    """Each step's workspace is its own: interleaved launches on two streams give each cache's result."""
    a, qa, outa = check_attend(2, 2, [700, 90], 8, 4, 2, 64, "bf16", "chain")
    b, qb, outb = check_attend(3, 3, [300, 0, 41], 8, 4, 2, 64, "bf16", "chain")
    qa, qb = qa.to(dev()), qb.to(dev())
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = []
    for _ in range(20):
        for s, c, q in zip(streams, (a, b), (qa, qb)):
            with torch.cuda.stream(s):
                outs.append(c.attend(q))
    torch.cuda.synchronize()
    for k, o in enumerate(outs):
        assert torch.equal(o, outb if k % 2 else outa)


@param("value", (float("nan"), float("inf")))
@param("dtype,T,H,D", [("f32", 5, 2, 64), ("f32", 40, 4, 64), ("bf16", 20, 8, 128), ("f16", 64, 2, 64)])
def test_attend_what_another_branch_holds(dtype, T, H, D, value):
    """A node's key, query and value that are no numbers leave the outputs of all nodes that do not see it
    as they were: the same sums in the same order."""
    cache, q1, _ = check_attend(3, 2, [130, 3], T, H, 2, D, dtype, "chain")
    parents = torch.zeros(T, dtype=torch.int32, device=dev())
    parents[0] = -1
    q1, bad = q1.to(dev()), T // 2
    others = [t for t in range(T) if t != bad]

    def step():
        out = cache.attend(q1, parents=parents)
        return [x[:, :, others].clone() for x in (out, *cache.draft_msgs, *cache.draft_lses)]

    want = step()
    q1[:, :, bad] = value
    for t in (*cache.draft_qs, *cache.draft_vs):
        t[:, :, bad] = value
    for x, y in zip(step(), want):
        assert bool(y.isfinite().all()) and torch.equal(x, y)


def test_attend_takes_any_strides_of_q1():
    from poly_attention import DraftCache

    d = dev()
    g = torch.Generator().manual_seed(3)
    cache = DraftCache.empty(order=2, batch=2, kv_heads=2, dim_head=64, capacity=50, max_drafts=4,
                             device=d, counts=torch.tensor([50, 7], dtype=torch.int32, device=d))
    fill_cache(cache, g, d)
    q = torch.randn(2, 4, 4, 64, generator=g).bfloat16().to(d)
    want = cache.attend(q)
    wide = torch.zeros(2, 4, 4, 67, dtype=torch.bfloat16, device=d)
    wide[..., 3:] = q
    turned = q.transpose(2, 3).contiguous().transpose(2, 3)
    for x in (wide[..., 3:], turned, q.permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3)):
        assert torch.equal(cache.attend(x), want)


# ---------------------------------------------------------------------------------------


@param("dtype", ("bf16", "f16", "f32"))
@param("order,B,T,H,hk,D,rot,shape", [
    (2, 1, 1, 2, 1, 64, 64, "btr"), (2, 3, 5, 4, 2, 128, 64, "btr"), (3, 2, 17, 3, 1, 40, 40, "tr"),
    (2, 2, 4, 8, 8, 96, 0, None), (4, 2, 3, 2, 2, 256, 256, "r"), (2, 33, 16, 2, 1, 32, 2, "btr"),
    (2, 1, 64, 16, 4, 8, 8, "tr"),
])
def test_append(dtype, order, B, T, H, hk, D, rot, shape):
    from poly_attention import DraftCache

    d = dev()
    g = torch.Generator().manual_seed(order + B + T + D)
    cache = DraftCache.empty(order=order, batch=B, kv_heads=hk, dim_head=D, capacity=9, max_drafts=T + 2 if T < 63 else T,
                             dtype=DT[dtype], device=d)
    for t in (*cache.draft_qs, *cache.draft_vs):
        t.fill_(7.0)

    def proj(h):  # a projection's output seen per head
        return torch.randn(B, T, h, D, generator=g).to(DT[dtype]).permute(0, 2, 1, 3)

    qs = [proj(H)] + [proj(hk) for _ in range(order)]
    vs = [proj(hk) for _ in range(order - 1)]
    ws = [(1 + 0.3 * torch.randn(D, generator=g)).to(DT[dtype] if i % 2 else torch.float32) for i in range(order + 1)]
    angles = full = None
    if rot:
        size = {"btr": (B, T, rot), "tr": (T, rot), "r": (rot,)}[shape]
        angles = torch.randn(size, generator=g) * 1000
        full = angles.expand(B, T, rot)
    q1 = cache.append([q.to(d) for q in qs], [v.to(d) for v in vs], [w.to(d) for w in ws], eps=1e-5,
                      angles=None if angles is None else angles.to(d))
    for k, (got, src) in enumerate(zip((q1, *cache.draft_qs), qs)):
        want, tol = DO.rows(src, ws[k], 1e-5, full)
        assert_within(got[:, :, :T], want, tol, f"q{k + 1}")
    for got, src in zip(cache.draft_vs, vs):
        assert torch.equal(got[:, :, :T].cpu(), src)
    for t in (*cache.draft_qs, *cache.draft_vs):
        assert bool((t[:, :, T:] == 7.0).all())


def test_append_refuses_to_drop_a_gradient():
    from poly_attention import DraftCache

    c = DraftCache.empty(order=2, batch=1, kv_heads=2, dim_head=64, capacity=9, dtype=torch.float32, device=dev())
    row = lambda h: torch.zeros(1, h, 3, 64, device=dev())  # noqa: E731
    for k in (0, 2, "weight"):
        qs, vs = [row(2), row(2), row(2)], [row(2)]
        weights = [torch.ones(64, device=dev()) for _ in qs]
        if k == "weight":
            weights[1].requires_grad_()
        else:
            qs[k].requires_grad_()
        with pytest.raises(RuntimeError, match="inference-only"):
            c.append(qs, vs, weights, eps=1e-6)
        with torch.no_grad():
            c.append(qs, vs, weights, eps=1e-6)


def test_append_positions_of_a_rotary_module():
    """inv_freq: the angle of a node is its row's count plus its depth, as the single-token prologue
    forms it (fp32 here: the position is exact)."""
    from poly_attention import DraftCache
    from poly_attention.rotary import RotaryEmbedding

    d = dev()
    g = torch.Generator().manual_seed(1)
    rotary = RotaryEmbedding(64, interpolate_factor=2.0).to(d)
    counts = torch.tensor([0, 1000, 77], dtype=torch.int32, device=d)
    cache = DraftCache.empty(order=2, batch=3, kv_heads=2, dim_head=64, capacity=2000, max_drafts=6,
                             dtype=torch.float32, device=d, counts=counts)
    parents = torch.tensor([[-1, 0, 0, 2, 3, 1], [-1, -1, 1, 2, 0, 4], [-1, 0, -2, 2, 1, 4]],
                           dtype=torch.int32, device=d)
    qs = [torch.randn(3, 2, 6, 64, generator=g).to(d) for _ in range(3)]
    kw = dict(eps=1e-5, parents=parents)
    q1 = cache.append(qs, qs[:1], [None] * 3, inv_freq=rotary.freqs, interp=2.0, **kw)
    got = [q1, *[t.clone() for t in cache.draft_qs]]
    with torch.no_grad():
        angles = rotary(cache.positions(6, parents).float() / 2.0)
    q1 = cache.append(qs, qs[:1], [None] * 3, angles=angles, **kw)
    present = torch.tensor([[x is not None for x in DO.walk_tree(p)] for p in parents.tolist()], device=d)
    for a, b in zip(got, (q1, *cache.draft_qs)):
        assert torch.equal(a[present[:, None].expand(3, 2, 6)], b[present[:, None].expand(3, 2, 6)])


# ---------------------------------------------------------------------------------------

# (seed, B, T, V, dtype, tree, with draft probabilities, temperatures)
VERIFY_CASES = [
    (1, 1, 1, 1, "f32", "chain", False, "ones"),
    (2, 3, 1, 257, "bf16", "chain", True, "ones"),
    (3, 4, 6, 256, "f32", "chain", False, "none"),
    (4, 5, 9, 1009, "f16", "tree", False, "mixed"),
    (5, 4, 16, 2003, "bf16", "tree", True, "mixed"),
    (6, 3, 64, 333, "f32", "tree", False, "ones"),
    (7, 3, 33, 130, "f32", "tree", True, "ones"),
    (8, 6, 12, 8192, "bf16", "holes", False, "mixed"),
    (9, 2, 4, 50257, "f32", "tree", True, "ones"),
    (10, 2, 5, 24577, "bf16", "tree", False, "greedy"),
    (11, 3, 8, 4099, "f16", "holes", True, "greedy"),
    (12, 4, 8, 1024, "bf16", "tree", True, "mixed"),  # the most that one launch takes, and one more
    (13, 4, 8, 1025, "f16", "tree", False, "ones"),
    (14, 3, 8, 512, "f32", "holes", True, "mixed"),
    (15, 3, 9, 512, "f32", "tree", False, "mixed"),
    (16, 2, 24, 40001, "bf16", "tree", True, "ones"),
    (17, 3, 7, 9001, "f16", "forest", True, "mixed"),
]


def verify_inputs(case):
    """logits, tokens, parents (lists), uniforms, noise, temperature, draft probabilities."""
    seed, B, T, V, dtype, kind, with_probs, temps = case
    g = torch.Generator().manual_seed(seed)
    logits = 2 * torch.randn(B, T, V, generator=g)
    parents = [make_tree(T, g, kind) for _ in range(B)]
    if kind == "holes":
        parents[-1][0] = -2  # a row without any node
    tokens = torch.randint(0, V, (B, T), generator=g)
    probs = None
    if with_probs:
        probs = torch.softmax(logits + 0.5 * torch.randn(B, T, V, generator=g), -1)
        for b in range(B):
            for t in range(1, T):
                p = min(max(parents[b][t], 0), T - 1)
                tokens[b, t] = torch.multinomial(probs[b, p], 1, generator=g)[0]
    else:
        for b in range(B):
            for t in range(1, T):
                p = min(max(parents[b][t], 0), T - 1)
                logits[b, p, tokens[b, t]] = torch.logsumexp(logits[b, p], 0) + 3 * torch.rand(1, generator=g)[0] - 1.5
    if T > 4:
        tokens[0, 2], tokens[0, 3] = V + 5, -7  # outside the vocabulary
        tokens[-1, 2] = tokens[-1, 1]            # the same token twice
    logits = logits.to(DT[dtype])
    if temps == "greedy":
        logits[0, 0, V // 2] = logits[0, 0].max() + 1
        logits[0, 0, V // 3] = logits[0, 0, V // 2]  # a tie
        if T > 1:
            tokens[0, 1] = V // 3
    u = torch.rand(B, T, generator=g)
    noise = -torch.log(torch.rand(B, V, generator=g).clamp(min=1e-30))
    temperature = {"ones": torch.ones(B), "none": None, "mixed": torch.tensor([0.8, 0.0, 1.5, 1.0, 0.0, 0.6])[:B],
                   "greedy": torch.zeros(B)}[temps]
    return logits, tokens, parents, u, noise, temperature, probs


def run_verify(inputs, d):
    from poly_attention import verify_drafts

    logits, tokens, parents, u, noise, temp, probs = inputs
    return verify_drafts(logits.to(d), tokens.to(d), torch.tensor(parents, dtype=torch.int32, device=d),
                         uniforms=u.to(d), noise=noise.to(d), temperature=None if temp is None else temp.to(d),
                         draft_probs=None if probs is None else probs.to(d))


def assert_walk(got, want):
    path, kept, token = (t.cpu() for t in got)
    T = path.shape[1]
    assert kept.tolist() == [len(p) for p, _ in want]
    assert path.tolist() == [p + [-1] * (T - len(p)) for p, _ in want]
    assert token.tolist() == [t for _, t in want]


@param("case", VERIFY_CASES)
def test_verify(case):
    inputs = verify_inputs(case)
    want, _ = DO.verify(*inputs)
    assert_walk(run_verify(inputs, dev()), want)


def test_verify_greedy_call_and_strides():
    """Without random numbers every row is greedy; logits and the rest as views."""
    from poly_attention import verify_drafts

    d = dev()
    logits, tokens, parents, _, _, _, _ = verify_inputs((20, 3, 7, 515, "bf16", "tree", False, "ones"))
    want, _ = DO.verify(logits, tokens, parents, None, None, None, None)
    par = torch.tensor(parents, device=d)
    for x in (logits.to(d), torch.nn.functional.pad(logits.to(d), (3, 2))[..., 3:-2],
              logits.to(d).transpose(0, 1).contiguous().transpose(0, 1),
              logits.to(d).transpose(1, 2).contiguous().transpose(1, 2)):
        wide = torch.zeros(3, 9, dtype=torch.int64, device=d)
        wide[:, 1:8] = tokens.to(d)
        assert_walk(verify_drafts(x, wide[:, 1:8], par), want)


def test_verify_logits_without_a_number():
    from poly_attention import verify_drafts

    d = dev()
    inf = float("inf")
    logits = torch.zeros(4, 2, 9000)
    logits[0] = -inf
    logits[1, 0, 8999] = float("nan")
    logits[2] = -inf
    logits[2, :, 8500] = 3.0  # one finite logit
    logits[3, :, 4:] = -inf   # a vocabulary cut down to four
    tokens = torch.tensor([[0, 1], [0, 1], [0, 8500], [0, 8]])
    u, noise = torch.full((4, 2), 0.5), torch.ones(4, 9000)
    noise[3, 2] = 0.5
    path, kept, token = verify_drafts(logits.to(d), tokens.to(d), None, uniforms=u.to(d), noise=noise.to(d))
    assert kept.tolist() == [1, 1, 2, 1] and token.tolist() == [-1, -1, 8500, 2]
    path, kept, token = verify_drafts(logits.to(d), tokens.to(d))
    assert kept.tolist() == [1, 1, 2, 1] and token.tolist() == [-1, 0, 8500, 0]


def test_verify_temperatures_near_zero_and_infinite():
    """A temperature so small that 1 / temperature is infinite puts all of p on the largest logit; an
    infinite one spreads it over every logit that is not -inf."""
    from poly_attention import verify_drafts

    d = dev()
    for V in (16, 8192):
        logits = torch.arange(V, dtype=torch.float32, device=d).expand(2, 1, V).contiguous()
        logits[:, :, 0] = -float("inf")
        noise = torch.ones(2, V, device=d)
        noise[:, 5] = 0.5
        noise[:, 0] = 0.25
        path, kept, token = verify_drafts(
            logits, torch.zeros(2, 1, dtype=torch.int64, device=d), uniforms=torch.zeros(2, 1, device=d),
            noise=noise, temperature=torch.tensor([1e-40, float("inf")], device=d))
        assert kept.tolist() == [1, 1] and token.tolist() == [V - 1, 5]


def test_verify_residual_of_nothing():
    """A draft distribution equal to the target's leaves nothing of p after a rejection (which a number
    below 1 never causes): p then stays as it was, with one child and with two."""
    from poly_attention import verify_drafts

    d = dev()
    for V in (8, 8192):
        logits, probs = torch.zeros(2, 3, V, device=d), torch.full((2, 3, V), 1.0 / V, device=d)
        tokens = torch.tensor([[0, 3, 5], [0, 5, 3]], device=d)
        noise = torch.ones(2, V, device=d)
        noise[0, 6] = noise[1, 5] = 0.5
        parents = torch.tensor([[-1, 0, 0], [-1, 0, -2]], device=d)
        path, kept, token = verify_drafts(logits, tokens, parents, uniforms=torch.ones(2, 3, device=d), noise=noise,
                                          draft_probs=probs)
        assert kept.tolist() == [1, 1] and token.tolist() == [6, 5]


def test_verify_keeps_the_target_distribution():
    """Over many rows with their own random numbers the first token behind node 0 is distributed as the
    target's softmax, with drafts chosen and with drafts drawn (two children each): with 40000 rows a
    frequency is off by 5 sqrt(p (1 - p) / 40000) with probability below 1e-6 per entry."""
    from poly_attention import verify_drafts

    d = dev()
    B, V = 40000, 12
    g = torch.Generator(device=d).manual_seed(0)
    base = torch.randn(V, generator=g, device=d)
    p = torch.softmax(base, 0)
    q = torch.softmax(base + torch.randn(V, generator=g, device=d), 0)
    parents = torch.tensor([-1, 0, 0], dtype=torch.int32, device=d)
    logits = base.expand(B, 3, V)
    for drawn in (False, True):
        tokens = torch.zeros(B, 3, dtype=torch.int64, device=d)
        if drawn:
            tokens[:, 1:] = torch.multinomial(q, 2 * B, replacement=True, generator=g).view(B, 2)
        else:
            tokens[:, 1], tokens[:, 2] = 3, 7
        u = torch.rand(B, 3, generator=g, device=d)
        e = torch.empty(B, V, device=d).exponential_(generator=g)
        path, kept, token = verify_drafts(logits, tokens, parents, uniforms=u, noise=e,
                                          draft_probs=q.expand(B, 3, V) if drawn else None)
        first = torch.where(kept > 1, tokens.gather(1, path[:, 1:2].clamp(min=0).long())[:, 0], token)
        freq = torch.bincount(first, minlength=V).double().cpu() / B
        want = p.double().cpu()
        assert bool(((freq - want).abs() <= 5 * (want * (1 - want) / B).sqrt()).all()), (drawn, freq, want)
        share = (kept > 1).double().mean().item()
        if drawn:
            assert share > 0
        else:  # p_3 + (1 - p_3) p_7 / (1 - p_3): what is kept are the two tokens' probabilities
            both = (want[3] + want[7]).item()
            assert abs(share - both) <= 5 * (both * (1 - both) / B) ** 0.5


# ---------------------------------------------------------------------------------------


def random_caches(layers, order, B, hk, D, cap, slots, counts, dtype, d, g):
    from poly_attention import DraftCache

    n = torch.tensor(counts, dtype=torch.int32, device=d)
    caches = [DraftCache.empty(order=order, batch=B, kv_heads=hk, dim_head=D, capacity=cap, max_drafts=slots,
                               dtype=DT[dtype], device=d, counts=n) for _ in range(layers)]
    for c in caches:
        fill_cache(c, g, d, stale=3.0)
    return caches


BUFS = ("qs", "vs", "msgs", "lses")


@param("layers,order,B,hk,D,dtype", [(1, 2, 3, 2, 64, "bf16"), (3, 3, 3, 1, 40, "f32"), (30, 2, 3, 1, 8, "f16")])
def test_commit(layers, order, B, hk, D, dtype):
    from poly_attention import commit_drafts

    d = dev()
    g = torch.Generator().manual_seed(layers)
    counts, cap, slots = [5, 0, 30], 33, 9
    caches = random_caches(layers, order, B, hk, D, cap, slots, counts, dtype, d, g)
    path = torch.tensor([[0, 2, 3, 7, -1, -1, -1], [0, 1, 2, -1, -1, -1, -1], [8, 0, 8, 4, 5, 6, 1]],
                        dtype=torch.int32, device=d)
    kept = torch.tensor([4, 0, 7], dtype=torch.int32, device=d)
    want = []
    for c in caches:
        for name in BUFS:
            for dst, src in zip(getattr(c, name), getattr(c, "draft_" + name)):
                w = dst.clone()
                w[0, :, 5:9] = src[0][:, [0, 2, 3, 7]]
                w[2, :, 30:33] = src[2][:, [8, 0, 8]]  # four more do not fit
                want.append(w)
    commit_drafts(caches, path, kept)
    got = [t for c in caches for name in BUFS for t in getattr(c, name)]
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert caches[0].lengths() == [9, 0, 33]
    with pytest.raises(RuntimeError, match="overflow"):
        caches[0].check_overflow()


def test_commit_bad_paths_and_views():
    """An entry that is no slot ends a path; a count out of range is taken as the bound; path as a view."""
    from poly_attention import commit_drafts

    d = dev()
    g = torch.Generator().manual_seed(2)
    caches = random_caches(1, 2, 4, 2, 64, 20, 4, [3, -4, 99, 6], "bf16", d, g)
    before = caches[0].qs[0].clone()
    wide = torch.full((4, 12), 50, dtype=torch.int32, device=d)
    wide[:, 2:7] = torch.tensor([[0, 1, 4, 2, 3], [3, 2, -1, 0, 0], [0, 1, 2, 3, 0], [-1, 0, 1, 2, 3]], device=d)
    commit_drafts(caches, wide[:, 2:7], torch.tensor([5, 2 ** 31 - 1, 2, 4], dtype=torch.int32, device=d))
    assert caches[0].lengths() == [5, 2, 20, 6]
    want, src = before.clone(), caches[0].draft_qs[0]
    want[0, :, 3:5] = src[0][:, [0, 1]]
    want[1, :, 0:2] = src[1][:, [3, 2]]
    assert torch.equal(caches[0].qs[0], want)
    assert int(caches[0].overflow) == 1


# ---------------------------------------------------------------------------------------
# refusals that need tensors on the GPU


def test_refusals():
    from poly_attention import DraftCache, commit_drafts, verify_drafts

    d = dev()
    c = DraftCache.empty(order=2, batch=2, kv_heads=2, dim_head=64, capacity=32, max_drafts=4, device=d)
    q = torch.zeros(2, 4, 3, 64, dtype=torch.bfloat16, device=d)
    kv = q[:, :2]
    ok = dict(qs=[q, kv, kv], vs=[kv], weights=[None] * 3, eps=1e-6)

    def bad(error, fn, *args, **kw):
        with pytest.raises(error):
            fn(*args, **kw)

    bad(ValueError, c.attend, q[:, :3])
    bad(ValueError, c.attend, q[:1])
    bad(ValueError, c.attend, q[..., :32])
    bad(ValueError, c.attend, torch.zeros(2, 4, 5, 64, dtype=torch.bfloat16, device=d))
    bad(TypeError, c.attend, q.float())
    bad(ValueError, c.attend, q.cpu())
    bad(RuntimeError, c.attend, q.clone().requires_grad_())
    bad(ValueError, c.attend, q, parents=torch.zeros(2, 4, dtype=torch.int32, device=d))
    bad(TypeError, c.attend, q, parents=torch.zeros(2, 3, device=d))
    bad(TypeError, c.attend, q, parents=torch.zeros(2, 3, dtype=torch.uint8, device=d))
    bad(ValueError, commit_drafts, [], torch.zeros(2, 4, dtype=torch.int32, device=d), torch.zeros(2, dtype=torch.int32, device=d))
    bad(ValueError, c.attend, q, parents=torch.zeros(3, dtype=torch.int32))
    for change in (dict(qs=[q, kv]), dict(vs=[kv, kv]), dict(weights=[None]), dict(qs=[q, q, kv]),
                   dict(angles=torch.zeros(3, 65, device=d)), dict(angles=torch.zeros(3, 66, device=d)),
                   dict(angles=torch.zeros(4, 64, device=d)), dict(angles=torch.zeros(3, 64)),
                   dict(weights=[torch.ones(32, device=d), None, None]),
                   dict(angles=torch.zeros(3, 64, device=d), inv_freq=torch.zeros(32, device=d)),
                   dict(inv_freq=torch.zeros(32, device=d), interp=0.0)):
        bad(ValueError, c.append, **{**ok, **change})
    bad(RuntimeError, c.append, **{**ok, "vs": [kv.clone().requires_grad_()]})
    path, kept = torch.zeros(2, 4, dtype=torch.int32, device=d), torch.zeros(2, dtype=torch.int32, device=d)
    other = DraftCache.empty(order=2, batch=2, kv_heads=2, dim_head=64, capacity=32, max_drafts=4, device=d)
    bigger = DraftCache.empty(order=2, batch=2, kv_heads=2, dim_head=64, capacity=33, max_drafts=4, device=d,
                              counts=c.counts)
    bad(ValueError, commit_drafts, [c, other], path, kept)
    bad(ValueError, commit_drafts, [c, bigger], path, kept)
    bad(TypeError, commit_drafts, [c], path.long(), kept)
    bad(ValueError, commit_drafts, [c], path[:1], kept)
    bad(ValueError, commit_drafts, [c], path, kept[:1])
    bad(ValueError, commit_drafts, [c], path.cpu(), kept)
    x, tok = torch.zeros(2, 3, 50, device=d), torch.zeros(2, 3, dtype=torch.int64, device=d)
    u, e = torch.zeros(2, 3, device=d), torch.ones(2, 50, device=d)
    bad(ValueError, verify_drafts, x[0], tok)
    bad(ValueError, verify_drafts, x, tok[:, :2])
    bad(TypeError, verify_drafts, x, tok.int())
    bad(ValueError, verify_drafts, x, tok, uniforms=u)
    bad(ValueError, verify_drafts, x, tok, temperature=torch.ones(2, device=d))
    bad(ValueError, verify_drafts, x, tok, uniforms=u, noise=e[:, :49])
    bad(TypeError, verify_drafts, x, tok, uniforms=u.double(), noise=e)
    bad(ValueError, verify_drafts, x, tok, uniforms=u, noise=e, draft_probs=x[:, :2])
    bad(ValueError, verify_drafts, x, tok.cpu())


# ---------------------------------------------------------------------------------------
# the steps together, through the modules


def make_module(order, kv_heads, d, dtype, **kw):
    from poly_attention import NPolyAttention, Order2PolyAttention

    cfg = dict(heads=4, kv_heads=kv_heads, dim_head=64, causal=True, **kw)
    if order == 2:
        return Order2PolyAttention(dim=64, **cfg).to(d, dtype).eval(), O.order2_forward, cfg
    return (NPolyAttention(dim=64, order=order, **cfg).to(d, dtype).eval(), O.npoly_forward,
            dict(cfg, order=order))


@param("order,kv_heads,dtype", [(2, 4, torch.float32), (2, 2, torch.bfloat16), (2, 1, torch.float32),
                                (3, 4, torch.bfloat16), (3, 2, torch.float32), (4, 1, torch.float32)])
def test_drafted_steps_equal_the_parallel_forward(order, kv_heads, dtype):
    """Rows of different prompt lengths, three drafted steps of trees; after each some way down the tree is
    kept.  Every node's output equals the last output of the parallel causal forward over its row's kept
    tokens and its ancestors (reference tests:103-179 pattern)."""
    from poly_attention import DraftCache, commit_drafts

    d = dev()
    torch.manual_seed(order)
    m, fwd, cfg = make_module(order, kv_heads, d, dtype)
    params = {k: v.float().cpu() for k, v in m.state_dict().items()}
    lens = [6, 3, 1]
    B, T = len(lens), 6
    prompt = torch.randn(B, max(lens), 64).to(dtype)
    table = O.rotary_freqs(64, torch.arange(64))
    rows = [prompt[b, :n].float() for b, n in enumerate(lens)]
    g = torch.Generator().manual_seed(9)
    with torch.no_grad():
        _, cache = m(prompt.to(d), rotary_pos_emb=table[:max(lens)].to(d), return_cache=True)
        dc = DraftCache(cache, capacity=32, max_drafts=8, lengths=lens)
        for step in range(3):
            trees = [make_tree(T, g, "tree") for _ in range(B)]
            x = torch.randn(B, T, 64, generator=g).to(dtype)
            par = torch.tensor(trees, dtype=torch.int32, device=d)
            pos = dc.positions(T, par).cpu().long()
            out, same = m(x.to(d), rotary_pos_emb=table[pos].to(d), cache=dc, parents=par, return_cache=True)
            assert same is dc
            path, kept = torch.full((B, T), -1, dtype=torch.int32), []
            for b in range(B):
                ways = DO.walk_tree(trees[b])
                for t in range(T):
                    seq = torch.cat([rows[b], x[b, ways[t]].float()])[None]
                    ref = fwd(params, cfg, seq, rotary_pos_emb=table[:seq.shape[1]])[:, -1]
                    assert_parity(out[b:b + 1, t], ref, dtype, f"step {step} row {b} node {t}")
                keep = ways[int(torch.randint(0, T, (1,), generator=g))]
                keep = keep[:1 + (step + b) % 4]
                path[b, :len(keep)] = torch.tensor(keep)
                kept.append(len(keep))
                rows[b] = torch.cat([rows[b], x[b, keep].float()])
            commit_drafts([dc], path.to(d), torch.tensor(kept, dtype=torch.int32, device=d))
            assert dc.lengths() == [len(r) for r in rows]


@param("order,dtype", [(2, torch.float32), (3, torch.bfloat16)])
def test_module_rotary_root_value_and_gates(order, dtype):
    """A module's own rotary, root value, gates and soft clamp: drafted steps of one token equal the
    StaticCache's, and a chain of five the same five steps."""
    from poly_attention import DraftCache, StaticCache, commit_drafts

    d = dev()
    torch.manual_seed(3)
    m, _, _ = make_module(order, 4, d, dtype, use_rotary_embed=True, multiply_root_value=True, attn_gate=True,
                          softclamp_value=20.0, prenorm=True)
    rotary, m.rotary_emb = m.rotary_emb.float(), None
    m.rotary_emb = rotary
    x = torch.randn(2, 12, 64).to(d, dtype)
    zero = torch.zeros(2, 1, dtype=torch.int32, device=d)
    one = torch.ones(2, dtype=torch.int32, device=d)
    with torch.no_grad():
        _, cache = m(x[:, :7], return_cache=True)
        sc = StaticCache(cache, capacity=20)
        single = DraftCache(cache, capacity=20)
        chain = DraftCache(cache, capacity=20)
        want, got = [], []
        for i in range(7, 12):
            want.append(m(x[:, i:i + 1], cache=sc))
            got.append(m(x[:, i:i + 1], cache=single))
            commit_drafts([single], zero, one)
        both = m(x[:, 7:], cache=chain)
    want = torch.cat(want, 1)
    assert_parity(torch.cat(got, 1), want, dtype, "one token a step", roundings=2)
    assert_parity(both, want, dtype, "a chain", roundings=2)


class TinyLM(torch.nn.Module):
    def __init__(self, order, d):
        super().__init__()
        from poly_attention import NPolyAttention

        torch.manual_seed(0)
        self.emb = torch.nn.Embedding(40, 64)
        self.layers = torch.nn.ModuleList([NPolyAttention(64, order=order, heads=4, kv_heads=2, dim_head=32,
                                                          causal=True, prenorm=True) for _ in range(2)])
        self.out = torch.nn.Linear(64, 40)
        self.to(d)

    def forward(self, tokens, angles, caches=None, parents=None):
        x = self.emb(tokens)
        new = []
        for i, layer in enumerate(self.layers):
            kw = {} if caches is None else dict(cache=caches[i], parents=parents)
            y, c = layer(x, rotary_pos_emb=angles, return_cache=True, **kw)
            x = x + y
            new.append(c)
        return self.out(x), new


@param("captured", (False, True))
def test_drafted_decoding_gives_the_greedy_tokens(captured):
    """A decoding loop over two layers: trees of drafts, some of them right, decided greedily; the tokens are
    those of the parallel forward, one after another.  Captured: one graph, replayed per step with the
    drafts and counts of that step."""
    from poly_attention import DraftCache, commit_drafts, verify_drafts

    d = dev()
    B, T, steps = 3, 5, 12
    lm = TinyLM(3, d).eval()
    table = O.rotary_freqs(32, torch.arange(128)).to(d)
    g = torch.Generator().manual_seed(4)
    prompt = torch.randint(0, 40, (B, 9), generator=g).to(d)
    lens = [9, 4, 6]
    with torch.no_grad():
        # the truth: each row alone, token by token through the parallel forward
        truth = []
        for b in range(B):
            row = prompt[b:b + 1, :lens[b]]
            for _ in range(steps * T + T):
                logits, _ = lm(row, table[:row.shape[1]])
                row = torch.cat([row, logits[:, -1:].argmax(-1)], 1)
            truth.append(row[0].tolist())
        _, caches = lm(prompt, table[:9])
        counts = torch.tensor([n for n in lens], dtype=torch.int32, device=d)
        caches = [DraftCache(c, 120, max_drafts=T, counts=counts) for c in caches]
        tokens = torch.zeros(B, T, dtype=torch.int64, device=d)
        parents = torch.tensor([-1, 0, 0, 1, 2], dtype=torch.int32, device=d)

        def step():
            angles = table[caches[0].positions(T, parents).long()]
            logits, _ = lm(tokens, angles, caches, parents)
            path, kept, token = verify_drafts(logits, tokens, parents)
            commit_drafts(caches, path, kept)
            return path, kept, token

        done = list(lens)  # decided tokens; the last one is not cached yet
        last = [truth[b][n] for b, n in enumerate(done)]

        def draft():
            # node 0 the last token; of two ways one may be right
            rows = []
            for b in range(B):
                nxt = truth[b][done[b] + 1:done[b] + 3]
                wrong = (nxt[0] + 1) % 40
                right_first = bool(torch.randint(0, 2, (1,), generator=g))
                second = nxt[1] if bool(torch.randint(0, 2, (1,), generator=g)) else (nxt[1] + 3) % 40
                a, c = (nxt[0], wrong) if right_first else (wrong, nxt[0])
                rows.append([last[b], a, c, second if right_first else 0, 0 if right_first else second])
            tokens.copy_(torch.tensor(rows))

        graph = None
        if captured:
            draft()
            start = counts.clone()
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                step()
            torch.cuda.current_stream().wait_stream(side)
            counts.copy_(start)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                result = step()
        for _ in range(steps):
            draft()
            if graph is None:
                result = step()
            else:
                graph.replay()
            path, kept, token = (t.tolist() for t in result)
            for b in range(B):
                way = [tokens[b, t].item() for t in path[b][:kept[b]]]
                new = way + [token[b]]
                assert new == truth[b][done[b]:done[b] + len(new)], (b, done[b])
                done[b] += kept[b]
                last[b] = token[b]
            assert caches[0].lengths() == done
        assert max(done) - max(lens) > steps  # some drafts were kept
        caches[0].check_overflow()
