"""GPU: the paged cache's attention where a row's positions are many units -- joins in one and in two steps, at once on two
streams, replayed --, what is not finite behind few rows, rotary embeddings far along, and copies of large
pages."""

import pytest
import torch

import pages_oracle as PO
from test_gpu_27_pages import DT, assert_within, check_attend, dev, fill, inputs, make

pytestmark = pytest.mark.gpu
param = pytest.mark.parametrize


@param("counts, new, H, hk, D, dtype, ps", [
    ([70000], [1], 2, 1, 64, "bf16", 256),             # over a hundred units of a tile
    ([40000, 5, 33000], [3, 5, 16], 2, 1, 64, "f16", 64),
    ([30011], [8], 4, 1, 128, "bf16", 32),             # 32 rows of a key head
    ([9000, 700], [30, 1], 1, 1, 256, "bf16", 128),
    ([5000, 1300], [33, 20], 2, 1, 96, "f32", 16),     # several tiles of a chunk, each of several units
    ([20000], [16], 1, 1, 8, "f32", 16),
    ([12000], [300], 2, 1, 128, "f16", 4096),          # many rows, few and many units
    ([6000, 129], [257, 129], 8, 2, 64, "bf16", 16),
])
def test_many_units(counts, new, H, hk, D, dtype, ps):
    check_attend(2, counts, new, H, hk, D, dtype, ps)


@param("dtype", ["bf16", "f16", "f32"])
@param("D", [64, 128, 256])
@param("counts, new, heads", [([100], [6], 2), ([3000], [6], 2), ([3000], [16], 4), ([21], [21], 2)])
def test_few_rows_see_nothing_behind_them(counts, new, heads, D, dtype):
    """Infinities and NaN at later tokens of a chunk of few rows reach no earlier token, in one unit and in several."""
    from poly_attention import PagedCache

    outs = []
    for bad in (False, True):
        g = torch.Generator().manual_seed(3)
        t, o = make(counts, new, 16, g)
        cache = PagedCache(t, order=2, kv_heads=2, dim_head=D, dtype=DT[dtype])
        fill(cache, o, g)
        q1 = inputs(o, heads, D, DT[dtype], False, g).cuda()
        if bad:
            for p, x in ((counts[0] - 3, float("inf")), (counts[0] - 1, float("nan")), (counts[0] - 2, -float("inf"))):
                page, slot = o.pages[0][p // 16], p % 16
                cache.values[0][page, :, slot, ::3] = x
                cache.keys[0][page, :, slot] = x
        outs.append(cache.attend(q1))
    a, b = outs
    m = new[0] - 3
    assert bool(torch.isfinite(a.float()).all())
    # the same products in the same order but for those of values that are no numbers, whose weights are 0
    assert torch.equal(a[:, :, :m], b[:, :, :m])
    assert not bool(torch.isfinite(b[:, :, -1, ::3].float()).any())


@param("dtype", ["bf16", "f32"])
def test_a_value_that_is_infinite(dtype):
    """A value of infinity that all rows see is theirs, and of no other feature."""
    from poly_attention import PagedCache

    g = torch.Generator().manual_seed(6)
    t, o = make([60], [4], 16, g)
    cache = PagedCache(t, order=2, kv_heads=1, dim_head=64, dtype=DT[dtype])
    fill(cache, o, g)
    q1 = inputs(o, 1, 64, DT[dtype], False, g).cuda()
    cache.values[0][o.pages[0][3], 0, 9, 5] = float("inf")     # the second token of the chunk
    got = cache.attend(q1).float()[0, 0]
    assert bool(torch.isfinite(got[0]).all())
    for i in (1, 2, 3):
        bad = ~torch.isfinite(got[i])
        assert bool(bad[5])


def test_two_layers_at_once():
    """Two caches of one table on two streams at once, and a graph of one between them."""
    from poly_attention import PagedCache

    g = torch.Generator().manual_seed(12)
    t, o = make([9000, 4000], [2, 1], 64, g)
    caches = [PagedCache(t, order=2, kv_heads=1, dim_head=64, dtype=torch.bfloat16) for _ in range(2)]
    q1 = []
    for c in caches:
        fill(c, o, g)
        q1.append(inputs(o, 4, 64, torch.bfloat16, False, g).cuda())
    want = [c.attend(q) for c, q in zip(caches, q1)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                got[k].append(caches[k].attend(q1[k]))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = caches[0].attend(q1[0])
    for _ in range(5):
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[0])
        got[1].append(caches[1].attend(q1[1]))
        got[0].append(caches[0].attend(q1[0]))
    for k in range(2):
        assert all(torch.equal(x, want[k]) for x in got[k])


@param("dtype", ["bf16", "f16", "f32"])
@param("first", [0, 4093, 60000])
def test_rotary_far_along(dtype, first):
    """A module's frequencies at far positions: 16-bit types take sines and cosines that are 2^-20 off."""
    from poly_attention import PagedCache

    d, dt = dev(), DT[dtype]
    g = torch.Generator().manual_seed(4)
    t, o = make([first + 40], [40], 64, g)
    cache = PagedCache(t, order=2, kv_heads=2, dim_head=64, dtype=dt)
    qs = [inputs(o, 2, 64, dt, False, g) for _ in range(3)]
    v = inputs(o, 2, 64, dt, False, g)
    inv = 10000.0 ** -(torch.arange(0, 64, 2).float() / 64)
    q1 = cache.append([q.to(d) for q in qs], v.to(d), [None] * 3, eps=1e-6, inv_freq=inv.to(d))
    for i in range(40):
        pos = torch.tensor(float(first + i)).to(dt).float()
        a = (pos * inv).repeat_interleave(2)
        x = qs[0][0, :, i]
        y, tol = PO.append(x, None, 1e-6, a, dt)
        turned = torch.stack([x[:, 1::2], x[:, 0::2]], -1).flatten(-2)
        assert_within(q1[0, :, i], y, tol + (x.double().abs() + turned.double().abs()) * 2.0 ** -20, f"token {i}")


@param("ps, hk, D, dtype", [(4096, 4, 128, "bf16"), (16, 2, 8, "f32"), (256, 3, 40, "f16")])
@param("held", [1, 5, 255])
def test_copies_of_any_page(ps, hk, D, dtype, held):
    """A fork's copy of a partly filled page, of the positions that it holds in every array, and a compaction's of whole ones."""
    from poly_attention import PagedCache, PageTable

    held = min(held, ps - 1)
    t = PageTable(3, pages=8, page_size=ps, capacity=2 * ps)
    caches = [PagedCache(t, order=n, kv_heads=hk, dim_head=D, dtype=DT[dtype]) for n in (2, 3)]
    t.extend([ps, 0, held])                       # pages 0 and 1
    for c in caches:
        for x in c.arrays():
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(x.numel())).to(x.dtype))
    was = [x.clone() for c in caches for x in c.arrays()]
    t.select([-1, 2, 2])                          # page 0 is free, page 1 of two rows
    t.extend([0, 1, 1])
    torch.cuda.synchronize()
    assert t.pages[1, 0].item() == 0 and t.pages[2, 0].item() == 1
    now = [x for c in caches for x in c.arrays()]
    for x, y in zip(now, was):
        assert torch.equal(x[0, :, :held], y[1, :, :held]), "the copy"
        assert torch.equal(x[0, :, held:], y[0, :, held:]) and torch.equal(x[1:], y[1:]), "nothing else"
    t.select([-1, -1, 2])
    t.compact()
    assert t.pages[2, 0].item() == 0
    for x, y in zip(now, was):
        assert torch.equal(x[0], y[1]) and torch.equal(x[1:], y[1:])


@param("D", [64, 128])
def test_captured_chunks(D):
    """Chunks of many and of few rows, captured and replayed between eager calls over other contents."""
    from poly_attention import PagedCache

    d = dev()
    g = torch.Generator().manual_seed(21)
    t, o = make([900, 300, 2000], [400, 1, 30], 64, g)
    cache = PagedCache(t, order=3, kv_heads=2, dim_head=D, dtype=torch.bfloat16)
    fill(cache, o, g)
    xs = [(inputs(o, 8, D, torch.bfloat16, True, g).to(d), inputs(o, 2, D, torch.bfloat16, True, g).to(d)) for _ in range(4)]
    want = [cache.attend(q, [v]) for q, v in xs]
    q, v = (x.clone() for x in xs[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.attend(q, [v])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = cache.attend(q, [v])
    for k in (1, 3, 0, 2, 2):
        q.copy_(xs[k][0])
        v.copy_(xs[k][1])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[k])
        assert torch.equal(cache.attend(*[xs[3 - k][0], [xs[3 - k][1]]]), want[3 - k])


@param("rows", [1000, 8192])
def test_thousands_of_rows(rows):
    """Every row finds its chunk and its pages: packed and padded steps give the same, and each row what it gives alone."""
    from poly_attention import PagedCache, PageTable

    d = dev()
    g = torch.Generator().manual_seed(rows)
    more = torch.randint(0, 4, (rows,), generator=g)
    more[0], more[-1] = 3, 2
    T, hk, D = 3, 2, 64
    steps = [more, (more + 1) % 4]
    total = [int(m.sum()) for m in steps]
    qs = [[torch.randn(rows, hk, T, D, generator=g).to(torch.bfloat16).to(d) for _ in range(4)] for _ in steps]
    got = []
    for packed in (False, True):
        t = PageTable(rows, pages=rows + 40, page_size=16, capacity=32, device=d)
        c = PagedCache(t, order=2, kv_heads=hk, dim_head=D)
        outs = []
        for m, q in zip(steps, qs):
            t.extend(m.to(d, torch.int32))
            here = (torch.arange(T) < m[:, None]).to(d)                                  # [rows, T]
            if packed:
                q = [x.transpose(1, 2)[here].transpose(0, 1)[None].contiguous() for x in q]
            q1 = c.append(q[:3], q[3], [None] * 3, eps=1e-6)
            y = c.attend(q1)
            if packed:
                z = torch.zeros(rows, T, hk, D, dtype=y.dtype, device=d)
                z[here] = y[0].transpose(0, 1)
                y = z.transpose(1, 2)
            outs.append(y)
        assert t.counts.tolist() == (steps[0] + steps[1]).tolist() and not t.overflow.item()
        assert t.starts[-1].item() == total[1]
        used = t.pages[t.pages >= 0]
        assert used.numel() == used.unique().numel() == int((t.refs > 0).sum())
        got.append(outs)
    for a, b in zip(*got):
        assert torch.equal(a, b)
    for b in (0, 1, 63, 64, rows // 2, rows - 1):                                        # alone
        t = PageTable(1, pages=4, page_size=16, capacity=32, device=d)
        c = PagedCache(t, order=2, kv_heads=hk, dim_head=D)
        for k, (m, q) in enumerate(zip(steps, qs)):
            n = int(m[b])
            t.extend([n])
            if not n:
                continue
            one = [x[b:b + 1, :, :n].contiguous() for x in q]
            y = c.attend(c.append(one[:3], one[3], [None] * 3, eps=1e-6))
            assert torch.equal(y, got[0][k][b:b + 1, :, :n])
