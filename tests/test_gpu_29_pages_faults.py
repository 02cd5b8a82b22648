"""GPU: faults that the paged cache had, one test each."""

import weakref

import pytest
import torch

from test_gpu_27_pages import DT, dev, fill, inputs, make

pytestmark = pytest.mark.gpu
param = pytest.mark.parametrize


# ---------------------------------------------------------------------------------------
# what captured steps hold


def test_no_cache_joins_a_captured_table():
    """A captured extend copies the shared pages of the caches there were: another one is refused (nothing is replayed here)."""
    from poly_attention import PagedCache, PageTable

    d = dev()
    t = PageTable(2, pages=6, page_size=16, capacity=64)
    new = lambda: PagedCache(t, order=2, kv_heads=1, dim_head=8, dtype=torch.float32)  # noqa: E731
    caches = [new()]
    more = torch.ones(2, dtype=torch.int32, device=d)
    t.extend(more)
    caches.append(new())                       # nothing was captured yet
    t.extend(more)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        t.extend(more)
    with pytest.raises(RuntimeError, match="captured"):
        new()
    assert len(t.caches) == 2
    t.extend(more)                             # the table's own calls go on


def test_the_scratch_stays():
    """Its size is the table's alone: no further cache moves it."""
    from poly_attention import PagedCache, PageTable

    dev()
    t = PageTable(3, pages=6, page_size=16, capacity=64)
    where = []
    caches = []
    for _ in range(3):
        caches.append(PagedCache(t, order=2, kv_heads=1, dim_head=8, dtype=torch.float32))
        t.extend([1, 0, 1])
        where.append(t._t.scratch)
    assert where[0] and where == where[:1] * 3


def test_captured_table_calls_after_much_else():
    """Graphs of a table's calls replayed after eager calls and allocations of all sizes: the pages, counts and copies of the
    eager calls."""
    from poly_attention import PagedCache, PageTable

    d = dev()
    runs = []
    for captured in (False, True):
        t = PageTable(4, pages=40, page_size=16, capacity=128)
        caches = [PagedCache(t, order=2, kv_heads=1, dim_head=8, dtype=torch.float32) for _ in range(2)]
        for k, x in enumerate(x for c in caches for x in c.arrays()):
            x.copy_(torch.arange(x.numel(), device=d).view(x.shape) + k)
        more, index = (torch.zeros(4, dtype=torch.int32, device=d) for _ in range(2))
        calls = [lambda: t.extend(more), lambda: t.select(index), t.compact]
        calls[0]()
        graphs = []
        if captured:
            torch.cuda.synchronize()
            for call in calls:
                graphs.append(torch.cuda.CUDAGraph())
                with torch.cuda.graph(graphs[-1]):
                    call()
        seen = []
        for step in range(6):
            more.copy_(torch.tensor([[20, 5, 0, 3], [1, 1, 1, 1], [0, 17, 2, 1]][step % 3]))
            index.copy_(torch.tensor([[0, 0, 2, 1], [1, -1, 2, 1]][step % 2]))
            junk = [torch.full((n,), 0x7f7f7f7f, dtype=torch.int32, device=d) for n in (4, 64, 200, 1000, 5000, 100000)]
            for k in range(3):
                graphs[k].replay() if captured else calls[k]()
            torch.cuda.synchronize()
            del junk
            seen.append([x.clone() for x in (t.pages, t.counts, t.refs, t.new, t.starts)])
            seen[-1] += [x.clone() for c in caches for x in c.arrays()]
            t.free([step % 4])                 # an eager call between the replays
        runs.append(seen)
    for a, b in zip(*runs):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


# ---------------------------------------------------------------------------------------
# caches that are given up


def test_a_cache_that_is_gone_is_not_copied():
    """Its memory is others' at once, and the table's calls leave it alone."""
    from poly_attention import PagedCache, PageTable

    d = dev()
    t = PageTable(3, pages=8, page_size=16, capacity=64)
    caches = [PagedCache(t, order=2, kv_heads=1, dim_head=64, dtype=torch.float32) for _ in range(2)]
    t.extend([5, 40, 0])
    gone = [weakref.ref(x) for x in caches[0].arrays()]
    assert t._call_struct.count == 10
    del caches[0]
    assert all(r() is None for r in gone)
    theirs = [torch.full((8, 1, 16, 64), 7.0, device=d) for _ in range(200)]
    t.select([0, 1, 0])
    t.extend([1, 0, 1])                        # row 0 copies the page that it shares
    t.free([0])
    t.compact()
    assert t._call_struct.count == 5
    assert all(bool((x == 7).all()) for x in theirs)
    assert t.counts.tolist() == [0, 40, 6]


def test_a_captured_call_keeps_its_arrays():
    from poly_attention import PagedCache, PageTable

    d = dev()
    t = PageTable(3, pages=8, page_size=16, capacity=64)
    caches = [PagedCache(t, order=2, kv_heads=1, dim_head=64, dtype=torch.float32) for _ in range(2)]
    index = torch.tensor([0, 1, 0], dtype=torch.int32, device=d)
    more = torch.tensor([1, 0, 1], dtype=torch.int32, device=d)
    t.extend([5, 40, 0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        t.select(index)
        t.extend(more)
    keys = weakref.ref(caches[0].keys[0])
    del caches[0]
    assert keys() is not None and len(t.caches) == 1
    theirs = [torch.full((8, 1, 16, 64), 7.0, device=d) for _ in range(200)]
    for step in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert t.counts.tolist() == [6 + step, 40, 6 + step]
    t.extend([1, 1, 1])                        # eager calls go on
    assert all(bool((x == 7).all()) for x in theirs)
    del t, caches, graph


@param("what", ["append", "attend"])
def test_a_captured_step_keeps_its_cache(what):
    """The step alone is captured, and the cache given up while its table lives."""
    from poly_attention import PagedCache, PageTable

    d = dev()
    g = torch.Generator().manual_seed(1)
    t = PageTable(2, pages=8, page_size=16, capacity=64)
    cache = PagedCache(t, order=2, kv_heads=1, dim_head=64, dtype=torch.float32)
    qs = [torch.randn(2, 1, 4, 64, generator=g).to(d) for _ in range(4)]
    t.extend([4, 3])

    def step():
        q1 = cache.append(qs[:3], qs[3], [None] * 3, eps=1e-6)
        return cache.attend(q1) if what == "attend" else q1

    want = step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step()
    kept = [weakref.ref(x) for x in (*cache.arrays(), cache._tickets)]
    del step, cache
    assert not t.caches and all(r() is not None for r in kept)
    theirs = [torch.full((8, 1, 16, 64), 7.0, device=d) for _ in range(200)]
    for _ in range(3):
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
    assert all(bool((x == 7).all()) for x in theirs)
    del graph, t
    assert all(r() is None for r in kept)


@param("dtype", [torch.uint64, torch.uint32, torch.int64])
def test_counts_of_any_type(dtype):
    from poly_attention import PageTable

    d = dev()
    t = PageTable(2, pages=8, page_size=16, capacity=64)
    t.extend(torch.tensor([3, 17], dtype=dtype).to(d))
    assert t.counts.tolist() == [3, 17]
    t.extend(torch.tensor([(1 << 31) + 1 if dtype == torch.uint32 else (1 << 32) + 1, 1], dtype=dtype).to(d))
    assert t.counts.tolist() == [3, 18] and t.new.tolist() == [0, 1] and bool(t.overflow.item())


# ---------------------------------------------------------------------------------------
# numbers that are none


@param("dtype", ["bf16", "f16", "f32"])
@param("counts, new, heads, D, lo, hi", [
    ([100], [1], 2, 64, 0, 32),                # all that one wave has, of a unit
    ([100], [1], 2, 64, 0, 16),                # a half of it (fp32: the same)
    ([100], [100], 2, 64, 0, 100),             # all there is
    ([9000], [3], 4, 64, 0, 8000),             # whole units of several
    ([9000], [40], 2, 128, 4000, 8000),        # in two steps of the join
    ([300], [200], 2, 64, 0, 64),              # many rows, one unit
    ([5000], [300], 2, 64, 0, 2048),           # many rows, several units
    ([5000], [300], 2, 128, 0, 4500),
    ([5000], [300], 4, 96, 2048, 4500),
])
def test_keys_that_are_no_numbers(counts, new, heads, D, dtype, lo, hi):
    """Softmaxes over a score that is no number are none, wherever the others of its wave or unit are none either."""
    from poly_attention import PagedCache

    dev()
    g = torch.Generator().manual_seed(4)
    t, o = make(counts, new, 16, g)
    cache = PagedCache(t, order=3, kv_heads=2, dim_head=D, dtype=DT[dtype])
    fill(cache, o, g)
    n, m = counts[0], new[0]
    for p in range(lo, hi):
        cache.keys[0][o.pages[0][p // 16], 1, p % 16] = float("nan")
    q1 = inputs(o, heads, D, DT[dtype], False, g).cuda()
    v = inputs(o, 2, D, DT[dtype], False, g).cuda()
    out = cache.attend(q1, [v]).float().cpu()
    sees = torch.arange(n - m, n) >= lo
    half = heads // 2
    assert bool(torch.isfinite(out[0, :half]).all())
    assert bool(torch.isnan(out[0, half:, sees]).all())
    assert bool(torch.isfinite(out[0, half:, ~sees]).all())
    for lse, value in zip(cache.lses, cache.values[1:]):
        where = [(o.pages[0][p // 16], p % 16) for p in range(n - m, n)]
        got = torch.stack([lse[page, 1, slot] for page, slot in where]).cpu()
        assert torch.equal(torch.isnan(got), sees)
        got = torch.stack([value[page, 1, slot] for page, slot in where]).float().cpu()
        assert torch.equal(torch.isnan(got).all(-1), sees)


@param("dtype", ["bf16", "f16", "f32"])
@param("D, rot", [(64, 32), (128, 2), (40, 14)])
def test_features_that_are_not_turned(D, rot, dtype):
    """They are as they were beside an infinite one."""
    from poly_attention import PagedCache

    d = dev()
    g = torch.Generator().manual_seed(5)
    t, o = make([20, 9], [7, 9], 16, g)
    cache = PagedCache(t, order=2, kv_heads=2, dim_head=D, dtype=DT[dtype])
    qs = [inputs(o, 2, D, DT[dtype], False, g).to(d) for _ in range(3)]
    v = inputs(o, 2, D, DT[dtype], False, g).to(d)
    for x in qs:
        x[..., rot + 1::4] = float("inf")
        x[..., rot + 2::4] = float("nan")
    q1 = cache.append(qs, v, [None] * 3, eps=1e-6, angles=torch.randn(rot, generator=g).to(d))
    for b, n in enumerate(o.new):
        assert torch.equal(q1[b, :, :n, rot:].nan_to_num(77), qs[0][b, :, :n, rot:].nan_to_num(77))
        assert bool(torch.isfinite(q1[b, :, :n, :rot]).all())


# ---------------------------------------------------------------------------------------
# rows that do not get their pages


def test_rows_behind_one_that_finds_no_pages():
    """As the documentation says: behind it none that needs a page, with free ones there, and those that need none do."""
    from poly_attention import PageTable

    dev()
    t = PageTable(5, pages=8, page_size=16, capacity=160)
    t.extend([10, 10, 16, 5, 0])
    assert t.pages[:, 0].tolist() == [0, 1, 2, 3, -1] and t.free_pages() == 4
    t.extend([100, 3, 1, 12, 1])               # row 0 needs six pages of the four, row 1 none, row 2 one, rows 3 and 4 one each
    assert t.new.tolist() == [0, 3, 0, 0, 0] and t.counts.tolist() == [10, 13, 16, 5, 0] and t.free_pages() == 4
    assert t.starts.tolist() == [0, 100, 103, 104, 116, 117] and bool(t.overflow.item())
    t.overflow.zero_()
    t.extend([151, 3, 1, 12, 1])               # row 0 passes its capacity: the others are not affected
    assert t.new.tolist() == [0, 3, 1, 12, 1] and t.free_pages() == 1 and bool(t.overflow.item())


def test_a_row_that_waits_for_a_shared_page():
    from poly_attention import PageTable

    dev()
    t = PageTable(3, pages=3, page_size=16, capacity=64)
    t.extend([20, 0, 5])
    t.select([0, 0, 2])
    t.extend([1, 1, 1])                        # rows 0 and 1 write page 1, no page is free for row 0's copy
    assert t.new.tolist() == [0, 0, 1] and t.refs.tolist() == [2, 2, 1] and bool(t.overflow.item())
    t.free([0])
    t.extend([0, 1, 1])
    assert t.new.tolist() == [0, 1, 1] and t.refs.tolist() == [1, 1, 1]
