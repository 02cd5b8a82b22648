"""GPU: faults that the paged cache had, one test each."""

import weakref

import pytest
import torch

from test_gpu_27_pages import dev

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
