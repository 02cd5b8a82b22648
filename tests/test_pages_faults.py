"""Faults that the paged cache had and that show without a GPU, one test each."""

import copy
import gc
import io
import weakref

import pytest
import torch

from test_pages import cache, table


def test_no_cache_joins_a_captured_table():
    t = table()
    first = cache(t)
    t._captured = True                         # as a captured call leaves it
    with pytest.raises(RuntimeError, match="captured"):
        cache(t)
    assert t.caches == [first]


@pytest.fixture
def no_collector():
    gc.collect()
    gc.disable()
    yield
    gc.enable()


def test_what_is_given_up_is_gone(no_collector):
    """Caches and their table are let go without the collector of cycles, and a cache alone while its table lives."""
    t = table()
    caches = [cache(t), cache(t, order=3), cache(t)]
    kept = [weakref.ref(x) for x in (t, caches[1], caches[1].keys[0], caches[2].values[1], t.counts)]
    caches[1:2] = []
    assert [r() is None for r in kept] == [False, True, True, False, False]
    assert t.caches == caches
    caches.append(cache(t))
    assert t.caches == caches
    del t, caches
    assert all(r() is None for r in kept)


def test_copies_are_let_go_too(no_collector):
    t = table()
    caches = [cache(t), cache(t)]
    other = copy.deepcopy(caches)
    assert other[0].table is other[1].table is not t and other[0].table.caches == other and t.caches == caches
    kept = weakref.ref(other[0].table), weakref.ref(other[1].keys[0])
    del other
    assert all(r() is None for r in kept)
    assert copy.deepcopy(caches[1]).table.caches[0:] != caches


def test_a_table_copied_by_itself_has_its_caches():
    t = table()
    caches = [cache(t), cache(t)]
    t.counts.fill_(3)
    caches[1].keys[0].fill_(5.0)
    for other in (copy.deepcopy(t), copy.deepcopy({"t": t, "c": caches})["t"]):
        assert len(other.caches) == 2 and all(c.table is other for c in other.caches)
        assert bool((other.caches[1].keys[0] == 5).all()) and other.counts.tolist() == [3, 3]
        assert other.caches[1].keys[0].data_ptr() != caches[1].keys[0].data_ptr()
    again = copy.deepcopy(other)
    assert len(again.caches) == 2 and again.caches[0] is not other.caches[0]


def test_saved_and_loaded():
    t = table()
    caches = [cache(t), cache(t, order=3)]
    caches[1].keys[2].fill_(5.0)
    for what in (t, caches):
        file = io.BytesIO()
        torch.save(what, file)
        file.seek(0)
        got = torch.load(file, weights_only=False)
        got = got.caches if what is t else got
        assert [c.order for c in got] == [2, 3] and got[0].table is got[1].table and got[0].table.caches == got
        assert bool((got[1].keys[2] == 5).all()) and got[0].table._t.counts == got[0].table.counts.data_ptr()


def test_steps_of_many_shapes_are_not_kept(monkeypatch):
    """A packed step has another total each time."""
    c = cache()
    monkeypatch.setattr(c, "_check_q1", lambda q1: None)  # it wants the GPU
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: False)

    class Planned(Exception):
        pass

    def attend(n):
        c.attend(torch.zeros(1, 2, n, 64))

    made = []
    monkeypatch.setattr(c, "_attend_plan", lambda q1: made.append(q1.shape[2]) or "plan")
    monkeypatch.setattr(c, "_check_tokens", lambda shape: (_ for _ in ()).throw(Planned))
    for n in range(1, 400):
        with pytest.raises(Planned):
            attend(n)
    with pytest.raises(Planned):
        attend(399)                            # a shape of late
    assert made == list(range(1, 400)) and 1 <= len(c._plans) <= 64


@pytest.mark.parametrize("dtype, x, want", [
    (torch.uint64, [(1 << 32) + 1, 5], [(1 << 31) - 1, 5]), (torch.uint64, [(1 << 64) - 1, 0], [(1 << 31) - 1, 0]),
    (torch.uint32, [(1 << 32) - 1, 1 << 31], [(1 << 31) - 1] * 2), (torch.uint16, [65535, 1], [65535, 1]),
    (torch.int64, [(1 << 40), -(1 << 40)], [(1 << 31) - 1, -(1 << 31) + 1]), (torch.int8, [-1, 3], [-1, 3]),
])
def test_numbers_of_any_type(dtype, x, want):
    """Numbers that do not fit stay outside every range, instead of becoming others."""
    got = table()._rows_tensor(torch.tensor(x, dtype=dtype), "more")
    assert got.dtype == torch.int32 and got.tolist() == want


@pytest.mark.parametrize("x", [[1.5, 2], [1, 2.0], ["1", 2], [None, 1]])
def test_lists_hold_whole_numbers(x):
    with pytest.raises(TypeError, match="whole"):
        table()._rows_tensor(x, "lengths")
