"""Paged cache: what is refused, by the classes and by the C entry points (before any launch, so without a GPU), and
the lists that the GPU tests hold the table to."""

import copy
import ctypes

import pytest
import torch

import pages_oracle as PO
from poly_attention import NPolyAttention, PagedCache, PageTable, PolyAttention, _lib


def table(**kw):
    args = dict(rows=2, pages=6, page_size=16, capacity=64, device="cpu")
    args.update(kw)
    return PageTable(args.pop("rows"), **args)


def cache(t=None, **kw):
    args = dict(order=2, kv_heads=2, dim_head=64, dtype=torch.float32)
    args.update(kw)
    return PagedCache(t or table(), **args)


@pytest.mark.parametrize("kw", [dict(rows=0), dict(rows=8193), dict(pages=0), dict(page_size=8), dict(page_size=48),
                                dict(page_size=8192), dict(capacity=0), dict(capacity=(1 << 30) + 1)])
def test_table_refusals(kw):
    with pytest.raises(ValueError):
        table(**kw)


@pytest.mark.parametrize("kw, error", [
    (dict(order=1), ValueError), (dict(order=9), ValueError), (dict(kv_heads=0), ValueError),
    (dict(dim_head=20), ValueError), (dict(dim_head=136), ValueError), (dict(dim_head=264), ValueError),
    (dict(dtype=torch.float64), TypeError),
])
def test_cache_refusals(kw, error):
    with pytest.raises(error):
        cache(**kw)


def test_capacity_is_whole_pages():
    t = table(capacity=33)
    assert t.capacity == 48 and t.pages.shape == (2, 3)


def test_calls_need_the_gpu():
    t = table()
    c = cache(t)
    q = torch.zeros(2, 2, 3, 64)
    for call in (lambda: t.extend([1, 1]), lambda: t.select([0, 1]), lambda: t.compact(), lambda: t.free([0]),
                 lambda: c.append([q] * 3, q, [None] * 3, eps=1e-6), lambda: c.attend(q)):
        with pytest.raises(RuntimeError):
            call()
    for m in (PolyAttention(dim=32, heads=2, use_flash_kernel=False),
              NPolyAttention(dim=32, order=3, heads=2, use_flash_kernel=False)):
        with pytest.raises(RuntimeError):
            m(torch.zeros(2, 3, 32), cache=c)


def test_copies_have_tables_of_their_own():
    t = table()
    caches = [cache(t), cache(t, order=3)]
    other = copy.deepcopy(caches)
    assert other[0].table is other[1].table is not t and other[0].table.caches == other
    assert other[0].keys[0].data_ptr() != caches[0].keys[0].data_ptr()
    assert other[0].table._t.counts == other[0].table.counts.data_ptr() != t.counts.data_ptr()


def test_positions():
    t = table(rows=3, pages=9)
    t.counts.copy_(torch.tensor([5, 0, 20]))
    t.new.copy_(torch.tensor([2, 0, 3]))
    t.starts.copy_(torch.tensor([0, 2, 2, 5]))
    assert t.positions(3).tolist() == [[3, 4, 5], [0, 1, 2], [17, 18, 19]]
    assert t.positions(5, packed=True).tolist() == [[3, 4, 17, 18, 19]]


# ---------------------------------------------------------------------------------------
# the C entry points: every refusal comes before a launch (the addresses are never read)

FAKE = 0x10000


def fill_table(t):
    t.rows, t.pages, t.page_size, t.max_pages = 3, 10, 64, 4
    t.table = t.counts = t.refs = t.fresh = t.starts = t.overflow = t.scratch = FAKE


def view(v, heads, dtype=_lib.PA_BF16, sn=64, sh=4096, sb=65536):
    v.ptr, v.sb, v.sh, v.sn, v.heads, v.dtype = FAKE, sb, sh, sn, heads, dtype


def attend_args(order=3):
    P = _lib.PaPaged()
    fill_table(P.t)
    P.tokens, P.packed, P.heads, P.kv_heads, P.dim, P.order, P.dtype = 5, 0, 4, 2, 64, order, _lib.PA_BF16
    P.scale = 0.125
    view(P.q, 4)
    view(P.out, 4)
    for t in range(order):
        L = P.levels[t]
        L.keys = L.values = FAKE
        if t < order - 1:
            L.lses = FAKE
        if 0 < t < order - 1:
            view(L.vmul, 2)
    P.workspace_bytes = _lib.load().pa_paged_attend_workspace(ctypes.byref(P))
    P.workspace = P.tickets = FAKE
    return P


def set_field(P, path, value):
    *head, name = path.split(".")
    for h in head:
        P = P[int(h)] if h.isdigit() else getattr(P, h)
    setattr(P, name, value)


TABLE_REFUSALS = [("t.rows", 0, -1), ("t.pages", 0, -1), ("t.max_pages", 0, -1), ("t.table", None, -1),
                  ("t.counts", None, -1), ("t.refs", None, -1), ("t.fresh", None, -1), ("t.starts", None, -1),
                  ("t.page_size", 8, -2), ("t.page_size", 65, -2), ("t.page_size", 8192, -2),
                  ("t.rows", 8193, -2), ("t.max_pages", 1 << 25, -2)]


@pytest.mark.parametrize("path, value, want", TABLE_REFUSALS + [
    ("tokens", 0, -1), ("heads", 3, -1), ("kv_heads", 0, -1), ("order", 1, -1), ("order", 9, -1), ("dtype", 7, -1),
    ("dim", 0, -1), ("dim", 20, -2), ("dim", 264, -2), ("q.ptr", None, -1), ("out.ptr", None, -1), ("q.heads", 2, -1),
    ("q.dtype", _lib.PA_F16, -1), ("q.sn", 63, -2), ("out.ptr", FAKE + 8, -2), ("levels.0.keys", None, -1),
    ("levels.1.values", None, -1), ("levels.0.lses", None, -1), ("levels.1.vmul.ptr", None, -1),
    ("levels.1.vmul.heads", 4, -1), ("levels.2.keys", FAKE + 4, -2), ("workspace", None, -4), ("tickets", None, -1),
    ("workspace", FAKE + 8, -4), ("workspace_bytes", 15, -4), ("tokens", 1 << 30, -2)])
def test_attend_refuses(path, value, want):
    lib = _lib.load()
    P = attend_args()
    set_field(P, path, value)
    assert lib.pa_paged_attend(ctypes.byref(P), None) == want
    assert lib.pa_paged_attend(None, None) == _lib.PA_EINVAL


def append_args():
    P = _lib.PaPageRows()
    fill_table(P.t)
    P.tokens, P.dim, P.count, P.eps = 5, 64, 2, 1e-6
    for k in range(2):
        view(P.items[k].src, 2)
    view(P.items[0].out, 2)
    P.items[1].pages = FAKE
    return P


@pytest.mark.parametrize("path, value, want", TABLE_REFUSALS + [
    ("tokens", 0, -1), ("dim", 0, -1), ("dim", 12, -2), ("count", 0, -1), ("count", 11, -1), ("items.0.src.ptr", None, -1),
    ("items.0.src.heads", 0, -1), ("items.1.src.dtype", _lib.PA_F32, -1), ("items.0.out.heads", 1, -1),
    ("items.0.out.dtype", _lib.PA_F32, -1), ("items.1.pages", None, -1), ("items.0.pages", FAKE, -1),
    ("items.1.src.sn", 60, -2), ("items.1.pages", FAKE + 8, -2), ("tokens", 1 << 28, -2)])
def test_append_refuses(path, value, want):
    P = append_args()
    set_field(P, path, value)
    assert _lib.load().pa_page_append(ctypes.byref(P), None) == want


@pytest.mark.parametrize("angles", [dict(angles=FAKE, rot_dim=3), dict(angles=FAKE, rot_dim=66),
                                    dict(angles=FAKE, rot_dim=4, angles_dtype=5), dict(inv_freq=FAKE, rot_dim=4, interp=0.0)])
def test_append_refuses_angles(angles):
    P = append_args()
    for k, v in angles.items():
        setattr(P, k, v)
    assert _lib.load().pa_page_append(ctypes.byref(P), None) == _lib.PA_EINVAL


@pytest.mark.parametrize("path, value, want", TABLE_REFUSALS + [("t.scratch", None, -4), ("t.scratch", FAKE + 8, -4)])
@pytest.mark.parametrize("name", ["pa_page_select", "pa_page_extend", "pa_page_compact"])
def test_table_calls_refuse(name, path, value, want):
    C = _lib.PaPageCall()
    fill_table(C.t)
    C.index = C.more = FAKE
    set_field(C, path, value)
    call = getattr(_lib.load(), name)
    assert call(ctypes.byref(C), None) == want
    fill_table(C.t)
    C.index = C.more = None
    C.count = 1  # arrays are missing
    assert call(ctypes.byref(C), None) == _lib.PA_EINVAL
    assert call(None, None) == _lib.PA_EINVAL


def test_sizes_of_nothing():
    lib = _lib.load()
    assert lib.pa_page_scratch(None) == 0 and lib.pa_page_scratch(ctypes.byref(_lib.PaPageTable())) == 0
    assert lib.pa_paged_attend_workspace(None) == 0
    assert lib.pa_paged_attend_workspace(ctypes.byref(_lib.PaPaged())) == 0


# ---------------------------------------------------------------------------------------
# the lists


def test_oracle_table():
    t = PO.Table(3, 6, 16, 64)
    assert t.extend([20, 16, 0]) == [] and t.pages == [[0, 1], [2], []]
    t.select([0, 1, 0])
    assert t.refs == [2, 2, 1, 0, 0, 0] and t.counts == [20, 16, 20]
    # both write page 1: the first row copies it, the last keeps it
    assert t.extend([1, 0, 1]) == [(1, 3, 4)] and t.pages == [[0, 3], [2], [0, 1]]
    assert t.refs == [2, 1, 1, 1, 0, 0] and t.starts == [0, 1, 1, 2]
    # two pages are left: row 1 needs three, the rows behind it none
    assert t.extend([2, 40, 1]) == [] and t.new == [2, 0, 1] and t.overflow
    t.select([-1, 1, 2], [9, 9, 17])
    assert t.counts == [0, 9, 17] and t.refs == [1, 1, 1, 0, 0, 0]
    t.select([-1, 1, -1])
    assert t.compact() == [(2, 0)] and t.pages == [[], [0], []]


def test_oracle_table_waits():
    """A row that is to keep a shared page does not write it while a row before it still has it."""
    t = PO.Table(3, 2, 16, 64)
    t.extend([20, 0, 0])
    t.select([0, 0, -1])
    t.overflow = False
    assert t.extend([1, 1, 0]) == [] and t.new == [0, 0, 0] and t.overflow


@pytest.mark.parametrize("dtype, tokens", [(_lib.PA_F32, 1 << 27), (_lib.PA_BF16, 1 << 29)])
def test_attend_refuses_more_units_than_a_launch_has(dtype, tokens):
    P = attend_args(2)
    P.dtype = P.q.dtype = P.out.dtype = dtype
    P.heads = P.q.heads = P.out.heads = 2
    P.tokens = tokens
    P.workspace_bytes = _lib.load().pa_paged_attend_workspace(ctypes.byref(P))
    assert _lib.load().pa_paged_attend(ctypes.byref(P), None) == _lib.PA_EUNSUPPORTED


def test_attend_refuses_more_heads_than_tickets():
    P = attend_args(2)
    P.heads = P.q.heads = P.out.heads = P.kv_heads = 5000
    P.workspace_bytes = _lib.load().pa_paged_attend_workspace(ctypes.byref(P))
    assert _lib.load().pa_paged_attend(ctypes.byref(P), None) == _lib.PA_EUNSUPPORTED
