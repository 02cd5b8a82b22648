"""A poly KV cache in pages: rows of any lengths in one pool, chunks of new tokens at once, rows that share what
they have in common.  No counterpart in the reference, whose cached step takes one token of one position for
the whole batch (poly_attention.py:283-287, n_poly_attention.py:196-207).

A ``PageTable`` says which pages of a pool each row has, for all layers of a model; a ``PagedCache`` is one
layer's keys, values and logsumexps in such pages.  A step brings every row a chunk of new tokens: a prompt's, a
piece of one, a single token, or none::

    table = PageTable(rows=32, pages=4096, page_size=64, capacity=8192)
    caches = [PagedCache(table, order=2, kv_heads=8, dim_head=128) for _ in range(layers)]

    table.extend(more)                       # more[b] new tokens for row b: pages for them
    logits = model(tokens, caches)           # each layer: layer(x, cache=)

``x`` is [rows, T, dim], row b's tokens first and padding behind them, or packed, [1, sum(more), dim], one
row's tokens behind the other's.  A token attends to its row's cached positions and to the tokens of its own chunk
up to itself.  T holds the longest chunk, packed all of them: tokens of a chunk behind it would count as cached without
having been written (a list given to ``extend`` is checked for it, device numbers cannot be).  Rows are forked, freed, cut and reordered with ``PageTable.select``; pages are shared until
one of their rows writes to them.

All of it works on the device's counts, without a host synchronisation, so a step of fixed shapes can be captured
into a HIP graph.  The calls are for the GPU and for inference.
"""

from __future__ import annotations

import copy
import ctypes
import operator
import weakref
from typing import Optional, Sequence

import torch
from torch import Tensor

from . import _lib
from ._lib import DTYPE_CODE, PA_MAX_PAGE_ROWS
from .drafts import _call, _need, _no_tangents, _rows16, _set_view

_PLANS = 32  # shapes of steps that a cache keeps the calls' structures for: packed steps may each have another
_NO_GRAD = "PagedCache steps are inference-only: run them under torch.no_grad()"


def _capturing(device) -> bool:
    if device.index == torch._C._cuda_getDevice():
        return torch._C._cuda_isCurrentStreamCapturing()
    with torch.cuda.device(device):
        return torch._C._cuda_isCurrentStreamCapturing()


class PageTable:
    """Which pages each of ``rows`` rows has, out of a pool of ``pages`` pages of ``page_size`` positions (a power
    of two, 16 to 4096); a row holds at most ``capacity`` positions (whole pages).

    Device tensors, int32, written in place and always the same objects: ``pages`` [rows, pages of a row] (position
    p of row b is place p % page_size of page ``pages[b, p // page_size]``; -1 behind a row's pages),
    ``counts`` [rows] (positions, with the chunk's), ``new`` [rows] (the chunk's tokens), ``starts`` [rows + 1]
    (the first token of each row's chunk in a packed step), ``refs`` [pool] (how many entries name a page; 0:
    free) and ``overflow`` [1].  ``pages``, ``counts`` and ``refs`` together are the state: a copy of the three can be
    written back, as long as the caches' pages were not given to others in between.

    ``caches`` are those that there are: a cache holds its table, not the table its caches, and the pages of one that is given
    up are free memory again, but for pages that a captured call has (of the cache, or of the table), which stay as long as the
    table.  A table whose own calls were captured takes no further caches.

    A table and its caches take one call at a time; others may be used at once, on any streams.  ``copy.deepcopy`` of
    the list of its caches, or of the table, copies the pool; a table copied by itself holds its copies of the caches."""

    def __init__(self, rows: int, *, pages: int, page_size: int = 64, capacity: int, device="cuda"):
        _need(1 <= rows <= PA_MAX_PAGE_ROWS, f"rows {rows}: 1 to {PA_MAX_PAGE_ROWS}")
        _need(16 <= page_size <= 4096 and page_size & (page_size - 1) == 0,
              f"page_size {page_size}: a power of two, 16 to 4096")
        _need(1 <= pages <= 1 << 30, f"pages {pages}: 1 to 2^30")
        _need(1 <= capacity <= 1 << 30, f"capacity {capacity}: 1 to 2^30")
        self.rows, self.pool, self.page_size = rows, pages, page_size
        most = -(-capacity // page_size)
        self.capacity = most * page_size
        i32 = dict(dtype=torch.int32, device=torch.device(device))
        self.pages = torch.full((rows, most), -1, **i32)
        self.counts, self.new = torch.zeros(rows, **i32), torch.zeros(rows, **i32)
        self.refs, self.starts = torch.zeros(pages, **i32), torch.zeros(rows + 1, **i32)
        self.overflow = torch.zeros(1, **i32)
        self.device = self.counts.device
        self._expected = None  # the chunks' tokens, where the host knows them
        self._setup(())

    def _setup(self, caches) -> None:
        """What holds addresses, and the caches."""
        self._t = t = _lib.PaPageTable()
        t.rows, t.pages, t.page_size, t.max_pages = self.rows, self.pool, self.page_size, self.pages.shape[1]
        t.table, t.counts, t.refs = self.pages.data_ptr(), self.counts.data_ptr(), self.refs.data_ptr()
        t.fresh, t.starts, t.overflow = self.new.data_ptr(), self.starts.data_ptr(), self.overflow.data_ptr()
        self._call_struct = self._scratch = self._arrays = None
        self._captured = False  # a call of the table
        self._kept: list = []  # tensors that captured calls have, of the table and of its caches
        self._caches = weakref.WeakValueDictionary(enumerate(caches))
        self._listed = 0  # caches whose arrays are on the list

    @property
    def caches(self) -> list:
        return list(self._caches.values())

    def _add(self, cache) -> None:
        self._caches[max(self._caches, default=-1) + 1] = cache
        self._call_struct = None  # its list of arrays grows

    def _state(self) -> dict:
        gone = ("_t", "_call_struct", "_scratch", "_arrays", "_captured", "_kept", "_caches", "_listed", "_own")
        return {k: v for k, v in self.__dict__.items() if k not in gone}

    def __getstate__(self):
        return {**self._state(), "_own": self.caches}

    def __setstate__(self, state) -> None:
        self.__dict__.update(state)
        self.device = self.counts.device
        self._setup(self._own)

    def _copy(self, memo):
        """A copy without caches."""
        other = memo[id(self)] = object.__new__(type(self))
        other.__setstate__({**copy.deepcopy(self._state(), memo), "_own": []})
        return other

    def __deepcopy__(self, memo):
        other = self._copy(memo)
        other._own = [copy.deepcopy(c, memo) for c in self.caches]
        return other

    def _struct(self):
        """The structure of the table's own calls.  Captured steps hold the addresses of its scratch and of the list of
        arrays: the scratch stays as long as the table, and the list from the first captured call on."""
        c = self._call_struct
        if c is None or (self._listed != len(self._caches) and not self._captured):
            _need(self.device.type == "cuda", "a PageTable's calls need the GPU (libpolyattn)", RuntimeError)
            if _capturing(self.device):
                raise RuntimeError("PageTable: run one eager call before capturing steps (the list of its caches is "
                                   "written then)")
            if self._scratch is None:
                size = _lib.load().pa_page_scratch(ctypes.byref(self._t))
                self._scratch = torch.empty(size, dtype=torch.uint8, device=self.device)
                self._t.scratch = self._scratch.data_ptr()
            caches = self.caches
            arrays = b"".join(bytes(_lib.PaPageArray(x.data_ptr(), x.shape[1], x.element_size() * (x.shape[3] if x.dim() == 4 else 1)))
                              for cache in caches for x in cache.arrays())
            c = _lib.PaPageCall()
            c.count = len(arrays) // ctypes.sizeof(_lib.PaPageArray)
            if arrays:
                self._arrays = torch.frombuffer(bytearray(arrays), dtype=torch.uint8).to(self.device)
                c.arrays = self._arrays.data_ptr()
            c.t = self._t
            self._call_struct, self._listed = c, len(caches)
        elif not self._captured and _capturing(self.device):
            self._captured = True
            self._kept += [x for cache in self.caches for x in cache.arrays()]
        return c

    def _rows_tensor(self, x, what: str) -> Tensor:
        if isinstance(x, Tensor):
            _need(not x.is_floating_point() and not x.is_complex() and x.dtype != torch.bool, f"{what}: whole numbers, not {x.dtype}", TypeError)
            _need(x.shape == (self.rows,), f"{what}: [{self.rows}], not {list(x.shape)}")
            if x.device == self.device:
                if x.dtype != torch.int32:  # whatever does not fit is far outside every range
                    y, most = x.to(torch.int64), (1 << 31) - 1
                    if x.dtype == torch.uint64:
                        y = torch.where(y < 0, most, y)
                    x = y.clamp(-most, most).to(torch.int32)
                return x.contiguous()
            x = x.tolist()
        _need(len(x) == self.rows, f"{what}: one for each of the {self.rows} rows")
        return torch.tensor([max(-1, min(v, (1 << 31) - 1)) for v in self._whole(x, what)], dtype=torch.int32, device=self.device)

    @staticmethod
    def _whole(x, what: str) -> list:
        try:
            return [operator.index(v) for v in x]
        except TypeError:
            raise TypeError(f"{what}: whole numbers") from None

    def extend(self, more) -> None:
        """``more[b]`` new tokens for every row (whole numbers, an int32 tensor on the device or a list): their pages are
        taken from the free ones, lowest first, in the order of the rows, and ``counts``, ``new`` and ``starts``
        follow.  A row whose last page is partly filled and shared first gets a copy of it, in every cache; the
        last of the rows that write such a page keeps it.  A row whose pages are not to be had, or that would pass
        the capacity, gets none of its tokens and sets ``overflow`` (which stays until it is cleared): nothing of them is
        cached and their outputs are 0.  Pages are dealt out in the order of the rows: behind a row that did not
        find its pages none that needs one gets any, however few, nor does a row that was to keep a page which such a
        row still shares.  The others, and rows behind one that passes the capacity, get theirs."""
        c = self._struct()
        host = not isinstance(more, Tensor) or more.device.type == "cpu"
        tensor = self._rows_tensor(more, "more")
        if host:
            each = [max(v, 0) for v in (more.tolist() if isinstance(more, Tensor) else self._whole(more, "more"))]
            self._expected = (max(each), sum(each))
        else:
            self._expected = None
        c.more = tensor.data_ptr()
        _call(_lib.load().pa_page_extend, self.counts, "pa_page_extend", ctypes.byref(c))

    def select(self, index, lengths=None) -> None:
        """Row b becomes what row ``index[b]`` was, or its first ``lengths[b]`` positions, for all rows at once; -1 (or
        any number that is no row): an empty row.  Indexes may repeat (a fork), permute rows, and drop them.  Pages
        are shared, and free when the last row that has them lets go.  There is no chunk afterwards (``new`` 0)."""
        c = self._struct()
        index = self._rows_tensor(index, "index")
        c.index = index.data_ptr()
        if lengths is None:
            c.lengths = None
        else:
            lengths = self._rows_tensor(lengths, "lengths")
            c.lengths = lengths.data_ptr()
        self._expected = None
        _call(_lib.load().pa_page_select, self.counts, "pa_page_select", ctypes.byref(c))

    def fork(self, row: int, copies: Sequence[int]) -> None:
        """The rows ``copies`` become what ``row`` is (what they held is freed)."""
        self._check_rows((row, *copies))
        self.select([row if b in set(copies) else b for b in range(self.rows)])

    def free(self, rows: Sequence[int]) -> None:
        """The rows hold nothing any more."""
        self._check_rows(rows)
        gone = set(int(r) for r in rows)
        self.select([-1 if b in gone else b for b in range(self.rows)])

    def truncate(self, lengths) -> None:
        """Every row keeps its first ``lengths[b]`` positions (all of them where it has no more)."""
        self.select(list(range(self.rows)), lengths)

    def _check_rows(self, rows) -> None:
        _need(all(0 <= int(r) < self.rows for r in rows), f"rows: 0 to {self.rows - 1}")

    def compact(self) -> None:
        """The pages in use move to the front of the pool, in every cache: those behind the first ones go, in their
        order, to the free places among them."""
        c = self._struct()
        _call(_lib.load().pa_page_compact, self.counts, "pa_page_compact", ctypes.byref(c))

    def positions(self, tokens: int, packed: bool = False) -> Tensor:
        """Positions of a step's tokens, [rows, tokens] or packed [1, tokens] (for ``RotaryEmbedding(positions)`` as
        the layers' ``rotary_pos_emb``)."""
        first, i = self.counts - self.new, torch.arange(tokens, dtype=torch.int32, device=self.device)
        if not packed:
            return first[:, None] + i
        row = (torch.searchsorted(self.starts, i, right=True) - 1).clamp(0, self.rows - 1)
        return (first[row] + i - self.starts[row])[None]

    def lengths(self) -> list:
        """Positions held by each row (reads the device: synchronises)."""
        return self.counts.tolist()

    def free_pages(self) -> int:
        """Pages that no row has (reads the device: synchronises)."""
        return int((self.refs == 0).sum().item())

    def check_overflow(self) -> None:
        """Raise if a row did not get its pages (reads the device flag: synchronises)."""
        if int(self.overflow.item()):
            raise RuntimeError(f"PageTable overflow: tokens that found no page in the pool of {self.pool}, or no room in "
                               f"the capacity {self.capacity}, were dropped")


class PagedCache:
    """One layer's poly KV cache in the pages of ``table``.

    Level t of the attention, 0 the deepest, has ``keys[t]`` and ``values[t]`` [pool, kv_heads, page_size, dim_head] and,
    but for the last, ``lses[t]`` fp32 [pool, kv_heads, page_size].  It scores ``keys[t]`` with the next level's
    keys as queries (the last level's are q1), and leaves its result, times the next level's projected values
    where that is a middle one, in ``values[t + 1]``: one array per level, where the tuple caches hold the
    projected values and the results apart.  Written in place, always the same objects."""

    def __init__(self, table: PageTable, *, order: int, kv_heads: int, dim_head: int, dtype=torch.bfloat16):
        _need(2 <= order <= _lib.PA_MAX_ORDER, f"order {order}: 2 to {_lib.PA_MAX_ORDER}")
        _need(kv_heads >= 1, "kv_heads: at least 1")
        _need(dtype in DTYPE_CODE, f"{dtype}: float32, float16 or bfloat16", TypeError)
        _need(8 <= dim_head <= 256 and dim_head % (8 if dim_head <= 128 else 16) == 0,
              f"dim_head {dim_head}: a multiple of 8 up to 128, of 16 up to 256")
        self.table, self.order, self.kv_heads, self.dim_head, self.dtype = table, order, kv_heads, dim_head, dtype
        # a captured step would go on without it: a page of it that rows share would not be copied before one of them writes
        _need(not table._captured, "a call of the table was captured, and its graph copies the pages of the caches that the "
              "table had then: make the caches before, or take another table", RuntimeError)

        def rows(m):
            return tuple(torch.empty(table.pool, kv_heads, table.page_size, dim_head, dtype=dtype, device=table.device)
                         for _ in range(m))

        self.keys, self.values = rows(order), rows(order)
        self.lses = tuple(torch.empty(table.pool, kv_heads, table.page_size, dtype=torch.float32, device=table.device)
                          for _ in range(order - 1))
        # of attend, 0 between calls
        self._tickets = torch.zeros(_lib.PA_PAGED_TICKETS * _lib.PA_TICKET_STRIDE, dtype=torch.int32, device=table.device)
        self._plans: dict = {}
        self._captured = False
        table._add(self)

    def __getstate__(self):
        return {k: v for k, v in self.__dict__.items() if k not in ("_plans", "_captured")}

    def __setstate__(self, state) -> None:
        self.__dict__.update(state)
        self._plans = {}
        self._captured = False

    def __deepcopy__(self, memo):
        table = memo.get(id(self.table)) or self.table._copy(memo)
        other = memo[id(self)] = object.__new__(type(self))
        other.__setstate__({**copy.deepcopy({k: v for k, v in self.__getstate__().items() if k != "table"}, memo), "table": table})
        table._add(other)
        return other

    @property
    def device(self):
        return self.table.device

    def arrays(self) -> tuple:
        """All arrays of pages."""
        return (*self.keys, *self.values, *self.lses)

    # -------------------------------------------------------------------------------------

    def _hold(self) -> None:
        """A captured call has the cache's addresses: its tensors stay as long as the table."""
        self._captured = True
        self.table._kept += [*self.arrays(), self._tickets]

    def _keep(self, kind: str, shape, plan):
        if len(self._plans) >= _PLANS:
            del self._plans[next(iter(self._plans))]
        self._plans[kind, shape] = plan
        return plan

    def _check_rows(self, t: Tensor, what: str, shape: tuple) -> None:
        _need(t.shape == shape, f"{what}: {list(shape)}, not {list(t.shape)}")
        _need(t.dtype == self.dtype, f"{what}: {t.dtype}, the cache holds {self.dtype}", TypeError)
        _need(t.device == self.device, f"{what}: on another device than the cache")

    def _check_q1(self, q1: Tensor) -> None:
        t = self.table
        _need(self.device.type == "cuda", "a PagedCache step needs the GPU (libpolyattn)", RuntimeError)
        _need(q1.dim() == 4, "q1: [rows or 1, heads, tokens, dim_head]")
        B, H, T, d = q1.shape
        _need(B in (t.rows, 1), f"q1: {t.rows} rows, or 1 (packed), not {B}")
        _need(T >= 1, "a step takes at least one token")
        _need(H >= 1 and H % self.kv_heads == 0, f"{H} heads over {self.kv_heads} kv_heads")
        self._check_rows(q1, "q1", (B, H, T, self.dim_head))

    def _check_tokens(self, shape) -> None:
        known = self.table._expected
        if known is not None:
            packed = shape[0] != self.table.rows
            most = known[1] if packed else known[0]
            _need(most <= shape[2], f"{shape[2]} tokens: extend() was given {most}")

    def append(self, qs: Sequence[Tensor], v: Tensor, weights: Sequence[Optional[Tensor]], *, eps: float,
               angles: Optional[Tensor] = None, inv_freq: Optional[Tensor] = None, interp: float = 1.0) -> Tensor:
        """The query/key norms and the rotary embedding of the chunks' tokens, into the rows' pages.

        ``qs`` = (q1, ..., q_{order+1}) [rows, heads, T, d], or packed [1, heads, total, d], and ``v`` = the deepest
        level's values are a layer's projections seen per head (q1 of any number of heads that kv_heads divides,
        the others of kv_heads); ``weights`` the RMSNorm weights of ``qs`` (None: not normalised).  ``angles``: rotary
        angles [rows or 1, T, r], [T, r] or [r] of the tokens; or ``inv_freq`` (fp32 [r / 2]) a rotary module's
        frequencies at the tokens' positions, with its ``interp``olation factor.  The result is rounded once.
        Returns q1, 0 behind the chunks."""
        q1 = qs[0]
        order = self.order
        _need(len(qs) == order + 1 and len(weights) == len(qs), f"order {order}: {order + 1} qs and weights")
        _no_tangents(*qs, v, *weights, angles, inv_freq)
        plan = self._plans.get(("append", q1.shape))
        if plan is None:
            self._check_q1(q1)
            plan = self._keep("append", q1.shape, self._append_plan(q1))
        self._check_tokens(q1.shape)
        if not self._captured and torch._C._cuda_isCurrentStreamCapturing():
            self._hold()
        P, kv = plan
        B, H, T, d = q1.shape
        dtype, device, grad = self.dtype, self.device, torch.is_grad_enabled()
        index, unit = device.index, dtype.itemsize
        keep = []
        P.eps = eps
        self._set_angles(P, angles, inv_freq, interp, B, T, keep)
        shape, items = q1.shape, P.items
        for k, src in enumerate((*qs, v)):
            if src.shape != shape or src.dtype is not dtype or src.get_device() != index:
                self._check_rows(src, f"q{k + 1}" if k <= order else "v", shape)
            w = weights[k] if k <= order else None
            if grad and (src.requires_grad or (w is not None and w.requires_grad)):
                raise RuntimeError(_NO_GRAD)
            shape = kv
            s0, s1, s2, s3 = src.stride()
            ptr = src.data_ptr()
            if s3 != 1 or ((s0 | s1 | s2) * unit | ptr) & 15:
                src = _rows16(src)
                keep.append(src)
                s0, s1, s2, _ = src.stride()
                ptr = src.data_ptr()
            it = items[k]
            view = it.src
            view.ptr, view.sb, view.sh, view.sn = ptr, s0, s1, s2
            if w is None:
                it.norm_weight = None
                continue
            code = DTYPE_CODE.get(w.dtype)
            if code is None or w.shape != (d,) or w.get_device() != index:
                _need(False, f"norm weight {k}: [{d}] on the cache's device")
            if not w.is_contiguous():
                w = w.contiguous()
                keep.append(w)
            it.norm_weight, it.weight_dtype = w.data_ptr(), code
        out = torch.empty(B, H, T, d, dtype=dtype, device=device)
        P.items[0].out.ptr = out.data_ptr()
        _call(_lib.load().pa_page_append, out, "pa_page_append", ctypes.byref(P))
        return out

    def _append_plan(self, q1: Tensor):
        B, H, T, d = q1.shape
        P = _lib.PaPageRows()
        P.t = self.table._t
        P.tokens, P.packed, P.dim, P.count = T, int(B != self.table.rows), d, self.order + 2
        code = DTYPE_CODE[self.dtype]
        for k in range(self.order + 2):
            it = P.items[k]
            it.src.heads, it.src.dtype = H if k == 0 else self.kv_heads, code
            it.rotate = 1 if k <= self.order else 0
            if k:
                it.pages = (self.keys[self.order - k] if k <= self.order else self.values[0]).data_ptr()
        o = P.items[0].out
        o.heads, o.dtype, o.sb, o.sh, o.sn = H, code, H * T * d, T * d, d
        return P, (B, self.kv_heads, T, d)

    def _set_angles(self, P, angles, inv_freq, interp, B, T, keep) -> None:
        if angles is None and inv_freq is None:
            P.angles = P.inv_freq = None
            P.rot_dim = 0
            return
        _need(angles is None or inv_freq is None, "angles or inv_freq, not both")
        if angles is not None:
            _need(angles.dim() >= 1, "angles: at least one dimension")
            a, r = angles, angles.shape[-1]
            _need(a.device == self.device, "angles: on another device than the cache")
            _need(a.shape == (B, T, r) or a.shape == (T, r) or a.shape == (r,),
                  f"angles: [{B}, {T}, r], [{T}, r] or [r], not {list(a.shape)}")
            if a.dtype not in DTYPE_CODE or (a.stride(-1) != 1 and r > 1):
                a = a.detach().to(a.dtype if a.dtype in DTYPE_CODE else torch.float32).contiguous()
            P.inv_freq, P.angles, P.angles_dtype = None, a.data_ptr(), DTYPE_CODE[a.dtype]
            s = a.stride()
            P.angles_sb = s[0] if len(s) == 3 else 0
            P.angles_sn = s[-2] if len(s) >= 2 else 0
        else:
            _need(inv_freq.device == self.device and inv_freq.dim() == 1, "inv_freq: [r / 2] on the cache's device")
            _need(interp > 0, "interp: above 0")
            a = inv_freq.detach().to(torch.float32).contiguous()
            r = 2 * a.numel()
            P.angles, P.inv_freq, P.interp = None, a.data_ptr(), interp
        keep.append(a)
        _need(r % 2 == 0 and r <= self.dim_head, f"{r} angles: an even number up to dim_head = {self.dim_head}")
        P.rot_dim = r

    def attend(self, q1: Tensor, vs: Sequence[Tensor] = (), *, scale: Optional[float] = None,
               softclamp: Optional[float] = None) -> Tensor:
        """Every level of the poly attention for the chunks' tokens: each attends to its row's cached positions and to
        its chunk up to itself.  ``q1`` as ``append`` returns it; ``vs`` the projected values of the middle
        levels, (v3, ...) without the deepest (none at order 2), shaped as ``append``'s ``v``.  Writes
        ``values[1:]`` and ``lses`` of the tokens and returns the output, shaped as q1, 0 behind the chunks.
        ``scale`` defaults to dim_head ** -0.5.  May be repeated."""
        _no_tangents(q1, *vs)
        plan = self._plans.get(("attend", q1.shape))
        if plan is None:
            self._check_q1(q1)
            plan = self._keep("attend", q1.shape, self._attend_plan(q1))
        self._check_tokens(q1.shape)
        if not self._captured and torch._C._cuda_isCurrentStreamCapturing():
            self._hold()
        D, strides, kv = plan
        dtype, device = self.dtype, self.device
        if q1.dtype is not dtype or q1.device != device:
            self._check_q1(q1)
        if len(vs) != self.order - 2:
            _need(False, f"order {self.order}: {self.order - 2} vs")
        rows = _rows16(q1)
        grad = q1.requires_grad
        keep = []
        for k, v in enumerate(vs):
            if v.shape != kv or v.dtype is not dtype or v.device != device:
                self._check_rows(v, f"v{k + 3}", kv)
            grad = grad or v.requires_grad
            v = _rows16(v)
            keep.append(v)
            m = D.levels[self.order - 2 - k].vmul
            m.ptr = v.data_ptr()
            m.sb, m.sh, m.sn, _ = v.stride()
        if grad and torch.is_grad_enabled():
            raise RuntimeError(_NO_GRAD)
        # heads inner in memory: merging the heads afterwards is a view
        out = torch.empty_strided(q1.shape, strides, dtype=dtype, device=device)
        ws = torch.empty(D.workspace_bytes, dtype=torch.uint8, device=device)
        D.q.ptr = rows.data_ptr()
        D.q.sb, D.q.sh, D.q.sn, _ = rows.stride()
        D.out.ptr = out.data_ptr()
        D.scale = self.dim_head ** -0.5 if scale is None else scale
        D.softclamp = softclamp if softclamp else 0.0
        D.workspace = ws.data_ptr()
        _call(_lib.load().pa_paged_attend, out, "pa_paged_attend", ctypes.byref(D))
        return out

    def _attend_plan(self, q1: Tensor):
        B, H, T, d = q1.shape
        D = _lib.PaPaged()
        D.t = self.table._t
        code = DTYPE_CODE[self.dtype]
        D.tokens, D.packed, D.heads, D.kv_heads, D.dim = T, int(B != self.table.rows), H, self.kv_heads, d
        D.order, D.dtype = self.order, code
        for t in range(self.order):
            L = D.levels[t]
            L.keys, L.values = self.keys[t].data_ptr(), self.values[t].data_ptr()
            if t < self.order - 1:
                L.lses = self.lses[t].data_ptr()
            if 0 < t < self.order - 1:
                L.vmul.heads, L.vmul.dtype = self.kv_heads, code
        strides = (T * H * d, d, H * d, 1)
        for x in (D.q, D.out):
            x.heads, x.dtype = H, code
        D.out.sb, D.out.sh, D.out.sn, _ = strides
        D.tickets = self._tickets.data_ptr()
        D.workspace_bytes = _lib.load().pa_paged_attend_workspace(ctypes.byref(D))
        return D, strides, (B, self.kv_heads, T, d)
