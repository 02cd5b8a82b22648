"""Decoding with drafted tokens: a KV cache whose rows hold their own numbers of positions, one step
over several new tokens per row, the decision which of them stay, and the move behind the cached
positions.  No counterpart in the reference, whose cached step takes one token of one position for
the whole batch (poly_attention.py:283-287, n_poly_attention.py:196-207).

The T new tokens of a row (at most 64) are the nodes of a tree.  ``parents`` is an int32 tensor
[B, T], or [T] for one tree in all rows: the node that node t follows, lower than t, or -1 for a node
that follows the cached positions.  Any other value, or a parent that is absent itself, makes the node
absent: nothing attends to it and its outputs are 0.  None is a chain: each token follows the one
before.  Node 0 is usually the last token that was decided and is not cached yet, the others drafts
that follow it.  One step of a model::

    caches = [DraftCache(c, capacity, max_drafts=16, counts=counts) for c in layer_caches]
    logits = model(tokens, caches, parents)             # each layer: layer(x, cache=, parents=)
    path, kept, token = verify_drafts(logits, tokens, parents, uniforms=u, noise=e)
    commit_drafts(caches, path, kept)                    # token: node 0 of the next step

Every call works on the device counts alone, without a host synchronisation, so a step of fixed T can be
captured into a HIP graph.  The calls are for the GPU and for inference.
"""

from __future__ import annotations

import ctypes
import functools
import struct
from typing import Optional, Sequence

import torch
from torch import Tensor
from torch.autograd import forward_ad

from . import _lib
from ._lib import DTYPE_CODE, PA_MAX_DRAFTS, PA_MAX_MOVES


# the fields of a PaDraftItem that change from call to call
_PACK_SRC = struct.Struct("@Q3q").pack_into
_PACK_NORM = struct.Struct("@Qi").pack_into
_NORM_AT = _lib.PaDraftItem.norm_weight.offset
_NO_GRAD = "DraftCache steps are inference-only: run them under torch.no_grad()"


def _call(fn, t: Tensor, what: str, *args) -> None:
    """fn(*args, stream) on t's device and its current stream; raises on a failure status."""
    index = t.device.index
    if index == torch._C._cuda_getDevice():
        status = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            status = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if status:
        _lib.check(status, what)


def _need(ok: bool, what: str, error=ValueError) -> None:
    if not ok:
        raise error(what)


def _no_tangents(*tensors: Optional[Tensor]) -> None:
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None
                                              for t in tensors):
        raise RuntimeError(_NO_GRAD)


def _set_view(v, t: Tensor) -> None:
    v.ptr = t.data_ptr()
    s = t.stride()
    v.sb, v.sh, v.sn = s[0], s[1], s[2]
    v.heads = t.shape[1]
    v.dtype = DTYPE_CODE[t.dtype]


def _rows16(t: Tensor) -> Tensor:
    """``t`` [batch, heads, n, dim] with a unit feature stride and every row on 16 bytes, copied where it
    has not."""
    s0, s1, s2, s3 = t.stride()
    if s3 == 1 and not ((s0 | s1 | s2) * t.element_size() | t.data_ptr()) & 15:
        return t
    return t.new_empty(t.shape).copy_(t)  # contiguous() keeps the stride of a dimension of size 1, whatever it is


def _parents(parents: Optional[Tensor], batch: int, drafts: int, device) -> tuple:
    """(tensor to keep alive, address, elements between rows); a chain is (None, None, 0)."""
    if parents is None:
        return None, None, 0
    if (parents.dtype is torch.int32 and parents.device == device and parents.shape == (batch, drafts)
            and parents.stride(1) == 1):
        return parents, parents.data_ptr(), parents.stride(0)
    _need(parents.device == device, "parents: on another device than the cache")
    _need(parents.dtype in (torch.int64, torch.int32, torch.int16, torch.int8),
          f"parents: a signed integer tensor, not {parents.dtype}", TypeError)
    _need(parents.shape == (batch, drafts) or parents.shape == (drafts,),
          f"parents: [{batch}, {drafts}] or [{drafts}], not {list(parents.shape)}")
    if parents.dtype != torch.int32:
        parents = parents.clamp(-2, PA_MAX_DRAFTS).to(torch.int32)
    if parents.stride(-1) != 1 and drafts > 1:
        parents = parents.contiguous()
    return parents, parents.data_ptr(), parents.stride(0) if parents.dim() == 2 else 0


def draft_depths(parents: Tensor) -> Tensor:
    """Number of nodes between each node and the cached positions (0 for a node that follows them, and
    for an absent one whose parent is not a node), of parents [..., T]."""
    slot = torch.arange(parents.shape[-1], device=parents.device)
    inner = (parents >= 0) & (parents < slot)
    up = torch.where(inner, parents.long(), slot)
    depth = inner.to(torch.int32)
    for _ in range(6):  # up to 64 nodes: the distance covered doubles
        depth = depth + depth.gather(-1, up)
        up = up.gather(-1, up)
    return depth


class DraftCache:
    """A fixed-capacity poly KV cache with a position count per row, and slots for drafted tokens.

    ``cache``: a module's cache tuple (order 2 ``(q2, q3, v3, lse23, msg)``, order n ``(qs, vs,
    lses, msgs)``), whose positions are copied in.  ``lengths``: how many of them each row holds (a
    list or tensor [B]); a right-padded causal prefill leaves exactly those valid.  Default: all.
    ``counts``: an int32 device tensor [B] shared by the caches of one model's layers, which
    ``commit_drafts`` advances once for all of them; it then holds the rows' counts already and
    ``lengths`` is not given.

    The buffers are contiguous: ``qs`` (keys of every level), ``vs``, ``msgs`` [B, kv_heads, capacity,
    dim_head] and ``lses`` fp32 [B, kv_heads, capacity] -- one copy per key head, where the tuple cache
    repeats msg and lse for the query heads of a group, which are equal -- and ``draft_qs``,
    ``draft_vs``, ``draft_msgs``, ``draft_lses`` with ``max_drafts`` slots in place of the capacity.

    The buffers and ``counts`` are written in place and stay the same objects.  A cache takes one step at
    a time; caches of their own may be used at once, on any streams.  ``copy.deepcopy`` between two steps gives a
    cache of its own, to follow two continuations; caches that share a ``counts`` are copied together
    (``copy.deepcopy(caches)``), and their copies share one.

    A count reaches the capacity at most: tokens that do not fit are dropped by ``commit_drafts``, which
    sets the device flag ``overflow``; ``check_overflow()`` reads it.  Caches that are committed together
    share the flag of the first of them from then on.
    """

    def __init__(self, cache, capacity: int, *, max_drafts: int = 16, lengths=None,
                 counts: Optional[Tensor] = None):
        if isinstance(cache[0], Tensor):
            q2, q3, v3, lse, msg = cache
            qs, vs, lses, msgs = (q2, q3), (v3,), (lse,), (msg,)
        else:
            qs, vs, lses, msgs = cache
        B, hk, n, d = qs[0].shape
        _need(capacity >= n, f"capacity {capacity} below the {n} cached positions")
        _need(counts is None or lengths is None, "counts hold the rows' lengths: give one of the two")
        if counts is None:
            if lengths is None:
                counts = torch.full((B,), n, dtype=torch.int32, device=qs[0].device)
            else:
                lens = torch.as_tensor(lengths).reshape(-1)
                _need(lens.numel() == B and not lens.is_floating_point(),
                      f"lengths: {B} whole numbers")
                _need(bool(((lens >= 0) & (lens <= n)).all()), f"lengths: 0 to {n}")
                counts = lens.to(device=qs[0].device, dtype=torch.int32)
        self._allocate(len(qs), B, hk, d, capacity, max_drafts, qs[0].dtype, qs[0].device, counts)
        self.prefix = n
        for to, src in zip((*self.qs, *self.vs, *self.msgs, *self.lses), (*qs, *vs, *msgs, *lses)):
            rep = src.shape[1] // hk  # query heads of a group hold equal rows
            to.narrow(2, 0, n).copy_(src.detach()[:, ::rep])

    @classmethod
    def empty(cls, *, order: int, batch: int, kv_heads: int, dim_head: int, capacity: int,
              max_drafts: int = 16, dtype=torch.bfloat16, device="cuda",
              counts: Optional[Tensor] = None) -> "DraftCache":
        """A cache without positions (counts 0, or the given counts over buffers to be filled)."""
        self = cls.__new__(cls)
        device = torch.device(device)
        if counts is None:
            counts = torch.zeros(batch, dtype=torch.int32, device=device)
        self._allocate(order, batch, kv_heads, dim_head, capacity, max_drafts, dtype, counts.device
                       if device.type == counts.device.type and device.index is None else device,
                       counts)
        self.prefix = 0
        return self

    def _allocate(self, order, batch, kv_heads, dim_head, capacity, max_drafts, dtype, device, counts):
        _need(2 <= order <= _lib.PA_MAX_ORDER, f"order {order}: 2 to {_lib.PA_MAX_ORDER}")
        _need(batch >= 1 and kv_heads >= 1 and capacity >= 1, "batch, kv_heads, capacity: at least 1")
        _need(1 <= max_drafts <= PA_MAX_DRAFTS, f"max_drafts {max_drafts}: 1 to {PA_MAX_DRAFTS}")
        _need(dtype in DTYPE_CODE, f"{dtype}: float32, float16 or bfloat16", TypeError)
        _need(8 <= dim_head <= 256 and dim_head % (8 if dim_head <= 128 else 16) == 0,
              f"dim_head {dim_head}: a multiple of 8 up to 128, of 16 up to 256")
        _need(counts.dtype == torch.int32 and counts.shape == (batch,) and counts.is_contiguous()
              and counts.device == device,
              f"counts: a contiguous int32 tensor [{batch}] on the cache's device")
        self.order, self.batch, self.kv_heads, self.dim_head = order, batch, kv_heads, dim_head
        self.capacity, self.max_drafts, self.dtype, self.device = capacity, max_drafts, dtype, device
        self.counts = counts
        self.keys_rotated = False

        def rows(n, m):
            return tuple(torch.empty(batch, kv_heads, n, dim_head, dtype=dtype, device=device)
                         for _ in range(m))

        def sums(n):
            return tuple(torch.empty(batch, kv_heads, n, dtype=torch.float32, device=device)
                         for _ in range(order - 1))

        m = order - 1
        self.qs, self.vs, self.msgs, self.lses = (rows(capacity, order), rows(capacity, m),
                                                  rows(capacity, m), sums(capacity))
        self.draft_qs, self.draft_vs = rows(max_drafts, order), rows(max_drafts, m)
        self.draft_msgs, self.draft_lses = rows(max_drafts, m), sums(max_drafts)
        self._geometry = (batch, kv_heads, max_drafts, capacity)
        # rows' tickets of a commit, 0 between calls, and the flag of tokens past the capacity
        zeros = torch.zeros((batch + 1) * _lib.PA_TICKET_STRIDE, dtype=torch.int32, device=device)
        self._tickets, self.overflow = zeros[_lib.PA_TICKET_STRIDE:], zeros[:1]
        self._earlier = ()  # flags of commits with another first cache
        self._lay_out()

    def _lay_out(self) -> None:
        """What holds addresses of the buffers, which stay where they are: a commit's moves, and the other calls'
        structures."""
        row = self.dtype.itemsize * self.dim_head
        pairs = zip((*self.draft_qs, *self.draft_vs, *self.draft_msgs, *self.draft_lses),
                    (*self.qs, *self.vs, *self.msgs, *self.lses))
        self._moves = b"".join([_lib.PACK_MOVE.pack(src.data_ptr(), dst.data_ptr(), row if src.dim() == 4 else 4, 0)
                                for src, dst in pairs])
        self._plans = {}  # by the shape of q1

    def __getstate__(self):
        return {k: v for k, v in self.__dict__.items() if k not in ("_moves", "_plans")}

    def __setstate__(self, state) -> None:
        self.__dict__.update(state)
        self.device = self.counts.device  # a load may have moved the buffers
        self._lay_out()

    # -------------------------------------------------------------------------------------

    def _check_gpu(self) -> None:
        _need(self.device.type == "cuda", "a DraftCache step needs the GPU (libpolyattn)", RuntimeError)

    def _check_rows(self, t: Tensor, what: str, drafts: int, heads: int) -> None:
        _need(t.dim() == 4 and t.shape == (self.batch, heads, drafts, self.dim_head),
              f"{what}: [{self.batch}, {heads}, {drafts}, {self.dim_head}], not {list(t.shape)}")
        _need(t.dtype == self.dtype, f"{what}: {t.dtype}, the cache holds {self.dtype}", TypeError)
        _need(t.device == self.device, f"{what}: on another device than the cache")

    def _plan(self, kind: str, q1: Tensor):
        """The call's structure for q1's shape, whose constant fields are set once."""
        self._check_gpu()
        _need(q1.dim() == 4, "q1: [batch, heads, drafts, dim_head]")
        T, H = q1.shape[2], q1.shape[1]
        _need(1 <= T <= self.max_drafts, f"{T} tokens: 1 to max_drafts = {self.max_drafts}")
        _need(H >= 1 and H % self.kv_heads == 0, f"{H} heads over {self.kv_heads} kv_heads")
        self._check_rows(q1, "q1", T, H)
        plan = self._append_plan(T, H) if kind == "append" else self._attend_plan(T, H)
        self._plans[kind, q1.shape] = plan
        return plan

    def positions(self, drafts: int, parents: Optional[Tensor] = None) -> Tensor:
        """Positions [B, drafts] of a step's nodes: the row's count plus the node's depth (for
        ``RotaryEmbedding(positions)`` as the layers' ``rotary_pos_emb``)."""
        if parents is None:
            depth = torch.arange(drafts, dtype=torch.int32, device=self.device)
        else:
            _need(parents.shape in ((self.batch, drafts), (drafts,)),
                  f"parents: [{self.batch}, {drafts}] or [{drafts}], not {list(parents.shape)}")
            depth = draft_depths(parents)
        return self.counts[:, None] + depth

    def append(self, qs: Sequence[Tensor], vs: Sequence[Tensor], weights: Sequence[Optional[Tensor]],
               *, eps: float, parents: Optional[Tensor] = None, angles: Optional[Tensor] = None,
               inv_freq: Optional[Tensor] = None, interp: float = 1.0) -> Tensor:
        """The query/key norms and the rotary embedding of a step's tokens, into their draft slots.

        ``qs`` = (q1, ..., q_{order+1}) [B, heads, T, d] and ``vs`` = (v3, ...) are a layer's
        projections seen per head (q1 of any number of heads that kv_heads divides, the others of
        kv_heads); ``weights`` the RMSNorm weights of ``qs`` (None: that tensor is not normalised).
        ``angles``: rotary angles [B, T, r], [T, r] or [r] of the tokens; or ``inv_freq`` (fp32 [r / 2])
        a rotary module's frequencies at the nodes' positions, with its ``interp``olation factor.
        The result is rounded once.  Returns q1 [B, heads, T, d]; the others go to ``draft_qs`` and
        ``draft_vs``."""
        q1 = qs[0]
        _need(len(qs) == self.order + 1 and len(vs) == self.order - 1 and len(weights) == len(qs),
              f"order {self.order}: {self.order + 1} qs and weights, {self.order - 1} vs")
        _no_tangents(*qs, *vs, *weights, angles, inv_freq)
        plan = self._plans.get(("append", q1.shape)) or self._plan("append", q1)
        B, H, T, d = q1.shape
        dtype, device, grad = self.dtype, self.device, torch.is_grad_enabled()
        P, buf, offsets = plan
        keep = [qs, vs, weights]
        P.eps = eps
        parents, P.parents, P.parents_stride = _parents(parents, B, T, device)
        self._set_angles(P, angles, inv_freq, interp, T, keep)
        es, index, shape, kv, order = dtype.itemsize, device.index, q1.shape, self._kv_shape(T), self.order
        for k, off in enumerate(offsets):
            src = qs[k] if k <= order else vs[k - order - 1]
            if src.shape != shape or src.dtype is not dtype or src.device != device:
                self._check_rows(src, f"q{k + 1}" if k <= order else f"v{k - order + 2}", T, shape[1])
            if grad and src.requires_grad:
                raise RuntimeError(_NO_GRAD)
            shape = kv
            ptr = src.data_ptr()
            s0, s1, s2, s3 = src.stride()
            if s3 != 1 or ((s0 | s1 | s2) * es | ptr) & 15:
                src = _rows16(src)
                keep.append(src)
                ptr = src.data_ptr()
                s0, s1, s2, s3 = src.stride()
            _PACK_SRC(buf, off, ptr, s0, s1, s2)
            if k <= order:
                w = weights[k]
                if w is None:
                    _PACK_NORM(buf, off + _NORM_AT, 0, 0)
                    continue
                code = DTYPE_CODE.get(w.dtype)
                if code is None or w.dim() != 1 or w.numel() != d or w.device != device:
                    _need(False, f"norm weight {k}: [{d}] on the cache's device")
                if grad and w.requires_grad:
                    raise RuntimeError(_NO_GRAD)
                if w.stride(0) != 1:
                    w = w.contiguous()
                    keep.append(w)
                _PACK_NORM(buf, off + _NORM_AT, w.data_ptr(), code)
        out = torch.empty(B, H, T, d, dtype=dtype, device=device)
        P.items[0].out.ptr = out.data_ptr()
        _call(_lib.load().pa_draft_append, out, "pa_draft_append", ctypes.byref(P))
        return out

    def _append_plan(self, T: int, H: int):
        P = _lib.PaDraftRows()
        P.batch, P.drafts, P.dim, P.count = self.batch, T, self.dim_head, 2 * self.order
        P.counts = self.counts.data_ptr()
        for k, (it, out) in enumerate(zip(P.items, (None, *self.draft_qs, *self.draft_vs))):
            it.src.heads = it.out.heads = H if k == 0 else self.kv_heads
            it.src.dtype = it.out.dtype = DTYPE_CODE[self.dtype]
            it.rotate = 1 if k <= self.order else 0
            if k:
                _set_view(it.out, out)
            else:
                it.out.sb, it.out.sh, it.out.sn = H * T * self.dim_head, T * self.dim_head, self.dim_head
        step, base = ctypes.sizeof(_lib.PaDraftItem), _lib.PaDraftRows.items.offset
        return P, memoryview(P).cast("B"), [base + k * step for k in range(2 * self.order)]

    def _kv_shape(self, T: int) -> tuple:
        return (self.batch, self.kv_heads, T, self.dim_head)

    def _set_angles(self, P, angles, inv_freq, interp, T, keep) -> None:
        if angles is None and inv_freq is None:
            P.angles = P.inv_freq = None
            P.rot_dim = 0
            return
        _need(angles is None or inv_freq is None, "angles or inv_freq, not both")
        if angles is not None:
            _need(angles.dim() >= 1, "angles: at least one dimension")
            a, r = angles, angles.shape[-1]
            _need(a.device == self.device, "angles: on another device than the cache")
            _need(a.shape == (self.batch, T, r) or a.shape == (T, r) or a.shape == (r,),
                  f"angles: [{self.batch}, {T}, r], [{T}, r] or [r], not {list(a.shape)}")
            if a.dtype not in DTYPE_CODE or (a.stride(-1) != 1 and r > 1):
                a = a.detach().to(a.dtype if a.dtype in DTYPE_CODE else torch.float32).contiguous()
            P.inv_freq, P.angles, P.angles_dtype = None, a.data_ptr(), DTYPE_CODE[a.dtype]
            s = a.stride()
            P.angles_sb = s[0] if len(s) == 3 else 0
            P.angles_sn = s[-2] if len(s) >= 2 else 0
        else:
            _need(inv_freq.device == self.device and inv_freq.dim() == 1,
                  "inv_freq: [r / 2] on the cache's device")
            _need(interp > 0, "interp: above 0")
            a = inv_freq.detach().to(torch.float32).contiguous()
            r = 2 * a.numel()
            P.angles, P.inv_freq, P.interp = None, a.data_ptr(), interp
        keep.append(a)
        _need(r % 2 == 0 and r <= self.dim_head,
              f"{r} angles: an even number up to dim_head = {self.dim_head}")
        P.rot_dim = r

    def attend(self, q1: Tensor, *, parents: Optional[Tensor] = None, scale: Optional[float] = None,
               softclamp: Optional[float] = None) -> Tensor:
        """Every level of the poly attention for a step's nodes: each attends to its row's cached
        positions, to its ancestors and to itself.  ``q1`` [B, heads, T, d] as ``append`` returns it;
        the other levels' queries, keys and values are in the draft slots.  Writes ``draft_msgs`` and
        ``draft_lses`` and returns the output [B, heads, T, d].  ``scale`` defaults to
        dim_head ** -0.5."""
        _no_tangents(q1)
        plan = self._plans.get(("attend", q1.shape)) or self._plan("attend", q1)
        B, H, T, d = q1.shape
        dtype, device = self.dtype, self.device
        if q1.dtype is not dtype or q1.device != device:
            self._check_rows(q1, "q1", T, H)
        if q1.requires_grad and torch.is_grad_enabled():
            raise RuntimeError(_NO_GRAD)
        D, q, y, size, strides = plan
        rows = _rows16(q1)
        # heads inner in memory: merging the heads afterwards is a view
        out = torch.empty_strided((B, H, T, d), strides, dtype=dtype, device=device)
        ws = torch.empty(size, dtype=torch.uint8, device=device)
        parents, D.parents, D.parents_stride = _parents(parents, B, T, device)
        q.ptr = rows.data_ptr()
        q.sb, q.sh, q.sn, _ = rows.stride()
        y.ptr = out.data_ptr()
        D.scale = d ** -0.5 if scale is None else scale
        D.softclamp = softclamp if softclamp else 0.0
        D.workspace = ws.data_ptr()
        _call(_lib.load().pa_draft_attend, out, "pa_draft_attend", ctypes.byref(D))
        return out

    def _attend_plan(self, T: int, H: int):
        D = _lib.PaDraft()
        D.batch, D.kv_heads, D.heads, D.drafts = self.batch, self.kv_heads, H, T
        D.dim, D.order, D.capacity = self.dim_head, self.order, self.capacity
        D.counts = self.counts.data_ptr()
        cut = lambda t: t.narrow(2, 0, T)  # noqa: E731
        for t in range(self.order):  # deepest level first; chain level lvl scores q_{lvl+1} . q_{lvl+2}
            lvl = self.order - 1 - t
            L = D.levels[t]
            _set_view(L.k, self.qs[lvl])
            _set_view(L.dk, cut(self.draft_qs[lvl]))
            if t == 0:
                _set_view(L.v, self.vs[-1])
                _set_view(L.dv, cut(self.draft_vs[-1]))
            else:
                _set_view(L.bias, self.lses[t - 1])
                if lvl:
                    _set_view(L.v, self.vs[lvl - 1])
                    _set_view(L.dv, cut(self.draft_vs[lvl - 1]))
                    _set_view(L.vmul, self.msgs[t - 1])
                else:
                    _set_view(L.v, self.msgs[t - 1])
            if lvl:
                _set_view(L.q, cut(self.draft_qs[lvl - 1]))
                _set_view(L.out, cut(self.draft_msgs[t]))
                _set_view(L.lse, cut(self.draft_lses[t]))
        D.workspace_bytes = _lib.load().pa_draft_attend_workspace(ctypes.byref(D))
        _need(D.workspace_bytes > 0, f"{self.batch} rows, {H} heads, {T} tokens over {self.kv_heads} kv_heads: too many",
              NotImplementedError)
        last = D.levels[self.order - 1]
        strides = (T * H * self.dim_head, self.dim_head, H * self.dim_head, 1)
        for v in (last.q, last.out):
            v.heads, v.dtype = H, DTYPE_CODE[self.dtype]
        last.out.sb, last.out.sh, last.out.sn, _ = strides
        return D, last.q, last.out, D.workspace_bytes, strides

    def rotate_prefix(self, rotary) -> None:
        """Rotate the keys copied from a module's tuple cache in place, as the module's rotary rotates
        cached keys, once (a tuple cache of a module with its own rotary holds them unrotated)."""
        if self.keys_rotated:
            return
        if self.prefix:
            if self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("DraftCache with the module's own rotary: run one eager step before "
                                   "capturing steps (the cached prefix is rotated once, in place)")
            for q in self.qs:
                head = q.narrow(2, 0, self.prefix)
                head.copy_(rotary.rotate_queries_or_keys(head).detach())
        self.keys_rotated = True

    def check_overflow(self) -> None:
        """Raise if a commit ran past the capacity (reads the device flag: synchronises)."""
        if any(int(flag.item()) for flag in (self.overflow, *self._earlier)):
            raise RuntimeError(f"DraftCache overflow: tokens past the capacity {self.capacity} were "
                               "dropped")

    def lengths(self) -> list:
        """Positions held by each row (reads the device counts: synchronises)."""
        return [min(max(int(n), 0), self.capacity) for n in self.counts.tolist()]


def commit_drafts(caches: Sequence[DraftCache], path: Tensor, kept: Tensor) -> None:
    """Keep the nodes path[b, :kept[b]] of every row: their keys, values, level outputs and logsumexps move
    from the draft slots of every layer's cache behind the row's cached positions, and the counts
    advance.  ``caches`` are the layers of one model and share one ``counts`` tensor; ``path`` int32
    [B, n] and ``kept`` int32 [B] as ``verify_drafts`` returns them (a path ends early at an entry that is no
    slot; kept 0 leaves a row as it is).  Tokens past the capacity are dropped and flagged
    (``overflow``)."""
    _need(len(caches) > 0, "a commit needs at least one cache")
    c0 = caches[0]
    counts, geometry, device, flag = c0.counts, c0._geometry, c0.device, c0.overflow
    for c in caches:
        if c.counts is not counts or c._geometry != geometry:
            _need(c.counts is counts, "caches of one commit share one counts tensor")
            _need(False, "caches of one commit have the same batch, kv_heads, capacity and max_drafts")
    B, hk, slots, capacity = geometry
    if not (path.dtype is torch.int32 and kept.dtype is torch.int32 and path.device == device == kept.device
            and path.dim() == 2 and path.shape[0] == B and 1 <= path.shape[1] <= PA_MAX_DRAFTS
            and kept.shape == (B,) and path.stride(1) == 1 and kept.is_contiguous() and device.type == "cuda"):
        c0._check_gpu()
        for t, what in ((path, "path"), (kept, "kept")):
            _need(t.dtype == torch.int32, f"{what}: int32, not {t.dtype}", TypeError)
            _need(t.device == device, f"{what}: on another device than the caches")
        _need(path.dim() == 2 and path.shape[0] == B and 1 <= path.shape[1] <= PA_MAX_DRAFTS,
              f"path: [{B}, 1 to {PA_MAX_DRAFTS}], not {list(path.shape)}")
        _need(kept.shape == (B,), f"kept: [{B}], not {list(kept.shape)}")
        path, kept = path.contiguous(), kept.contiguous()
    for c in caches:  # all of them lose what does not fit
        if c.overflow is not flag:
            c._earlier, c.overflow = (*c._earlier, c.overflow), flag
    moves = c0._moves if len(caches) == 1 else b"".join([c._moves for c in caches])
    size = PA_MAX_MOVES * ctypes.sizeof(_lib.PaDraftMove)
    fn = _lib.load().pa_draft_commit
    for k in range(0, len(moves), size):
        part = moves if len(moves) <= size else moves[k:k + size]
        head = _lib.PACK_COMMIT.pack(
            B, hk, slots, capacity, len(part) // ctypes.sizeof(_lib.PaDraftMove), k + size >= len(moves),
            path.data_ptr(), path.stride(0), path.shape[1], kept.data_ptr(), counts.data_ptr(),
            flag.data_ptr(), c0._tickets.data_ptr())
        _call(fn, kept, "pa_draft_commit", head + part)


def verify_drafts(logits: Tensor, tokens: Tensor, parents: Optional[Tensor] = None, *,
                  uniforms: Optional[Tensor] = None, noise: Optional[Tensor] = None,
                  temperature: Optional[Tensor] = None, draft_probs: Optional[Tensor] = None):
    """Which drafted tokens stay, and the token that follows them.

    ``logits`` [B, T, V]: the target model's prediction behind every node; ``tokens`` int64 [B, T]: the
    nodes' tokens; p = softmax(logits / temperature) (``temperature`` fp32 [B], default 1; a row whose
    temperature is 0 puts all of p on the first of its largest logits).  From node 0, which is kept,
    the walk takes the nodes in order: a child of the current node with token x is kept, and becomes
    the current node, if uniforms[b, t] * q(x) < p(x); otherwise p becomes what is left of it:

    * with ``draft_probs`` fp32 [B, T, V] -- [b, t] the distribution that the children of node t were
      drawn from, independently: p = max(p - q, 0), normalised;
    * without (children chosen, not drawn): q(x) = 1, p without x, normalised.

    The next token is the i with the largest p_i / noise[b, i], the lowest of equals.  With ``uniforms``
    fp32 [B, T] uniform in [0, 1) and ``noise`` fp32 [B, V] drawn from Exp(1) the kept tokens and the
    next one are distributed as the target's own.  Without ``uniforms`` and ``noise`` every row is greedy.

    Returns path int32 [B, T] (the kept nodes, then -1), kept int32 [B] and token int64 [B].  A row whose
    node 0 is absent keeps nothing and gets token -1; so does, with its path kept, a row whose last p
    has no positive entry (logits that are NaN or all -inf).  A token outside the vocabulary is never
    kept."""
    _need(logits.is_cuda, "verify_drafts needs the GPU (libpolyattn)", RuntimeError)
    _need(logits.dim() == 3 and logits.dtype in DTYPE_CODE,
          "logits: [batch, drafts, vocabulary] in float32, float16 or bfloat16")
    B, T, V = logits.shape
    dev = logits.device
    _need(B >= 1 and 1 <= T <= PA_MAX_DRAFTS and V >= 1,
          f"logits {list(logits.shape)}: 1 to {PA_MAX_DRAFTS} drafts, a vocabulary")
    _need((uniforms is None) == (noise is None), "uniforms and noise go together")
    _need(uniforms is not None or (temperature is None and draft_probs is None),
          "temperature and draft_probs need uniforms and noise")
    if logits.stride(2) != 1 and V > 1:
        logits = logits.contiguous()
    keep = [logits]

    parents, par_ptr, par_stride = _parents(parents, B, T, dev)
    bt = (B, T)
    path = torch.empty(B, T, dtype=torch.int32, device=dev)
    kept = torch.empty(B, dtype=torch.int32, device=dev)
    token = torch.empty(B, dtype=torch.int64, device=dev)
    size = _verify_workspace(B, T, V)
    ws = torch.empty(size, dtype=torch.uint8, device=dev)
    sb, sn, _ = logits.stride()
    packed = _lib.PACK_VERIFY.pack(
        B, T, V, DTYPE_CODE[logits.dtype], logits.data_ptr(), sb, sn,
        *_fixed(tokens, "tokens", bt, torch.int64, dev, keep), par_ptr or 0, par_stride,
        *_fixed(uniforms, "uniforms", bt, torch.float32, dev, keep),
        *_fixed(noise, "noise", (B, V), torch.float32, dev, keep),
        *_fixed(temperature, "temperature", (B,), torch.float32, dev, keep),
        *_fixed(draft_probs, "draft_probs", (B, T, V), torch.float32, dev, keep),
        path.data_ptr(), kept.data_ptr(), token.data_ptr(), ws.data_ptr(), size)
    _call(_lib.load().pa_draft_verify, logits, "pa_draft_verify", packed)
    return path, kept, token


def _fixed(t: Optional[Tensor], what: str, shape: tuple, dtype, dev, keep: list) -> tuple:
    """Address and leading strides of an optional tensor that has to be of this shape and type."""
    if t is None:
        return _NOTHING[len(shape)]
    if t.dtype is not dtype or t.shape != shape or t.device != dev:
        _need(t.dtype == dtype, f"{what}: {dtype}, not {t.dtype}", TypeError)
        _need(t.shape == shape, f"{what}: {list(shape)}, not {list(t.shape)}")
        _need(False, f"{what}: on another device than logits")
    strides = t.stride()
    if strides[-1] != 1 and shape[-1] > 1:
        t = t.contiguous()
        keep.append(t)
        strides = t.stride()
    return (t.data_ptr(), *strides[:-1])


_NOTHING = tuple((0,) * n for n in range(4))


@functools.lru_cache(maxsize=256)
def _verify_workspace(B: int, T: int, V: int) -> int:
    P = _lib.PaVerify()
    P.batch, P.drafts, P.vocab = B, T, V
    size = _lib.load().pa_draft_verify_workspace(ctypes.byref(P))
    _need(size > 0, f"logits [{B}, {T}, {V}]: at most 65535 rows and 2^30 tokens", NotImplementedError)
    return size
