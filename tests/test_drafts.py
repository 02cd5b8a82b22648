"""Drafted tokens on the CPU: trees, what the entry points refuse (before any launch), and the inputs of
the GPU suite's verification cases, whose decisions must be clear of their borders."""

import ctypes

import pytest
import torch

import drafts_oracle as DO
from poly_attention import DraftCache, NPolyAttention, PolyAttention, _lib, commit_drafts, verify_drafts
from poly_attention.drafts import draft_depths
from test_gpu_25_drafts import VERIFY_CASES, verify_inputs

param = pytest.mark.parametrize


def empty(**kw):
    args = dict(order=2, batch=2, kv_heads=2, dim_head=64, capacity=32, max_drafts=8,
                dtype=torch.float32, device="cpu")
    args.update(kw)
    return DraftCache.empty(**args)


def test_depths():
    p = torch.tensor([[-1, 0, 1, 1, 3], [-1, 0, -2, 2, 9], [-1, -1, 0, 4, 3]])
    # an absent node's depth counts from the node that is none
    assert draft_depths(p).tolist() == [[0, 1, 2, 2, 3], [0, 1, 0, 1, 0], [0, 0, 1, 0, 1]]
    chain = torch.arange(-1, 63)
    assert draft_depths(chain).tolist() == list(range(64))
    c = empty(batch=1, counts=torch.tensor([5], dtype=torch.int32))
    assert c.positions(3).tolist() == [[5, 6, 7]]
    assert c.positions(5, p[0]).tolist() == [[5, 6, 7, 7, 8]]


def test_oracle_tree():
    assert DO.walk_tree([-1, 0, 1, 0, 5, 4, -2, 6]) == [[0], [0, 1], [0, 1, 2], [0, 3], None, None, None, None]


def test_cache_of_tensors_with_a_gradient():
    """A prefill outside torch.no_grad(): the buffers hold values, no graph."""
    q, v = (torch.randn(1, 2, 3, 8, requires_grad=True) * 1 for _ in range(2))
    c = DraftCache((q, q, v, v[..., 0], v), 5)
    assert not any(t.requires_grad for t in (*c.qs, *c.vs, *c.msgs, *c.lses))
    assert torch.equal(c.qs[0][:, :, :3], q) and torch.equal(c.lses[0][:, :, :3], v[..., 0])


def test_cache_from_tuples():
    q2, q3, v3 = (torch.randn(2, 2, 5, 64) for _ in range(3))
    lse, msg = torch.randn(2, 2, 5), torch.randn(2, 2, 5, 64)
    rep = lambda t: t.repeat_interleave(3, dim=1)  # noqa: E731
    c = DraftCache((q2, q3, v3, rep(lse), rep(msg)), 16, max_drafts=4, lengths=[5, 2])
    assert c.order == 2 and c.lengths() == [5, 2] and c.prefix == 5
    for got, want in ((c.qs[0], q2), (c.qs[1], q3), (c.vs[0], v3), (c.lses[0], lse), (c.msgs[0], msg)):
        assert torch.equal(got[:, :, :5], want)
    n = DraftCache(((q2, q3, v3), (v3, q2), (lse, lse), (msg, msg)), 8, counts=c.counts)
    assert n.order == 3 and n.counts is c.counts


@param("kw,error", [
    (dict(order=1), ValueError), (dict(order=9), ValueError), (dict(max_drafts=0), ValueError),
    (dict(max_drafts=65), ValueError), (dict(dim_head=20), ValueError), (dict(dim_head=136), ValueError),
    (dict(dim_head=264), ValueError), (dict(dtype=torch.float64), TypeError), (dict(batch=0), ValueError),
    (dict(capacity=0), ValueError), (dict(counts=torch.zeros(3, dtype=torch.int32)), ValueError),
    (dict(counts=torch.zeros(2, dtype=torch.int64)), ValueError),
])
def test_cache_refusals(kw, error):
    with pytest.raises(error):
        empty(**kw)


def test_tuple_refusals():
    t = torch.zeros(2, 2, 5, 64)
    tup = (t, t, t, t[..., 0], t)
    for kw in (dict(capacity=4), dict(capacity=8, lengths=[6, 1]), dict(capacity=8, lengths=[-1, 1]),
               dict(capacity=8, lengths=[1]), dict(capacity=8, lengths=[1.0, 2.0]),
               dict(capacity=8, lengths=[1, 2], counts=torch.zeros(2, dtype=torch.int32))):
        with pytest.raises(ValueError):
            DraftCache(tup, **kw)


def test_calls_need_the_gpu():
    c = empty()
    q = torch.zeros(2, 2, 3, 64)
    with pytest.raises(RuntimeError):
        c.attend(q)
    with pytest.raises(RuntimeError):
        c.append([q] * 3, [q], [None] * 3, eps=1e-6)
    with pytest.raises(RuntimeError):
        commit_drafts([c], torch.zeros(2, 8, dtype=torch.int32), torch.zeros(2, dtype=torch.int32))
    with pytest.raises(RuntimeError):
        verify_drafts(torch.zeros(2, 3, 11), torch.zeros(2, 3, dtype=torch.int64))
    for m in (PolyAttention(dim=32, heads=2, use_flash_kernel=False),
              NPolyAttention(dim=32, order=3, heads=2, use_flash_kernel=False)):
        with pytest.raises(RuntimeError):
            m(torch.zeros(2, 3, 32), cache=c)
        with pytest.raises(AssertionError):
            m(torch.zeros(2, 3, 32), parents=torch.tensor([-1, 0, 1]))


# ---------------------------------------------------------------------------------------
# the C entry points: every refusal comes before a launch (the addresses are never read)

FAKE = 0x10000


def view(v, heads, dtype, sn=64, sh=4096, sb=65536):
    v.ptr, v.sb, v.sh, v.sn, v.heads, v.dtype = FAKE, sb, sh, sn, heads, dtype


def attend_args(order=3):
    P = _lib.PaDraft()
    P.batch, P.kv_heads, P.heads, P.drafts, P.dim, P.order, P.capacity = 2, 2, 4, 5, 64, order, 300
    P.scale, P.counts = 0.125, FAKE
    for t in range(order):
        L, last = P.levels[t], t == order - 1
        for v in (L.k, L.v, L.dk):
            view(v, 2, _lib.PA_BF16)
        if not last:
            view(L.dv, 2, _lib.PA_BF16)
            view(L.lse, 2, _lib.PA_F32, sn=1)
        if 0 < t < order - 1:
            view(L.vmul, 2, _lib.PA_BF16)
        if t:
            view(L.bias, 2, _lib.PA_F32, sn=1)
        for v in (L.q, L.out):
            view(v, 4 if last else 2, _lib.PA_BF16)
    P.workspace_bytes = _lib.load().pa_draft_attend_workspace(ctypes.byref(P))
    P.workspace = FAKE
    return P


def broken(fn, args, path, value):
    *head, name = path.split(".")
    at = args
    for part in head:
        at = at[int(part)] if part.isdigit() else getattr(at, part)
    setattr(at, name, value)
    return fn(ctypes.byref(args), None)


@param("path,value,want", [
    ("batch", 0, "EINVAL"), ("kv_heads", 0, "EINVAL"), ("heads", 3, "EINVAL"), ("drafts", 0, "EINVAL"),
    ("drafts", 65, "EINVAL"), ("order", 1, "EINVAL"), ("order", 9, "EINVAL"), ("capacity", 0, "EINVAL"), ("capacity", 2 ** 30 + 1, "EUNSUPPORTED"),
    ("counts", None, "EINVAL"), ("dim", 0, "EINVAL"), ("dim", 60, "EUNSUPPORTED"),
    ("dim", 264, "EUNSUPPORTED"), ("dim", 136, "EUNSUPPORTED"), ("workspace", None, "EWORKSPACE"),
    ("workspace", FAKE + 4, "EWORKSPACE"), ("workspace_bytes", 16, "EWORKSPACE"),
    ("levels.0.k.ptr", None, "EINVAL"), ("levels.0.k.heads", 4, "EINVAL"),
    ("levels.0.v.dtype", 0, "EINVAL"), ("levels.0.bias.ptr", FAKE, "EINVAL"),
    ("levels.0.lse.ptr", None, "EINVAL"), ("levels.0.lse.dtype", 2, "EINVAL"),
    ("levels.1.vmul.ptr", None, "EINVAL"), ("levels.1.bias.ptr", None, "EINVAL"),
    ("levels.1.dv.ptr", None, "EINVAL"), ("levels.2.dv.ptr", FAKE, "EINVAL"),
    ("levels.2.q.heads", 2, "EINVAL"), ("levels.2.out.dtype", 1, "EINVAL"),
    ("levels.0.k.sn", 65, "EUNSUPPORTED"), ("levels.0.k.ptr", FAKE + 2, "EUNSUPPORTED"),
    ("levels.2.q.sh", 4, "EUNSUPPORTED"), ("levels.1.bias.sn", 2, "EUNSUPPORTED"),
])
def test_attend_entry_refuses(path, value, want):
    lib = _lib.load()
    assert broken(lib.pa_draft_attend, attend_args(), path, value) == getattr(_lib, "PA_" + want)


def test_entries_refuse_null_and_sizes():
    lib = _lib.load()
    for fn in (lib.pa_draft_attend, lib.pa_draft_append, lib.pa_draft_verify, lib.pa_draft_commit):
        assert fn(None, None) == _lib.PA_EINVAL
    assert lib.pa_draft_attend_workspace(None) == 0 == lib.pa_draft_verify_workspace(None)
    P = attend_args()
    P.drafts = 0
    assert lib.pa_draft_attend_workspace(ctypes.byref(P)) == 0


def rows_args():
    R = _lib.PaDraftRows()
    R.batch, R.drafts, R.dim, R.count, R.eps = 2, 5, 64, 2, 1e-6
    R.counts = R.inv_freq = FAKE
    R.rot_dim, R.interp = 32, 1.0
    for it in list(R.items)[:2]:
        view(it.src, 4, _lib.PA_BF16)
        view(it.out, 4, _lib.PA_BF16)
    R.items[0].norm_weight, R.items[0].weight_dtype = FAKE, _lib.PA_F32
    return R


@param("path,value,want", [
    ("batch", 0, "EINVAL"), ("drafts", 0, "EINVAL"), ("drafts", 65, "EINVAL"), ("count", 0, "EINVAL"),
    ("count", 17, "EINVAL"), ("dim", 36, "EUNSUPPORTED"), ("rot_dim", 31, "EINVAL"),
    ("rot_dim", 66, "EINVAL"), ("interp", 0.0, "EINVAL"), ("counts", None, "EINVAL"),
    ("items.0.src.ptr", None, "EINVAL"), ("items.1.out.ptr", None, "EINVAL"),
    ("items.1.out.heads", 2, "EINVAL"), ("items.1.src.dtype", 0, "EINVAL"),
    ("items.0.weight_dtype", 7, "EINVAL"), ("items.0.src.sn", 63, "EUNSUPPORTED"),
    ("items.1.out.ptr", FAKE + 8, "EUNSUPPORTED"),
])
def test_append_entry_refuses(path, value, want):
    assert broken(_lib.load().pa_draft_append, rows_args(), path, value) == getattr(_lib, "PA_" + want)


def verify_args():
    V = _lib.PaVerify()
    V.batch, V.drafts, V.vocab, V.dtype = 2, 5, 100, _lib.PA_BF16
    for name in ("logits", "tokens", "uniforms", "noise", "path", "kept", "token", "workspace"):
        setattr(V, name, FAKE)
    V.workspace_bytes = _lib.load().pa_draft_verify_workspace(ctypes.byref(V))
    return V


@param("path,value,want", [
    ("batch", 0, "EINVAL"), ("batch", 70000, "EUNSUPPORTED"), ("drafts", 65, "EINVAL"), ("vocab", 0, "EINVAL"),
    ("vocab", (1 << 30) + 1, "EUNSUPPORTED"), ("dtype", 3, "EINVAL"), ("logits", None, "EINVAL"),
    ("logits", FAKE + 1, "EINVAL"), ("tokens", None, "EINVAL"), ("noise", None, "EINVAL"),
    ("path", None, "EINVAL"), ("kept", None, "EINVAL"), ("token", None, "EINVAL"),
    ("workspace", None, "EWORKSPACE"), ("workspace_bytes", 8, "EWORKSPACE"),
])
def test_verify_entry_refuses(path, value, want):
    assert broken(_lib.load().pa_draft_verify, verify_args(), path, value) == getattr(_lib, "PA_" + want)


def commit_args():
    C = _lib.PaCommit()
    C.batch, C.kv_heads, C.slots, C.capacity, C.count, C.advance, C.path_len = 2, 2, 8, 32, 1, 1, 8
    C.path = C.kept = C.counts = C.tickets = FAKE
    C.moves[0].src = C.moves[0].dst = FAKE
    C.moves[0].row_bytes = 128
    return C


@param("path,value", [
    ("batch", 0), ("kv_heads", 0), ("slots", 0), ("slots", 65), ("capacity", 0), ("count", 129), ("count", -1),
    ("path_len", 65), ("path", None), ("kept", None), ("counts", None), ("tickets", None), ("moves.0.src", None),
    ("moves.0.dst", None), ("moves.0.row_bytes", 0), ("moves.0.row_bytes", 6), ("moves.0.src", FAKE + 8),
])
def test_commit_entry_refuses(path, value):
    assert broken(_lib.load().pa_draft_commit, commit_args(), path, value) == _lib.PA_EINVAL


# ---------------------------------------------------------------------------------------


@param("case", VERIFY_CASES)
def test_verification_inputs_are_clear_of_borders(case):
    """The kernel's probabilities are sums of up to 10^5 fp32 exponentials of arguments below 64: 2^-18
    relative is more than ten times their error."""
    _, margin = DO.verify(*verify_inputs(case))
    assert margin > 2.0 ** -18
