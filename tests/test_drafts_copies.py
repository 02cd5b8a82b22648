"""DraftCache as an object, on the CPU: a copy's calls go to the copy's buffers."""

import copy
import io

import pytest
import torch

from poly_attention import DraftCache, _lib
from test_drafts import empty

param = pytest.mark.parametrize


def addresses(c):
    """(source, destination) of every move that a commit of this cache makes."""
    size = _lib.PACK_MOVE.size
    return [_lib.PACK_MOVE.unpack(c._moves[k:k + size])[:2] for k in range(0, len(c._moves), size)]


def own_addresses(c):
    return [(s.data_ptr(), t.data_ptr()) for s, t in zip((*c.draft_qs, *c.draft_vs, *c.draft_msgs, *c.draft_lses),
                                                        (*c.qs, *c.vs, *c.msgs, *c.lses))]


def pickled(x):
    file = io.BytesIO()
    torch.save(x, file)
    file.seek(0)
    return torch.load(file, weights_only=False)


@param("how", (copy.deepcopy, pickled))
@param("order", (2, 4))
def test_a_copy_commits_into_its_own_buffers(how, order):
    c = empty(order=order)
    c.qs[0].normal_()
    c.counts[1] = 3
    c._plans["attend", (1,)] = _lib.PaDraft()  # as after a step: its structures hold addresses and cannot be copied
    other = how(c)
    assert addresses(c) == own_addresses(c)
    assert addresses(other) == own_addresses(other)
    assert not set(sum(addresses(other), ())) & set(sum(addresses(c), ()))
    assert other._plans == {} and len(c._plans) == 1
    assert torch.equal(other.qs[0], c.qs[0]) and other.lengths() == [0, 3]
    other.counts += 1
    assert c.lengths() == [0, 3] and other.capacity == c.capacity and other._geometry == c._geometry


@param("how", (copy.deepcopy, pickled))
def test_copies_of_a_models_caches_share_a_count(how):
    a = empty()
    b = empty(counts=a.counts)
    c, d = how([a, b])
    assert c.counts is d.counts and c.counts is not a.counts
    assert c._tickets.data_ptr() not in (a._tickets.data_ptr(), d._tickets.data_ptr())


@param("shape,strides,offset", [
    ((1, 2, 1, 8), (5, 8, 3, 1), 0),    # dimensions of size 1 have any stride and count as contiguous
    ((2, 1, 1, 8), (8, 7, 9, 1), 0),
    ((2, 3, 4, 8), (96, 32, 8, 1), 3),  # rows not on 16 bytes
    ((2, 3, 4, 8), (8, 16, 48, 2), 0),
    ((2, 3, 4, 8), (0, 0, 9, 1), 0),
])
def test_rows_are_copied_where_they_do_not_start_on_16_bytes(shape, strides, offset):
    from poly_attention.drafts import _rows16

    t = torch.arange(400, dtype=torch.bfloat16).as_strided(shape, strides, offset)
    r = _rows16(t)
    assert torch.equal(r, t) and r.stride(3) == 1 and r.data_ptr() % 16 == 0
    assert all(s * 2 % 16 == 0 for s in r.stride()[:3])
    assert _rows16(r) is r


def test_forward_mode_tangents_are_refused():
    """A step has no derivative, forward or backward: a dual tensor raises as one that requires a gradient does."""
    from torch.autograd import forward_ad

    c = empty()
    row = lambda: torch.zeros(2, 2, 3, 64)  # noqa: E731
    w = [torch.ones(64) for _ in range(3)]
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(row(), row())
        with pytest.raises(RuntimeError, match="inference-only"):
            c.attend(dual)
        for qs, vs, ws in (([row(), dual, row()], [row()], w), ([row()] * 3, [dual], w),
                           ([row()] * 3, [row()], [None, forward_ad.make_dual(w[0], w[1]), None])):
            with pytest.raises(RuntimeError, match="inference-only"):
                c.append(qs, vs, ws, eps=1e-6)
        with pytest.raises(RuntimeError, match="GPU"):  # no tangent: the check behind it
            c.attend(row())
