"""The C entry points of a drafted step at their limits, on the CPU: every refusal comes before a launch."""

import ctypes

import pytest

from poly_attention import _lib
from test_drafts import attend_args, commit_args, rows_args

param = pytest.mark.parametrize
MOST = (1 << 24) - 1  # workgroups of 256 threads in a grid's first dimension


@param("batch,kv_heads", [(MOST + 1, 1), (1 << 23, 2), (MOST, 1), (MOST // 2 + 1, 1)])
def test_attend_refuses_more_rows_than_a_grid_holds(batch, kv_heads):
    """The rows' own workgroups and those of the cached positions, or the join's, pass the limit."""
    lib, P = _lib.load(), attend_args(2)
    P.batch, P.kv_heads, P.heads, P.capacity = batch, kv_heads, kv_heads, 1
    for lvl in list(P.levels)[:2]:
        for name in ("k", "v", "dk", "dv", "bias", "lse", "q", "out"):
            getattr(lvl, name).heads = kv_heads
    assert lib.pa_draft_attend_workspace(ctypes.byref(P)) == 0
    assert lib.pa_draft_attend(ctypes.byref(P), None) == _lib.PA_EUNSUPPORTED


def test_attend_takes_as_many_as_a_grid_holds():
    lib, P = _lib.load(), attend_args(2)
    P.batch, P.kv_heads, P.heads, P.capacity = MOST // 2, 1, 1, 1
    assert lib.pa_draft_attend_workspace(ctypes.byref(P)) > 0


def test_append_and_commit_refuse_more_rows_than_a_grid_holds():
    lib, R, C = _lib.load(), rows_args(), commit_args()
    R.batch, R.drafts = MOST // 5 + 1, 5
    assert lib.pa_draft_append(ctypes.byref(R), None) == _lib.PA_EUNSUPPORTED
    C.batch = MOST + 1
    assert lib.pa_draft_commit(ctypes.byref(C), None) == _lib.PA_EUNSUPPORTED
