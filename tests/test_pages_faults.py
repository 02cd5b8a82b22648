"""Faults that the paged cache had and that show without a GPU, one test each."""

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
