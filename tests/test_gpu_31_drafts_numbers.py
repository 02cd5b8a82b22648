"""GPU: drafted attention over cached keys that are no numbers."""

import pytest
import torch

from test_gpu_25_drafts import DT, dev, fill_cache

pytestmark = pytest.mark.gpu
param = pytest.mark.parametrize


@param("dtype", ["bf16", "f16", "f32"])
@param("n, T, H, D, lo, hi", [
    (100, 1, 1, 64, 0, 32),        # all that one wave has, of a unit
    (100, 5, 2, 64, 0, 64),
    (9000, 3, 2, 64, 0, 8000),     # whole units
    (9000, 64, 8, 128, 0, 4096),   # blocks of many rows
    (300, 40, 4, 96, 0, 128),
])
def test_keys_that_are_no_numbers(n, T, H, D, lo, hi, dtype):
    """A softmax over such a score is none, also where all of a wave's or a unit's scores are."""
    from poly_attention import DraftCache

    d = dev()
    g = torch.Generator().manual_seed(n + T)
    cache = DraftCache.empty(order=2, batch=1, kv_heads=1, dim_head=D, capacity=n, max_drafts=T, dtype=DT[dtype], device=d,
                             counts=torch.tensor([n], dtype=torch.int32, device=d))
    fill_cache(cache, g, d)
    q1 = torch.randn(1, H, T, D, generator=g).to(DT[dtype]).to(d)
    assert bool(torch.isfinite(cache.attend(q1)).all())
    for x in cache.qs:
        x[:, :, lo:hi] = float("nan")
    out = cache.attend(q1)
    assert bool(torch.isnan(out).all())
    assert bool(torch.isnan(cache.draft_lses[0][:, :, :T]).all()) and bool(torch.isnan(cache.draft_msgs[0][:, :, :T]).all())
