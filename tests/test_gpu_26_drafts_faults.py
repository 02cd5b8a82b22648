"""GPU: drafted tokens, cases that once went wrong or could have: each test says which."""

import pytest
import torch

from test_gpu_25_drafts import BUFS, dev, random_caches

pytestmark = pytest.mark.gpu
param = pytest.mark.parametrize


def test_commit_many_buffers_at_one_count():
    """Every workgroup of a row moves to the count as it was before the call, however many draw their tickets
    before it (the count advances within the launch)."""
    from poly_attention import commit_drafts

    d = dev()
    g = torch.Generator().manual_seed(3)
    B, slots, cap = 5, 8, 200
    caches = random_caches(12, 3, B, 2, 64, cap, slots, [0, 3, 17, 150, 40], "bf16", d, g)  # 120 buffers: one launch
    bufs = [(dst, src) for c in caches for name in BUFS
            for dst, src in zip(getattr(c, name), getattr(c, "draft_" + name))]
    want = [dst.clone() for dst, _ in bufs]
    counts = caches[0].lengths()
    for step in range(12):
        path = torch.stack([torch.randperm(slots, generator=g) for _ in range(B)]).int()
        kept = torch.randint(0, 5, (B,), generator=g).int()
        commit_drafts(caches, path.to(d), kept.to(d))
        for b in range(B):
            for w, (_, src) in zip(want, bufs):
                w[b, :, counts[b]:counts[b] + kept[b]] = src[b][:, path[b, :kept[b]].tolist()]
            counts[b] += int(kept[b])
        assert caches[0].lengths() == counts
        for w, (dst, _) in zip(want, bufs):
            assert torch.equal(dst, w), step
