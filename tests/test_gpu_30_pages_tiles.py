"""GPU: chunks of many query rows (k_paged_tiles): head dims between the kernels' own, units of a few positions, and what is
not finite behind a token, with and without a soft clamp, in one unit and in several."""

import pytest
import torch

import pages_oracle as PO
from test_gpu_27_pages import DT, assert_within, check_attend, dev, fill, inputs, make

pytestmark = pytest.mark.gpu
param = pytest.mark.parametrize


@param("dtype", ["bf16", "f16"])
@param("D", [8, 40, 72, 96, 120])
@param("counts, new, packed", [([200, 150], [150, 70], False),             # one unit of a row each
                               ([3000, 90, 700], [200, 90, 1], True)])     # several, and few rows beside them
def test_head_dims_between(counts, new, packed, D, dtype):
    check_attend(3, counts, new, 4, 2, D, dtype, 32, packed)
    check_attend(2, counts, new, 4, 2, D, dtype, 16, not packed, softclamp=4.0)


def last_unit(n, m, rep, kv_heads, D):
    """Positions of the last unit of a single row's tiles, as the launch of many rows splits them: chunks of 128 positions, two
    at least to a unit, and no more units than the card has room for."""
    rows = m * rep
    tiles, chunks = -(-rows // 256), -(-n // 128)
    target = max(1, 256 * (1 if D > 64 else 2) // kv_heads)
    aim = max(target - tiles // 2, target // 2 + 1)
    size = max(-(-tiles * chunks // aim), 2)
    splits = -(-chunks // size)
    size = -(-chunks // splits)
    return n - (splits - 1) * size * 128


@param("softclamp", [None, 5.0])
@param("dtype", ["bf16", "f16"])
@param("D", [64, 128])
@param("n, m, H, hk, want", [(257, 200, 1, 1, 1), (320, 250, 1, 1, 64), (290, 90, 2, 1, 34), (1537, 300, 2, 2, 1)])
def test_units_of_a_few_positions(n, m, H, hk, want, D, dtype, softclamp):
    """One tile of 64 positions, or a part of one, is all that a workgroup of many rows has: where the GPU once faulted."""
    assert last_unit(n, m, 1, hk, D) == want <= 64
    check_attend(2, [n], [m], H, hk, D, dtype, 64, softclamp=softclamp)


@param("softclamp", [None, 4.0])
@param("dtype", ["bf16", "f16"])
@param("D", [64, 96, 128])
@param("counts, new", [([240], [100]), ([700], [200]), ([4000, 180], [300, 90])])
def test_what_a_token_does_not_see(counts, new, D, dtype, softclamp):
    """Infinities and NaN in the last tokens' keys, queries and values reach no earlier token: those stay within the bounds of
    what they see."""
    from poly_attention import PagedCache

    dev()
    g = torch.Generator().manual_seed(3)
    t, o = make(counts, new, 16, g)
    cache = PagedCache(t, order=3, kv_heads=2, dim_head=D, dtype=DT[dtype])
    host = fill(cache, o, g)
    q1, v = inputs(o, 4, D, DT[dtype], False, g), inputs(o, 2, D, DT[dtype], False, g)
    (out, tol), values, lses = PO.attend(q1, [v], host, o, False, D ** -0.5, softclamp)
    bad = [(3, float("inf")), (1, float("nan")), (2, -float("inf"))]
    q, w = q1.cuda(), v.cuda()
    for b, n in enumerate(counts):
        for k, x in bad:
            page, slot = o.pages[b][(n - k) // 16], (n - k) % 16
            for a in (*cache.keys, cache.values[0]):
                a[page, :, slot] = x
            w[b, :, new[b] - k] = x
            q[b, :, new[b] - k] = x
    got = cache.attend(q, [w], softclamp=softclamp)
    for b, n in enumerate(counts):
        m = new[b] - 3
        assert_within(got[b, :, :m], out[b, :, :m], tol[b, :, :m], f"row {b}")
        for x, (y, y_tol) in [*zip(cache.values[1:], values[1:]), *zip(cache.lses, lses)]:
            for p in range(n - new[b], n - 3):
                at = o.pages[b][p // 16], slice(None), p % 16
                assert_within(x[at], y[at], y_tol[at], f"position {p}")
        # the last token sees all of them
        assert not bool(torch.isfinite(got[b, :, new[b] - 1].float()).any())


@param("softclamp", [None, 6.0])
@param("dtype", ["bf16", "f16"])
@param("D", [64, 128])
@param("n, m", [(250, 200), (3000, 300)])
def test_what_is_cached_holds_more_than_one_rounding(n, m, D, dtype, softclamp):
    """Values that a level leaves in the cache for later levels and tokens are its averages, rounded once: weights that were
    rounded to the type as well would leave them sqrt(2) times as far from 64 bits (in norm).  Two numbers hold a weight to 2^-16,
    which beside the result's 2^-9 (fp16: 2^-22 beside 2^-12) is below a hundredth, and fp32 scores of some 10 are within 2^-19."""
    from poly_attention import PagedCache

    dev()
    g = torch.Generator().manual_seed(9)
    t, o = make([n], [m], 64, g)
    cache = PagedCache(t, order=3, kv_heads=2, dim_head=D, dtype=DT[dtype])
    fill(cache, o, g)
    q1, v = inputs(o, 4, D, DT[dtype], False, g).cuda(), inputs(o, 2, D, DT[dtype], False, g).cuda()
    cache.attend(q1, [v], softclamp=softclamp)
    rows = lambda x: PO.row_of(x, o.pages[0], n, 64).double()  # noqa: E731
    hidden = torch.arange(n, device="cuda") > torch.arange(n - m, n, device="cuda")[:, None]
    for lvl in range(2):
        s = rows(cache.keys[lvl + 1])[:, n - m:] @ rows(cache.keys[lvl]).transpose(1, 2) * D ** -0.5
        if softclamp:
            s = softclamp * torch.tanh(s / softclamp)
        if lvl:
            s = s + rows(cache.lses[0])[:, None]
        s = s.masked_fill(hidden, -float("inf"))
        want = s.softmax(-1) @ rows(cache.values[lvl])
        if not lvl:
            want = want * v[0].double()
        off = (rows(cache.values[lvl + 1])[:, n - m:] - want).norm()
        least = (want.to(DT[dtype]).double() - want).norm()
        assert off <= 1.1 * least, (lvl, (off / least).item())


@param("counts, new, packed", [([250, 100], [200, 1], True), ([6000, 130], [300, 90], False), ([90] * 40, [90] * 40, False)])
@param("D", [64, 128])
def test_whatever_the_workspace_held(counts, new, packed, D):
    """Every byte of a workspace that a call reads was written by it."""
    from poly_attention import PagedCache

    dev()
    g = torch.Generator().manual_seed(2)
    t, o = make(counts, new, 64, g)
    cache = PagedCache(t, order=2, kv_heads=2, dim_head=D, dtype=torch.bfloat16)
    fill(cache, o, g)
    q1 = inputs(o, 4, D, torch.bfloat16, packed, g).cuda()
    want = cache.attend(q1)
    size = cache._plans["attend", q1.shape][0].workspace_bytes
    for byte in (0, 255, 127, 1):
        torch.cuda.synchronize()
        torch.full((size,), byte, dtype=torch.uint8, device="cuda")  # the block that the call takes next
        assert torch.equal(cache.attend(q1), want)


@param("counts, new, H, hk, D", [([300, 5000], [1, 1], 128, 1, 128), ([40, 700, 64], [1, 0, 2], 160, 2, 64), ([513], [1], 72, 1, 96)])
@param("packed", [False, True])
def test_single_tokens_of_many_heads(counts, new, H, hk, D, packed):
    """More query heads of a key head than a few rows: single tokens are many rows too, with and without other levels'."""
    check_attend(2, counts, new, H, hk, D, "bf16", 64, packed)
    check_attend(3, counts, new, H, hk, D, "f16", 16, packed, softclamp=8.0)
