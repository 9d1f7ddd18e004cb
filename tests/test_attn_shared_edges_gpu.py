"""Attention of rows that share pages: caps of any size, page ids outside the pool."""
import math

import pytest

from test_attn_shared_gpu import PAGE, Batch, _ints, assert_near, behind, check

pytestmark = pytest.mark.gpu


def without_page_0(b):
    """Page 0 of the pool is nobody's."""
    spare = min(set(range(b.pages)) - set(b.table_np.ravel().tolist()))
    if spare:
        data = b.pool.tensor()
        data[spare] = data[0]
        b.table_np[b.table_np == 0] = spare
        b.table = _ints(b.table_np)
    assert 0 not in b.table_np
    return b.pool.tensor()[0]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("bad", [-1, -2 ** 31, 2 ** 31 - 1, "pages"])
def test_a_page_outside_the_pool_is_nobodys_page(ctx, bad, dtype):
    """Shared pages and a row's own: what stands in page 0 (of another request) has no part in the results, those of rows that attend
    a page outside the pool included, and rows that do not attend it are right."""
    import torch
    from cyb_b200 import qeng
    # rows that all attend the page, rows of which some do, a window that ends in it
    for groups, at, window, prompts in (([behind(40, [3, 20, 7])], 12, 0, False), ([(20, [100, 150, 200, 320])], 10, 0, False), ([(8, [128 - i for i in range(70)])], 7, 0, False),
                                        ([(30, list(range(300, 470)))], 25, 60, True), ([behind(2, [100, 5])], 5, 0, False)):
        b = Batch(ctx, groups, 8, 2, window=window, prompts=prompts, junk=0.0)
        nobody = without_page_0(b)
        want, mag = b.exact()
        bent = b.table_np.copy()
        shared = at < groups[0][0]
        bent[slice(None) if shared else 0, at] = b.pages if bad == "pages" else bad
        (pool, q, _, *rest), kw = b.args()
        got = []
        for what in (0.0, math.nan, math.inf, 100.0):
            nobody.fill_(what)
            got.append(ctx.attn_shared(pool, q, _ints(bent), *rest, **kw, dtype=getattr(torch, dtype)))
            with pytest.raises(qeng.QengError, match="status 1"):
                ctx.device_status()
        assert bool(torch.isfinite(got[0]).all())
        for other in got[1:]:
            assert torch.equal(other, got[0])
        sound = [t for t, n in enumerate(b.lens) if n <= at * PAGE or (window and n - window >= (at + 1) * PAGE) or (not shared and t != 0)]
        assert_near(got[0][sound], want[sound], mag[sound])
        b.pool.free()


@pytest.mark.parametrize("softcap", [0.25, 200.0, 256.0, 257.0, 1e3, 1e5, 1e8, 1e20])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_caps_far_from_the_scores(ctx, dtype, softcap):
    """A cap bends scores near it and leaves those far below alone: no error that grows with the cap."""
    check(ctx, [behind(21, [0, 1, 90, 33]), behind(0, [40]), behind(9, [3] * 70)], 12, 4, dtype, softcap=softcap)
    check(ctx, [(30, list(range(1, 470)))], 8, 2, dtype, softcap=softcap, prompts=True, window=333)


def test_caps_that_leave_32_bits_are_refused(ctx):
    """An infinite one, or one far below what scores are: rows would be NaN."""
    from cyb_b200 import qeng
    b = Batch(ctx, [behind(3, [5])], 8, 2)
    a, kw = b.args()
    for cap, scale in ((math.inf, 1.0), (2e30, 1.0), (1e-39, 1.0), (1e-30, 1e9)):
        with pytest.raises(qeng.QengError, match="leaves 32 bits"):
            ctx.attn_shared(*a, **kw, softcap=cap, scale=scale)
    b.pool.free()
    check(ctx, [behind(3, [5])], 8, 2, softcap=1e30)
    check(ctx, [behind(3, [5])], 8, 2, softcap=1e-30, scale=1.0)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("softcap", [30.0, 1000.0])
def test_a_cap_brings_infinite_scores_to_itself(ctx, softcap, dtype):
    """Among shared pages and a row's own; NaN stays NaN."""
    import torch
    for shared in (0, 6):
        b = Batch(ctx, [(6, [96, 80, 17, 3])], 4, 1, junk=0.0)
        b.table_np[:] = b.table_np[0]
        b.table, b.shared = _ints(b.table_np), [shared]
        data = b.pool.tensor()
        b.q[:, :, 0] = 1.0
        at = [int(b.table_np[0, k]) for k in (1, 4)]
        data[at[0], 0, 0, 5, 0], data[at[1], 0, 0, 9, 0] = math.inf, -math.inf
        a, kw = b.args()
        got = ctx.attn_shared(*a, **kw, softcap=softcap, dtype=getattr(torch, dtype))
        assert_near(got, *b.exact(softcap=softcap))
        data[at[0], 0, 0, 5, 0] = math.nan
        got = ctx.attn_shared(*a, **kw, softcap=softcap, dtype=getattr(torch, dtype))
        assert bool(torch.isnan(got[:2]).all()) and bool(torch.isfinite(got[3]).all())
        b.pool.free()
