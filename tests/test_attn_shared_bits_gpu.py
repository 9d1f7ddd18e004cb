"""Attention of rows that share pages: the same bits from call to call, f32 results against tight bounds."""
import pytest

from test_attn_shared_gpu import Batch, behind

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_the_same_bits_every_time(ctx, dtype):
    """Sums are cut and joined in an order that the sizes alone decide: alone, beside other work, and behind other calls."""
    import torch
    dt = getattr(torch, dtype)
    cases = [Batch(ctx, [behind(100, [5 * i for i in range(60)]), (20, list(range(1, 321)))], 32, 8), Batch(ctx, [(31, list(range(20, 480)))], 12, 4, prompts=True, window=300),
             Batch(ctx, [behind(600, [9, 300, 0])], 8, 8)]
    args = [b.args() for b in cases]
    torch.cuda.synchronize()
    first = [ctx.attn_shared(*a, **kw, softcap=cap, dtype=dt) for a, kw in args for cap in (0.0, 50.0)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    again = []
    for k in range(6):
        for i, (a, kw) in enumerate(args):
            with torch.cuda.stream(streams[(i + k) % 3]):
                again += [(2 * i + j, ctx.attn_shared(*a, **kw, softcap=cap, dtype=dt)) for j, cap in enumerate((0.0, 50.0))]
    torch.cuda.synchronize()
    for i, got in again:
        assert torch.equal(got, first[i])
    for b in cases:
        b.pool.free()
    ctx.device_status()


@pytest.mark.parametrize("softcap", [0.0, 30.0, 50.0, 2000.0])
@pytest.mark.parametrize("groups,heads,kv_heads", [([behind(9, [1, 40, 17, 300])], 8, 2), ([behind(130, [1, 600, 90, 33] * 9)], 32, 8),
                                                   ([behind(1000, [17, 2000])], 8, 1), ([behind(0, [3000, 5, 100])], 12, 4)])
def test_f32_results_to_their_last_bits(ctx, groups, heads, kv_heads, softcap):
    """The bound of the test of long sums: a sum is added to 32 times, cut to 2^-23 each time, before it is rounded to nearest, and
    2^-21 for scores and weights.  Rows with whole and with cut sums, of shared pages and of their own."""
    b = Batch(ctx, groups, heads, kv_heads)
    a, kw = b.args()
    got = ctx.attn_shared(*a, **kw, softcap=softcap)
    want, _ = b.exact(softcap=softcap)
    assert float((got.double() - want).norm() / want.norm()) < 32 * 2.0 ** -23 + 2.0 ** -21
    b.pool.free()
