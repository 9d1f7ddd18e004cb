"""Attention of rows that share their first pages (through the C ABI) against the definition in 64 bits."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
PAGE, HD = 16, 128


def _ints(v):
    import torch
    return torch.tensor(np.asarray(v, dtype=np.int32), device="cuda")


class Batch:
    """groups: a list of (shared pages, [lengths]).  `prompts`: the rows of a group have one table row.  Places that no row attends
    hold NaN."""

    def __init__(self, ctx, groups, heads, kv_heads, window=0, prompts=False, seed=0, spare=3, junk=math.nan):
        import torch
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.ctx, self.window, self.heads, self.kv_heads = ctx, window, heads, kv_heads
        self.first = [0]
        lens, rows, tables, at = [], [], [], 0
        width = max(1, max([p for p, _ in groups] + [-(-n // PAGE) for _, ls in groups for n in ls]))
        for p, ls in groups:
            shared = list(range(at, at + p))
            at += p
            for i, n in enumerate(ls):
                if prompts and i > 0:
                    rows.append(len(tables) - 1)
                else:
                    rows.append(len(tables))
                    m = 0 if prompts else max(0, -(-n // PAGE) - p)
                    tables.append(shared + list(range(at, at + m)) + [-1] * (width - p - m))
                    at += m
            lens += list(ls)
            self.first.append(len(lens))
        self.pages = at + spare
        order = torch.randperm(self.pages, generator=g, device="cuda").cpu().numpy()
        t = np.array(tables, np.int32).reshape(-1, width)
        self.table_np = np.where(t < 0, -1, order[np.maximum(t, 0)]).astype(np.int32)
        self.lens, self.rows, self.shared = lens, rows if prompts else None, [p for p, _ in groups]
        self.q = torch.randn(len(lens), heads, HD, generator=g, device="cuda").half()
        self.pool = ctx.kv_pool(self.pages, kv_heads)
        data = self.pool.tensor()
        values = torch.randn(data.shape, generator=g, device="cuda").half()
        used = torch.zeros(self.pages * PAGE, dtype=torch.bool, device="cuda")
        for t, n in enumerate(lens):
            a = max(0, n - window) if window else 0
            j = torch.arange(a, n, device="cuda")
            ids = torch.tensor(self.table_np[rows[t]], device="cuda").long()
            used[ids[j // PAGE] * PAGE + j % PAGE] = True
        used = used.view(self.pages, 1, 1, PAGE, 1)
        data.copy_(torch.where(used, values, torch.full_like(values, junk)))
        self.table = _ints(self.table_np)

    def args(self):
        return (self.pool, self.q, self.table, _ints(self.lens), _ints(self.first), _ints(self.shared)), dict(
            rows=None if self.rows is None else _ints(self.rows), window=self.window)

    def exact(self, scale=None, softcap=0.0):
        """Outputs, and sums of weights times magnitudes.  The kernels' weights are f16 numbers (or two) of up to 2^8 and more for the
        largest, so that a weight is a multiple of 2^-24 at least, off by 2^-25 / 2^8 of the largest: 2^-33 of every value's magnitude,
        which comes into the sums as 2^-19 (assert_near allows 2^-14 of them)."""
        import torch
        out = torch.zeros(len(self.lens), self.heads, HD, dtype=torch.float64, device="cuda")
        mag = torch.zeros_like(out)
        kv = self.pool.tensor()
        scale = HD ** -0.5 if scale is None else scale
        for t, n in enumerate(self.lens):
            a = max(0, n - self.window) if self.window else 0
            if n <= a:
                continue
            row = t if self.rows is None else self.rows[t]
            ids = torch.tensor(self.table_np[row, :-(-n // PAGE)], device="cuda").long()
            k, v = (kv[ids][:, :, i].transpose(0, 1).reshape(self.kv_heads, -1, HD)[:, a:n].double() for i in range(2))
            x = torch.einsum("hgd,hld->hgl", self.q[t].double().view(self.kv_heads, -1, HD), k) * scale
            if softcap:
                x = softcap * torch.tanh(x / softcap)
            w = torch.softmax(x, -1)
            out[t] = torch.einsum("hgl,hld->hgd", w, v).reshape(self.heads, HD)
            mag[t] = torch.einsum("hgl,hld->hgd", w + 2.0 ** -19, v.abs()).reshape(self.heads, HD)
        return out, mag


def assert_near(got, want, mag):
    """Half a step of the result's type; weights of 22 bits (f32 results) or 11; 2^-14 of every weight for scores: 128 products
    summed in f32 at magnitudes up to 2^6, in their exponent."""
    import torch
    step = torch.finfo(got.dtype).eps / 2
    weights = 2.0 ** -22 if got.dtype == torch.float32 else 2.0 ** -11
    d = (got.double() - want).abs()
    bound = step * want.abs() + (weights + 2.0 ** -14) * mag + 1e-30
    assert torch.isfinite(got).all()
    assert bool((d <= bound).all()), float((d / bound).max())


def check(ctx, groups, heads, kv_heads, dtype="float32", softcap=0.0, window=0, prompts=False, seed=0, scale=None):
    import torch
    b = Batch(ctx, groups, heads, kv_heads, window=window, prompts=prompts, seed=seed)
    a, kw = b.args()
    got = ctx.attn_shared(*a, **kw, scale=scale, softcap=softcap, dtype=getattr(torch, dtype))
    want, mag = b.exact(scale, softcap)
    assert_near(got, want, mag)
    for t, n in enumerate(b.lens):
        if n == 0:
            assert bool((got[t] == 0).all())
    ctx.device_status()
    b.pool.free()


def behind(pages, own):
    return pages, [pages * PAGE + n for n in own]


@pytest.mark.parametrize("heads,kv_heads", [(32, 8), (8, 1), (12, 4), (7, 1), (3, 3), (20, 4)])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_heads_and_types(ctx, heads, kv_heads, dtype):
    check(ctx, [behind(9, [1, 40, 17, 0, 16, 33])], heads, kv_heads, dtype, seed=heads)


@pytest.mark.parametrize("pages", [0, 1, 2, 7, 8, 9, 15, 16, 17, 33, 130])
@pytest.mark.parametrize("rows", [1, 3, 16, 17, 32, 33, 64, 65, 100])
def test_sizes(ctx, pages, rows):
    """Around the sizes of tiles (128 rows of heads, or two of them), stages of keys and pages."""
    check(ctx, [behind(pages, [(7 * i) % 50 for i in range(rows)])], 16, 4, "float16" if rows % 2 else "float32", seed=rows)


@pytest.mark.parametrize("pages", [299, 300, 304, 410, 1000])
@pytest.mark.parametrize("rows", [2, 150])
def test_many_blocks(ctx, pages, rows):
    """Several blocks and pieces of kv heads to a CTA, whose last block is whole or not."""
    check(ctx, [behind(pages, [(7 * i) % 50 for i in range(rows)])], 16, 8, seed=rows)
    check(ctx, [(pages, [pages * 16 - 30 * i for i in range(rows)])], 32, 8, "float16", seed=rows)
    check(ctx, [behind(pages, [i % 3 for i in range(rows)]), (pages - 37, [(pages - 37) * 16] * 40)], 8, 8, "bfloat16", window=4000)


def test_rows_that_end_inside_what_they_share(ctx):
    """Lengths of nothing, of one token, of page and stage borders, of all but one."""
    lens = [0, 1, 15, 16, 17, 127, 128, 129, 255, 256, 257, 300, 319, 320, 321, 400]
    for dtype in ("float32", "bfloat16"):
        check(ctx, [(20, lens)], 8, 2, dtype)
        check(ctx, [(20, [0] * 5)], 8, 2, dtype)
        check(ctx, [(20, [0] * 200 + [320])], 8, 2, dtype)


def test_groups(ctx):
    """Groups of none, one and many rows, with and without shared pages."""
    groups = [behind(3, [5]), (4, []), behind(0, [1, 100, 0]), behind(40, list(range(70))), (0, []), behind(1, [200] * 40), (7, [50]), behind(12, [3])]
    check(ctx, groups, 8, 2)
    check(ctx, groups, 8, 8, "bfloat16")
    check(ctx, [behind(i % 5, [i]) for i in range(1024)], 2, 1, "float16")


@pytest.mark.parametrize("window", [1, 15, 16, 17, 100, 128, 500, 639, 640, 641, 10000])
def test_windows(ctx, window):
    """A window that ends among a row's own pages, inside the shared ones, on their border, and beyond all."""
    check(ctx, [behind(40, [0, 1, 16, 50, 127, 300]), behind(2, [700, 3]), (40, [33, 639, 640])], 8, 2, "float32" if window % 2 else "float16", window=window)
    check(ctx, [(30, list(range(1, 470)))], 8, 2, "bfloat16", window=window, prompts=True)


@pytest.mark.parametrize("softcap", [1.0, 30.0, 50.0])
def test_softcap(ctx, softcap):
    check(ctx, [behind(21, [0, 1, 90, 33]), behind(0, [40])], 12, 4, softcap=softcap, scale=0.5)
    check(ctx, [behind(21, [0, 1, 90, 33])], 12, 4, "float16", softcap=softcap, window=200)


def test_scores_of_a_wide_range(ctx):
    """Maxima that grow from key to key by far, one weight that outweighs the rest, or all weights the same."""
    import torch
    for scale in (0.0, 1.0, 8.0):
        for dtype in (torch.float32, torch.bfloat16):
            b = Batch(ctx, [behind(70, [100, 0, 30])], 8, 2)
            b.q *= 0.25
            data = b.pool.tensor()
            data[:, :, 0] = torch.nan_to_num(data[:, :, 0])
            ramp = torch.linspace(0.1, 3, 70, device="cuda")
            ids = torch.tensor(b.table_np[0, :70], device="cuda").long()
            data[ids, :, 0] = (data[ids, :, 0] * ramp[:, None, None, None]).half()
            a, kw = b.args()
            got = ctx.attn_shared(*a, **kw, scale=scale, dtype=dtype)
            want, mag = b.exact(scale)
            # scores up to 2^9: 2^-11 of a weight
            d, step = (got.double() - want).abs(), torch.finfo(dtype).eps / 2
            assert bool((d <= step * want.abs() + (2.0 ** -11 + 2.0 ** -11) * mag).all())
            b.pool.free()


@pytest.mark.parametrize("prompts", [[1], [2, 1], [16], [17, 130], [300, 5, 64], [33] * 20, [700]])
@pytest.mark.parametrize("cached", [0, 1, 100, 128])
def test_prompts(ctx, prompts, cached):
    """Groups whose rows share all their pages and attend one key more from row to row."""
    groups = [(-(-(cached + n) // PAGE), [cached + i + 1 for i in range(n)]) for n in prompts]
    check(ctx, groups, 16, 4, "float16", prompts=True, seed=cached)
    check(ctx, groups, 8, 8, "float32", prompts=True, seed=cached)


def test_prompts_and_answers_in_one_call(ctx):
    import torch
    b = Batch(ctx, [(10, [1 + i for i in range(150)]), behind(30, [1, 70, 5]), behind(0, [99])], 8, 2)
    # the first group's rows are tokens of one request
    b.table_np[:150] = b.table_np[149]
    b.table = _ints(b.table_np)
    a, kw = b.args()
    got = ctx.attn_shared(*a, **kw)
    assert_near(got, *b.exact())
    b.pool.free()


def test_rows_left_alone_and_strides(ctx):
    """Rows that are in no group, or not there; rows of q and of the result with others between them."""
    import torch
    b = Batch(ctx, [behind(8, [3, 20, 0, 5]), behind(9, [40] * 40)], 8, 2)
    n = len(b.lens)
    want, mag = b.exact()
    big = torch.full((n + 7, 8 + 3, HD), 9.0, dtype=torch.float16, device="cuda")
    big[:n, :8] = b.q
    for dtype in (torch.float32, torch.bfloat16):
        out = torch.full((n + 7, 8 + 2, HD), 5.0, dtype=dtype, device="cuda")
        rows = list(range(n)) + [0] * 7
        gone = [0, 2, 20, n - 1]
        for t in gone[1:]:
            rows[t] = -1
        lens = list(b.lens) + [30] * 7
        first = [1] + b.first[1:]  # row 0 is in no group
        ctx.attn_shared(b.pool, big[:, :8], b.table, _ints(lens), _ints(first), _ints(b.shared), rows=_ints(rows), out=out[:, :8])
        live = [t for t in range(n) if t not in gone]
        assert_near(out[live, :8], want[live], mag[live])
        assert bool((out[:, 8:] == 5).all()) and bool((out[gone] == 5).all()) and bool((out[n:] == 5).all())
    b.pool.free()
    ctx.device_status()


@pytest.mark.parametrize("shared", [0, 10, 20])
def test_what_is_not_finite_reaches_the_rows_that_attend_it(ctx, shared):
    """V and K that are not finite in single places, attended by some rows of a tile, by all, or by none.  A value of infinity gives infinity or
    NaN: its weight is a sum of two numbers, hi + lo, with lo of either sign or zero, and infinity * hi + infinity * lo is NaN where lo <= 0."""
    import torch
    lens = [1, 20, 40, 60, 64, 100, 130, 160, 161, 200, 300, 320]
    for dtype in (torch.float32, torch.float16):
        for what, place, dims in [(math.inf, 59, [3]), (math.nan, 159, [0, 127]), (-math.inf, 0, [64]), (math.inf, 299, [5])]:
            b = Batch(ctx, [(20, lens)], 8, 2, junk=0.0)
            b.table_np[:] = b.table_np[-1]  # one sequence's pages for all
            b.table = _ints(b.table_np)
            b.shared = [shared]
            data = b.pool.tensor()
            data.copy_(torch.where(torch.isfinite(data), data, 0))
            pid = int(b.table_np[0, place // PAGE])
            data[pid, 1, 1, place % PAGE, dims] = what
            a, kw = b.args()
            got = ctx.attn_shared(*a, **kw, dtype=dtype)
            data[pid, 1, 1, place % PAGE, dims] = 0
            want, mag = b.exact()
            for t, n in enumerate(lens):
                hit = torch.zeros(8, HD, dtype=torch.bool, device="cuda")
                if n > place:
                    hit[4:, dims] = True
                assert not bool(torch.isfinite(got[t][hit]).any()), (what, n)
                keep = ~hit
                assert_near(got[t][keep], want[t][keep], mag[t][keep])
            # a score that is not a number, or infinite: NaN for the rows that attend it
            for bad in (math.nan, math.inf):
                data[pid, 0, 0, place % PAGE, 7] = bad
                b.q[:, :, 7] = b.q[:, :, 7].abs() + 0.25
                got = ctx.attn_shared(b.pool, b.q, *a[2:], **kw, dtype=dtype)
                data[pid, 0, 0, place % PAGE, 7] = 0.5
                want, mag = b.exact()
                for t, n in enumerate(lens):
                    if n > place:
                        assert bool(torch.isnan(got[t, :4]).all())
                        assert_near(got[t, 4:], want[t, 4:], mag[t, 4:])
                    else:
                        assert_near(got[t], want[t], mag[t])
            b.pool.free()
    ctx.device_status()


def test_scores_of_minus_infinity(ctx):
    """Such keys weigh nothing; a row that attends nothing else is NaN, as its formula says."""
    import torch
    for shared in (0, 5):
        b = Batch(ctx, [(5, [80, 16, 17, 1])], 4, 1, junk=0.0)
        b.table_np[:] = b.table_np[0]
        b.table, b.shared = _ints(b.table_np), [shared]
        data = b.pool.tensor()
        first = int(b.table_np[0, 0])
        b.q[:, :, 0] = 1.0
        data[first, 0, 0, :, 0] = -math.inf
        a, kw = b.args()
        got = ctx.attn_shared(*a, **kw)
        want, mag = b.exact()
        assert bool(torch.isnan(got[[1, 3]]).all())
        assert_near(got[[0, 2]], want[[0, 2]], mag[[0, 2]])
        b.pool.free()


def test_agrees_with_the_decode_attention(ctx):
    """The same table through qeng_attn_decode_ex, which reads every page for every row."""
    import torch
    for softcap, window in ((0.0, 0), (20.0, 0), (0.0, 300), (50.0, 77)):
        b = Batch(ctx, [behind(30, [1, 99, 230, 16])], 32, 8, window=window)
        a, kw = b.args()
        got = ctx.attn_shared(*a, **kw, softcap=softcap)
        want = ctx.attn_decode(b.pool, b.q, b.table, a[3], softcap=softcap, window=window)
        assert float((got - want).abs().max()) < 1e-4 * float(want.abs().max())
        b.pool.free()


def test_long_prefix_and_pages_past_32_bits(ctx):
    """20000 shared tokens in a pool of more than 4 GB, the pages at both its ends."""
    import torch
    pages, hkv, n = 70000, 8, 1250
    pool = ctx.kv_pool(pages, hkv)
    data = pool.tensor()
    g = torch.Generator(device="cuda").manual_seed(3)
    ids = torch.cat([torch.arange(pages - 1000, pages), torch.arange(300)]).cuda()[torch.randperm(1300, generator=g, device="cuda")]
    data[ids] = torch.randn((1300,) + tuple(data.shape[1:]), generator=g, device="cuda").half()
    own = torch.randperm(50, generator=g, device="cuda")
    table = torch.cat([ids[:n].expand(5, n), ids[n:][own].view(5, 10)], 1).to(torch.int32).contiguous()
    lens = [20000 + k for k in (0, 1, 16, 97, 160)]
    q = torch.randn(5, 16, HD, generator=g, device="cuda").half()
    b = Batch.__new__(Batch)
    b.window, b.heads, b.kv_heads, b.pool, b.lens, b.rows, b.q, b.table_np = 0, 16, hkv, pool, lens, None, q, table.cpu().numpy()
    for dtype in (torch.float32, torch.bfloat16):
        got = ctx.attn_shared(pool, q, table, _ints(lens), _ints([0, 5]), _ints([n]), dtype=dtype)
        assert_near(got, *b.exact())
    pool.free()


def test_reports_what_makes_no_sense(ctx):
    import torch
    from cyb_b200 import qeng
    b = Batch(ctx, [behind(9, [3, 20, 7]), behind(1, [5])], 8, 2, junk=0.0)
    (pool, q, table, lens, first, shared), kw = b.args()
    want, mag = b.exact()
    # page ids outside the pool: the others' results stand
    for bad in (-1, b.pages, 2 ** 31 - 1):
        t = table.clone()
        t[1, 10] = bad  # a page of row 1 alone
        got = ctx.attn_shared(pool, q, t, lens, first, shared)
        with pytest.raises(qeng.QengError, match="status 1"):
            ctx.device_status()
        assert_near(got[[0, 2, 3]], want[[0, 2, 3]], mag[[0, 2, 3]])
        t = table.clone()
        t[0, 4] = bad  # a shared one
        got = ctx.attn_shared(pool, q, t, lens, first, shared)
        with pytest.raises(qeng.QengError, match="status 1"):
            ctx.device_status()
        assert_near(got[3:], want[3:], mag[3:])
    # rows outside the table
    got = torch.full(q.shape, 5.0, device="cuda")
    ctx.attn_shared(pool, q, table, lens, first, shared, rows=_ints([0, 4, 2, 3]), out=got)
    with pytest.raises(qeng.QengError, match="status 6"):
        ctx.device_status()
    assert bool((got[1] == 5).all())
    assert_near(got[[0, 2, 3]], want[[0, 2, 3]], mag[[0, 2, 3]])
    # bounds of groups that do not ascend, or leave the call's rows: nothing is written
    for f in ([0, 3, 2], [0, 5, 4], [0, 3, 5], [-1, 3, 4], [0, -2147483648, 4], [0, 2147483647, 4]):
        got = torch.full(q.shape, 5.0, device="cuda")
        ctx.attn_shared(pool, q, table, lens, _ints(f), shared, out=got)
        with pytest.raises(qeng.QengError, match="status 6"):
            ctx.device_status()
        assert bool((got == 5).all())
    # pages shared beyond the table, lengths beyond it or below nothing: as far as there is one
    width = table.shape[1]
    one = Batch(ctx, [(4, [64, 64])], 8, 2)
    (p1, q1, t1, l1, f1, s1), _ = one.args()
    assert t1.shape[1] == 4
    got = ctx.attn_shared(p1, q1, t1, _ints([2 ** 31 - 1, -5]), f1, _ints([2 ** 31 - 1]))
    w1, m1 = one.exact()
    assert_near(got[:1], w1[:1], m1[:1])
    assert bool((got[1] == 0).all())
    got = ctx.attn_shared(p1, q1[:1], t1, l1[:1], _ints([0, 1]), _ints([-3]))
    assert_near(got, w1[:1], m1[:1])
    one.pool.free()
    b.pool.free()
    ctx.device_status()


def test_refusals(ctx):
    import torch
    from cyb_b200 import qeng
    pool = ctx.kv_pool(4, 2)
    x = torch.zeros(4096, dtype=torch.float32, device="cuda").data_ptr()

    def call(q=x, ldq=4 * HD, max_pages=1, table_rows=8, rows=x, lens=x, T=2, hq=4, first=x, G=1, cap=0.0, window=0, out=x, dt=0, ldo=4 * HD, scale=1.0):
        return qeng._lib.qeng_attn_shared(ctx.h, pool.h, q, ldq, x, max_pages, table_rows, rows, lens, T, hq, first, x, G, scale, cap, window, out, dt, ldo, None)
    for kw, code in [(dict(q=None), -1), (dict(lens=None), -1), (dict(first=None), -1), (dict(out=None), -1), (dict(T=0), -1), (dict(hq=0), -1),
                     (dict(max_pages=0), -1), (dict(table_rows=0), -1), (dict(G=0), -1), (dict(cap=-1.0), -1), (dict(cap=math.nan), -1), (dict(window=-1), -1), (dict(scale=-1.0), -1), (dict(scale=math.nan), -1),
                     (dict(dt=3), -1), (dict(dt=-1), -1), (dict(hq=3), -2), (dict(hq=18, ldq=18 * HD, ldo=18 * HD), -2), (dict(G=1025), -2), (dict(T=1 << 17, G=1024, hq=16, ldq=16 * HD, ldo=16 * HD, table_rows=1 << 17), -2),
                     (dict(T=1 << 20), -2), (dict(max_pages=(1 << 26) + 1), -2), (dict(rows=None, table_rows=1), -2), (dict(ldq=4 * HD - 8), -2),
                     (dict(ldo=4 * HD - 8), -2), (dict(q=x + 8), -3), (dict(out=x + 8), -3), (dict(ldq=4 * HD + 4), -3), (dict(ldo=4 * HD + 2), -3),
                     (dict(ldo=4 * HD + 4, dt=2), -3)]:
        assert call(**kw) == code, kw
    pool.free()
    ctx.device_status()


def test_streams_and_graphs(ctx):
    """Captured as the first call of a context, replayed beside calls of other shapes on other streams; two captured calls in turn."""
    import torch
    from cyb_b200 import qeng
    fresh = qeng.Context(0)
    small = Batch(fresh, [behind(40, [3, 70, 16, 300])], 8, 2)
    large = Batch(fresh, [behind(100, [5] * 90), (20, list(range(1, 321)))], 8, 2, seed=1)
    outs, graphs = [], []
    for b in (small, large):
        a, kw = b.args()
        out = torch.zeros(b.q.shape, dtype=torch.float32, device="cuda")
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            fresh.attn_shared(*a, **kw, out=out)
        outs.append((a, kw, out))
        graphs.append(g)
    wants = [b.exact() for b in (small, large)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    eager = []
    for k in range(12):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
            with torch.cuda.stream(streams[2 + i]):
                a, kw, _ = outs[1 - i]
                eager.append((1 - i, fresh.attn_shared(*a, **kw)))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert_near(outs[i][2], *wants[i])
    for i, got in eager:
        assert torch.equal(got, outs[i][2])  # the same sums in the same order
    fresh.device_status()
    del graphs
    small.pool.free()
    large.pool.free()
    fresh.close()


def test_from_request_lengths_to_attention(ctx):
    """A server's steps: a prompt that all share, answers behind it that grow by chunks and by single tokens, one of them ends and
    another takes its place.  Pages and slots from kv_plan, cache from rope_append, attention of every step against rotated rows in
    64 bits."""
    import torch
    hq, hkv, base, B, width = 8, 2, 1e4, 5, 24
    g = torch.Generator(device="cuda").manual_seed(9)
    pages = 90
    pool = ctx.kv_pool(pages, hkv)
    ring = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    ends = torch.tensor([0, pages], dtype=torch.int64, device="cuda")
    table = torch.zeros(B, width, dtype=torch.int32, device="cuda")
    lens = torch.zeros(B, dtype=torch.int32, device="cuda")
    keep = torch.full((B,), 6, dtype=torch.int32, device="cuda")  # 96 shared tokens
    story = [[] for _ in range(B)]  # q|k|v rows of every request so far

    def step(add, groups):
        """One plan, append and attention; groups: (first, shared pages) over the step's tokens, or None: a group per request."""
        nonlocal lens, ends
        plan = ctx.kv_plan(pool, lens, _ints(add), table, ring, ends, 200, keep=keep)
        lens, ends = plan.lens, plan.ends
        x = torch.randn(200, (hq + 2 * hkv) * HD, generator=g, device="cuda")
        q = torch.full((200, hq, HD), math.nan, dtype=torch.float16, device="cuda")
        ctx.rope_append(pool, x, plan.pos, plan.slots, base, out=q)
        if groups is None:  # rows of a request share all of its pages
            first, shared = plan.starts, (lens + PAGE - 1) // PAGE
        else:
            first, shared = _ints(groups[0]), _ints(groups[1])
        out = torch.full((200, hq, HD), 5.0, device="cuda")
        ctx.attn_shared(pool, q, table, plan.seen, first, shared, rows=plan.rows, out=out)
        ctx.device_status()
        at = 0
        for r, a in enumerate(add):
            if a < 0:
                story[r] = []
            for i in range(max(a, 0)):
                story[r].append(x[at])
                rows = torch.stack(story[r]).double().view(-1, hq + 2 * hkv, HD)
                ang = torch.arange(len(rows), device="cuda").double()[:, None, None] * base ** (-torch.arange(64, device="cuda").double() / 64)
                turn = torch.cat([rows[..., :64] * ang.cos() - rows[..., 64:] * ang.sin(), rows[..., 64:] * ang.cos() + rows[..., :64] * ang.sin()], -1)
                qq, k, v = turn[-1, :hq].half().double(), turn[:, hq:hq + hkv].half().double(), rows[:, hq + hkv:].half().double()
                w = torch.softmax(torch.einsum("hgd,lhd->hgl", qq.view(hkv, -1, HD), k) / HD ** 0.5, -1)
                want = torch.einsum("hgl,lhd->hgd", w, v).reshape(hq, HD)
                # a rounding of q or K to f16 may fall to the other side (f32 angles): 2^-10 of a score's 128 products
                assert float((out[at].double() - want).abs().max()) < 2e-3, (r, i)
                at += 1
        assert bool((out[at:] == 5).all())
        return plan

    step([96, 0, 0, 0, 0], None)                       # the shared prompt
    table[1:, :6] = table[0, :6]                       # four answers behind it
    lens = lens.clone()
    lens[1:] = 96
    for r in range(1, B):
        story[r] = list(story[0])
    step([1, 1, 30, 1, 17], None)                      # chunks, a group per request
    for _ in range(20):                                # single tokens, one group
        step([1] * B, ([0, B], [6]))
    step([0, 1, -1, 1, 0], ([0, 2], [6]))              # one ends
    assert int(lens[2]) == 0
    lens = lens.clone()
    lens[2] = 96                                       # another takes its place behind the prompt
    story[2] = list(story[0][:96])
    for _ in range(3):
        step([1, 1, 40, 1, 1], ([0, 2, 42, 44], [6, 6, 6]))
    pool.free()


def test_long_sums_of_f32_results(ctx):
    """Many blocks to a CTA: the MMAs cut the sums they add to, 2^-23 of them at most, and a sum is added to 32 times before it is rounded
    to nearest in memory (without that the error grows with the blocks, beyond 10^-5 here); 2^-21 for scores and weights."""
    import torch
    b = Batch(ctx, [(3000, [48000 - i for i in range(40)])], 32, 8)
    a, kw = b.args()
    got = ctx.attn_shared(*a, **kw)
    want, _ = b.exact()
    assert float((got.double() - want).norm() / want.norm()) < 32 * 2.0 ** -23 + 2.0 ** -21
    b.pool.free()


def test_many_rows(ctx):
    """30000 rows in 700 groups, some without pages, some without company, against the decode attention of every row by itself."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(6)
    rows, pages, width, hkv = 30000, 4000, 9, 2
    pool = ctx.kv_pool(pages, hkv)
    data = pool.tensor()
    data.copy_(torch.randn(data.shape, generator=g, device="cuda").half())
    table = torch.randint(0, pages, (rows, width), generator=g, device="cuda", dtype=torch.int32)
    first = torch.cat([torch.tensor([0], device="cuda"), torch.randint(0, rows + 1, (699,), generator=g, device="cuda").sort().values, torch.tensor([rows], device="cuda")])
    shared = torch.randint(-3, width + 1, (700,), generator=g, device="cuda").clamp(min=0)
    of = torch.searchsorted(first[1:], torch.arange(rows, device="cuda"), right=True)
    head = table[first[:-1].clamp(max=rows - 1)][of]  # every row begins with its group's first pages
    table = torch.where(torch.arange(width, device="cuda") < shared[of][:, None], head, table).contiguous()
    lens = torch.randint(0, width * PAGE + 1, (rows,), generator=g, device="cuda", dtype=torch.int32)
    lens[::7] = 0
    q = torch.randn(rows, 4, HD, generator=g, device="cuda").half()
    i32 = torch.int32
    for window in (0, 30):
        got = ctx.attn_shared(pool, q, table, lens, first.to(i32), shared.to(i32), window=window)
        want = ctx.attn_decode(pool, q, table, lens, window=window)
        assert float((got - want).abs().max()) < 1e-4 * float(want.abs().max())
    ctx.device_status()
    pool.free()


def test_contexts_of_two_threads(ctx):
    """Two contexts on one device, each with its stream and thread, over one pool."""
    import threading
    import torch
    from cyb_b200 import qeng
    b = Batch(ctx, [behind(50, [7 * i for i in range(40)]), (12, list(range(1, 193)))], 16, 4)
    a, kw = b.args()
    want, mag = b.exact()
    torch.cuda.synchronize()
    outs, bad = [[], []], []

    def work(k):
        try:
            c = qeng.Context(0)
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(15):
                    outs[k].append(c.attn_shared(*a, **kw))
                torch.cuda.current_stream().synchronize()
            c.device_status()
            c.close()
        except Exception as e:  # noqa: BLE001
            bad.append(e)
    threads = [threading.Thread(target=work, args=(k,)) for k in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad, bad
    for got in outs[0] + outs[1]:
        assert torch.equal(got, outs[0][0])
    assert_near(outs[0][0], want, mag)
    b.pool.free()
