"""The page planner and the rotary append by slots (through the C ABI) against plain restatements."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
PAGE, HD = 16, 128


def _t(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def plan_by_hand(lens, add, keep, table, ring, ends, cap, pages):
    """Request by request, token by token."""
    lens, table, ring = [int(x) for x in lens], table.copy(), ring.copy()
    R, width, size = len(lens), table.shape[1], len(ring)
    head, tail = int(ends[0]), int(ends[1])
    starts, toks, taken, freed, status, full = [0], [], 0, [], 0, False
    new_lens = list(lens)
    for r in range(R):
        n, a = lens[r], int(add[r])
        if not 0 <= n <= width * PAGE or (a > 0 and n + a > width * PAGE):
            status = 2
        elif a < 0:
            new_lens[r] = 0
            freed += [table[r, j] for j in range(min(max(0, int(keep[r])) if keep is not None else 0, -(-n // PAGE)), -(-n // PAGE))]
        elif a > 0 and not full:
            need = -(-(n + a) // PAGE) - -(-n // PAGE)
            if len(toks) + a > cap or taken + need > tail - head:
                full = True
            else:
                for j in range(need):
                    table[r, -(-n // PAGE) + j] = ring[(head + taken + j) % size]
                taken += need
                for p in range(n, n + a):
                    pid = int(table[r, p // PAGE])
                    toks.append((pid * PAGE + p % PAGE if 0 <= pid < pages else -1, p, p + 1, r))
                new_lens[r] = n + a
        starts.append(len(toks))
    for i, pid in enumerate(freed):
        ring[(tail + i) % size] = pid
    toks += [(-1, 0, 0, -1)] * (cap - len(toks))
    s = np.array(toks, np.int32).reshape(cap, 4).T
    return dict(starts=np.array(starts, np.int32), slots=s[0], pos=s[1], seen=s[2], rows=s[3], lens=np.array(new_lens, np.int32),
                ends=np.array([head + taken, tail + len(freed)], np.int64), table=table, ring=ring), status


def make_plan(rng, R, width, most_add, ends_share=0.1, spare=50, with_keep=False):
    lens = rng.integers(0, width * PAGE + 1, R).astype(np.int32)
    lens[rng.random(R) < 0.2] = 0
    room = width * PAGE - lens
    add = np.minimum(rng.integers(0, most_add + 1, R), room).astype(np.int32)
    add[rng.random(R) < ends_share] = -1
    held = -(-lens // PAGE)
    pages = int(held.sum()) + spare
    ids = rng.permutation(pages).astype(np.int32)
    table = np.full((R, width), 7, np.int32)
    at = 0
    for r in range(R):
        table[r, :held[r]] = ids[at:at + held[r]]
        at += held[r]
    size = pages + int(rng.integers(0, 5))
    head = int(rng.integers(0, 3 * size))
    ring = np.full(size, -5, np.int32)
    for i in range(spare):
        ring[(head + i) % size] = ids[at + i]
    keep = rng.integers(0, width + 2, R).astype(np.int32) if with_keep else None
    return lens, add, keep, table, ring, np.array([head, head + spare], np.int64), pages


def check_plan(ctx, lens, add, keep, table, ring, ends, pages, cap, in_place=False, stream=None):
    import torch
    pool = ctx.kv_pool(pages, 1)
    want, status = plan_by_hand(lens, add, keep, table, ring, ends, cap, pages)
    tl, ta, tt, tr, te = _t(lens), _t(add), _t(table), _t(ring), _t(ends)
    buf = ctx.kv_plan_buffers(len(lens), cap)
    if in_place:
        buf = buf._replace(lens=tl, ends=te)
    got = ctx.kv_plan(pool, tl, ta, tt, tr, te, cap, keep=None if keep is None else _t(keep), out=buf)
    torch.cuda.synchronize()
    for k in ("starts", "slots", "pos", "seen", "rows", "lens", "ends"):
        assert np.array_equal(getattr(got, k).cpu().numpy(), want[k]), k
    assert np.array_equal(tt.cpu().numpy(), want["table"])
    assert np.array_equal(tr.cpu().numpy(), want["ring"])
    if not in_place:
        assert np.array_equal(tl.cpu().numpy(), lens) and np.array_equal(te.cpu().numpy(), ends)
    pool.free()
    return status


@pytest.mark.parametrize("R,width,most_add,cap,spare", [
    (1, 1, 1, 1, 1), (1, 1, 16, 5, 3), (1, 300, 4000, 4097, 400), (2, 4, 40, 100, 1), (33, 5, 3, 64, 50), (64, 256, 1, 64, 64),
    (300, 40, 70, 8192, 2000), (300, 40, 70, 5000, 2000), (1000, 9, 130, 70001, 9000), (1024, 2, 1, 1024, 0), (1025, 3, 30, 9000, 700),
    (8192, 2, 9, 40000, 5000)])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan(ctx, R, width, most_add, cap, spare, in_place):
    """From one request to the most there may be, in one CTA and in clusters; several run out of tokens or pages on the way."""
    rng = np.random.default_rng(R * 7 + cap)
    for with_keep in (False, True):
        lens, add, keep, table, ring, ends, pages = make_plan(rng, R, width, most_add, spare=spare, with_keep=with_keep)
        assert check_plan(ctx, lens, add, keep, table, ring, ends, pages, cap, in_place) == 0
    ctx.device_status()


def test_plan_edges(ctx):
    """Nothing to do; a full table row; exactly the tokens and pages there are; one too many of either."""
    ring, ends = np.arange(10, 14, dtype=np.int32), np.array([2, 6], np.int64)
    table = np.arange(9, dtype=np.int32).reshape(3, 3)
    i = lambda *v: np.array(v, np.int32)  # noqa: E731
    for lens, add, cap in [(i(0, 0, 0), i(0, 0, 0), 1), (i(48, 32, 17), i(0, 16, 31), 47), (i(0, 0, 48), i(32, 32, 0), 64), (i(0, 0, 47), i(32, 32, 1), 64),
                           (i(0, 16, 0), i(48, 17, 1), 100), (i(16, 15, 0), i(0, 1, 48), 49), (i(16, 48, 33), i(-1, -7, -2147483648), 8)]:
        if (add < 0).any():
            e = np.array([4, 4], np.int64)
            r = np.full(9, -3, np.int32)
        else:
            e, r = ends, ring
        assert check_plan(ctx, lens, add, None, table, r, e, 16, cap) == 0, (lens, add)
        assert check_plan(ctx, lens, add, None, table, r, e, 16, cap, in_place=True) == 0, (lens, add)
    ctx.device_status()


def test_plan_reports_what_makes_no_sense(ctx):
    from cyb_b200 import qeng
    i = lambda *v: np.array(v, np.int32)  # noqa: E731
    ring, ends = np.arange(6, 12, dtype=np.int32), np.array([0, 6], np.int64)
    table = np.arange(6, dtype=np.int32).reshape(3, 2)
    # requests that outgrow their rows, or have lengths that cannot be: the others are served
    assert check_plan(ctx, i(30, -1, 5), i(3, 4, 2), None, table, ring, ends, 12, 16) == 2
    with pytest.raises(qeng.QengError, match="status 2"):
        ctx.device_status()
    assert check_plan(ctx, i(33, 2147483647, 5), i(-1, -1, 2147483647), None, table, ring, ends, 12, 16) == 2
    with pytest.raises(qeng.QengError, match="status 2"):
        ctx.device_status()
    # page ids outside the pool, in the table and in the ring: slots of -1
    bad = table.copy()
    bad[0, 0] = -2
    check_plan(ctx, i(3, 0, 16), i(2, 1, 5), None, bad, i(8, 99, 10, 11, 7, 6), ends, 12, 16)
    with pytest.raises(qeng.QengError, match="status 1"):
        ctx.device_status()
    # counters out of order, or more pages than the ring holds: nothing is taken or given, lengths stay
    pool = ctx.kv_pool(12, 1)
    for e, add in ((i(5, 3), i(1, 1, -1)), (i(-4, 0), i(1, 1, -1)), (i(0, 7), i(1, 1, 1)), (i(0, 6), i(0, 0, -1))):
        tt, tr = _t(table), _t(ring)
        p = ctx.kv_plan(pool, _t(i(0, 16, 20)), _t(add), tt, tr, _t(e.astype(np.int64)), 8)
        assert p.lens.tolist() == [0, 16, 20] and p.ends.tolist() == e.tolist() and p.starts.tolist() == [0] * 4
        assert np.array_equal(tt.cpu().numpy(), table) and np.array_equal(tr.cpu().numpy(), ring)
        with pytest.raises(qeng.QengError, match="status 6"):
            ctx.device_status()
    pool.free()


def test_plan_in_a_graph_and_beside_others(ctx):
    """A captured step that updates its own lengths and counters, replayed on another stream while plans of others run."""
    import torch
    rng = np.random.default_rng(4)
    R, width, steps = 50, 30, 40
    lens = rng.integers(0, 200, R).astype(np.int32)
    held = -(-lens // PAGE)
    pages = int(held.sum()) + R * 4
    ids = rng.permutation(pages).astype(np.int32)
    table = np.zeros((R, width), np.int32)
    at = 0
    for r in range(R):
        table[r, :held[r]] = ids[at:at + held[r]]
        at += held[r]
    ring = np.concatenate([ids[at:], np.zeros(at, np.int32)])
    ends = np.array([0, pages - at], np.int64)
    pool = ctx.kv_pool(pages, 1)
    tl, ta, tt, tr, te = _t(lens), _t(np.ones(R, np.int32)), _t(table), _t(ring), _t(ends)
    buf = ctx.kv_plan_buffers(R, 64)._replace(lens=tl, ends=te)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ctx.kv_plan(pool, tl, ta, tt, tr, te, 64, out=buf)
    other = make_plan(rng, 300, 9, 40, spare=900)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for k in range(steps):
        with torch.cuda.stream(side):
            g.replay()
        if k % 8 == 0:
            check_plan(ctx, *other, 6000)
    torch.cuda.synchronize()
    for _ in range(steps):
        w, status = plan_by_hand(lens, np.ones(R, np.int32), None, table, ring, ends, 64, pages)
        lens, table, ring, ends = w["lens"], w["table"], w["ring"], w["ends"]
    assert np.array_equal(tl.cpu().numpy(), lens) and np.array_equal(tt.cpu().numpy(), table) and np.array_equal(te.cpu().numpy(), ends)
    assert np.array_equal(buf.slots.cpu().numpy(), w["slots"])
    pool.free()
    ctx.device_status()


def test_plan_refusals(ctx):
    import torch
    from cyb_b200 import qeng
    pool = ctx.kv_pool(4, 1)
    z = torch.zeros(8200, dtype=torch.int32, device="cuda")
    e = torch.zeros(3, dtype=torch.int64, device="cuda")

    def call(R=1, max_pages=1, ring=8, cap=1, ends=e.data_ptr(), slots=z.data_ptr()):
        p = z.data_ptr()
        return qeng._lib.qeng_kv_plan(ctx.h, pool.h, R, p, p, None, p, max_pages, p, ring, ends, p, e.data_ptr(), p, slots, p, p, p, cap, None)
    for kw, code in [(dict(R=0), -1), (dict(R=-1), -1), (dict(max_pages=0), -1), (dict(ring=0), -1), (dict(cap=0), -1), (dict(slots=None), -1),
                     (dict(R=8193), -2), (dict(cap=(1 << 30) + 1), -2), (dict(max_pages=(1 << 26) + 1), -2), (dict(ring=(1 << 30) + 1), -2),
                     (dict(ends=e.data_ptr() + 4), -3)]:
        assert call(**kw) == code, kw
    pool.free()
    ctx.device_status()


# ---- the append ------------------------------------------------------------------------------------------------------------
def appended(x, pos, slots, base, hq, hkv, qg, kg, eps, pool):
    """In 64 bits: (q [T, Hq, 128], pool [pages, Hkv, 2, 16, 128]) before their rounding to f16."""
    t = len(x)
    x = x.astype(np.float64).reshape(t, hq + 2 * hkv, HD)
    ang = pos.astype(np.float64)[:, None] * float(base) ** (-2.0 * np.arange(64) / HD)
    c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
    heads = x[:, :hq + hkv].copy()
    if qg is not None:
        heads /= np.sqrt((heads ** 2).mean(-1, keepdims=True) + eps)
        heads[:, :hq] *= qg.astype(np.float64)
        heads[:, hq:] *= kg.astype(np.float64)
    a, b = heads[..., :64], heads[..., 64:]
    heads = np.concatenate([a * c - b * s, b * c + a * s], -1)
    pool = pool.astype(np.float64)
    for i in range(t):
        if slots[i] >= 0:
            pool[slots[i] // PAGE, :, 0, slots[i] % PAGE] = heads[i, hq:]
            pool[slots[i] // PAGE, :, 1, slots[i] % PAGE] = x[i, hq + hkv:]
    return heads[:, :hq], pool


def assert_half(got, want, size, far):
    """Half a step of f16, and what f32 arithmetic on values up to `size` may be off by (16 roundings of 2^-24; angles: 8 roundings of
    2^-53 of the position)."""
    d = np.abs(got.astype(np.float64) - want)
    assert np.all(d <= 2.0 ** -11 * np.abs(want) + 2.0 ** -25 + size * (2.0 ** -20 + far * 2.0 ** -50)), d.max()


@pytest.mark.parametrize("dt", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("t,hq,hkv,norm,far", [(1, 32, 8, False, 0), (1, 1, 1, True, 2 ** 31 - 1), (5, 5, 5, False, 100), (7, 12, 4, True, 10 ** 6), (64, 28, 4, False, 131072),
                                               (33, 40, 40, True, 5000), (300, 8, 1, True, 77), (129, 32, 32, False, 999999)])
def test_append(ctx, dt, t, hq, hkv, norm, far):
    import torch
    rng = np.random.default_rng(t * 100 + hq)
    pages = t // PAGE + 5
    width = (hq + 2 * hkv) * HD
    x = torch.from_numpy(rng.standard_normal((t, width + 16), dtype=np.float32)).cuda().to(getattr(torch, dt))[:, :width]  # strided rows
    pos = np.maximum(far - np.arange(t)[::-1], 0).astype(np.int32)
    slots = rng.permutation(pages * PAGE)[:t].astype(np.int32)
    if t > 4:
        slots[[1, t - 1]] = -1  # padding
    qg, kg = (1 + 0.2 * rng.standard_normal((2, HD))).astype(np.float32) if norm else (None, None)
    pool = ctx.kv_pool(pages, hkv)
    before = rng.standard_normal((pages, hkv, 2, PAGE, HD), dtype=np.float32).astype(np.float16)
    pool.tensor().copy_(_t(before))
    out = torch.full((t, hq * HD + 8), 7.0, dtype=torch.float16, device="cuda")
    view = out[:, :hq * HD].view(t, hq, HD)
    base = 1e6 if far > 1000 else 1e4
    ctx.rope_append(pool, x, _t(pos), _t(slots), base, q_gain=None if qg is None else _t(qg), k_gain=None if kg is None else _t(kg), eps=1e-6, out=view)
    q, want = appended(x.float().cpu().numpy(), pos, slots, base, hq, hkv, qg, kg, 1e-6, before)
    got = out.cpu().numpy()
    live = slots >= 0
    assert np.all(got[:, hq * HD:] == 7) and np.all(got[~live] == 7)
    size = 8.0 * (1.8 if norm else 1.0)
    assert_half(got[live, :hq * HD].reshape(-1, hq, HD), q[live], size, far)
    assert_half(pool.tensor().cpu().numpy(), want, size, far)
    pool.free()
    ctx.device_status()


def test_append_agrees_with_the_small_operators(ctx):
    """The rows that qeng_rope and qeng_kv_append leave."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(5)
    b, hq, hkv = 9, 8, 2
    x = torch.randn(b, (hq + 2 * hkv) * HD, device="cuda", generator=g)
    pos = torch.tensor([0, 1, 15, 16, 17, 31, 63, 64, 79], dtype=torch.int32, device="cuda")
    table = torch.randperm(b * 5, device="cuda", generator=g).to(torch.int32).view(b, 5)
    pools = [ctx.kv_pool(b * 5, hkv) for _ in range(2)]
    turned = ctx.rope_(x[:, :(hq + hkv) * HD].reshape(b, hq + hkv, HD).contiguous(), pos, 1e4)
    ctx.kv_append(pools[0], turned[:, hq:].contiguous(), x[:, (hq + hkv) * HD:].contiguous(), table, pos)
    slots = table[torch.arange(b, device="cuda"), pos // PAGE] * PAGE + pos % PAGE
    q = ctx.rope_append(pools[1], x, pos, slots, 1e4)
    for got, want in ((q, turned[:, :hq]), (pools[1].tensor(), pools[0].tensor())):
        d = (got.float() - want.float()).abs()
        assert bool((d <= 2.0 ** -10 * want.float().abs() + 2.0 ** -17).all()), float(d.max())
    for p in pools:
        p.free()


def test_append_reports_slots_outside_the_pool(ctx):
    import torch
    from cyb_b200 import qeng
    pool = ctx.kv_pool(2, 1)
    x = torch.ones(3, 3 * HD, device="cuda")
    q = torch.zeros(3, 1, HD, dtype=torch.float16, device="cuda")
    ctx.rope_append(pool, x, _t(np.zeros(3, np.int32)), _t(np.array([31, 32, 2 ** 31 - 1], np.int32)), 1e4, out=q)
    with pytest.raises(qeng.QengError, match="status 1"):
        ctx.device_status()
    assert bool((q[0] == 1).all()) and bool((q[1:] == 0).all())
    want = torch.zeros_like(pool.tensor())
    want[1, :, :, 15] = 1
    assert torch.equal(pool.tensor(), want)
    pool.free()


def test_append_refusals(ctx):
    import torch
    from cyb_b200 import qeng
    pool = ctx.kv_pool(2, 2)
    x = torch.zeros(4, 6 * HD, device="cuda")
    q = torch.zeros(4, 2 * HD, dtype=torch.float16, device="cuda")
    z = torch.zeros(64, dtype=torch.int32, device="cuda")

    def call(x_=x.data_ptr(), dt=0, T=4, ldx=6 * HD, hq=2, qg=None, kg=None, pos=z.data_ptr(), base=1e4, out=q.data_ptr(), ldq=2 * HD):
        return qeng._lib.qeng_rope_append(ctx.h, pool.h, x_, dt, T, ldx, hq, qg, kg, 1e-5, pos, z.data_ptr(), base, out, ldq, None)
    for kw, code in [(dict(x_=None), -1), (dict(dt=3), -1), (dict(dt=-1), -1), (dict(base=0.0), -1), (dict(base=math.nan), -1), (dict(pos=None), -1),
                     (dict(qg=x.data_ptr()), -1), (dict(kg=x.data_ptr()), -1), (dict(T=0), -2), (dict(hq=0), -2), (dict(hq=3), -2),
                     (dict(ldx=6 * HD - 4), -2), (dict(ldq=2 * HD - 8), -2), (dict(ldx=6 * HD + 2), -3), (dict(ldq=2 * HD + 4), -3),
                     (dict(x_=x.data_ptr() + 4), -3), (dict(out=q.data_ptr() + 2), -3)]:
        assert call(**kw) == code, kw
    pool.free()
    ctx.device_status()


def test_append_of_a_cache_past_32_bits(ctx):
    """Slots whose values lie beyond 2^32 bytes and 2^31 values of the pool."""
    import torch
    pages, hkv = 70000, 8  # 4.6 GB
    pool = ctx.kv_pool(pages, hkv)
    x = torch.randn(3, (8 + 2 * hkv) * HD, device="cuda")
    slots = np.array([pages * PAGE - 1, 65537 * PAGE + 3, 0], np.int32)
    ctx.rope_append(pool, x, _t(np.zeros(3, np.int32)), _t(slots), 1e4)
    d = pool.tensor()
    for i, s in enumerate(slots):
        assert torch.equal(d[s // PAGE, :, :, s % PAGE].transpose(0, 1).reshape(-1), x[i, 8 * HD:].half())
    assert int((d[65000:] != 0).sum()) <= 2 * 2 * hkv * HD
    pool.free()
    ctx.device_status()


def test_a_view_keeps_its_pool(ctx):
    import gc
    import weakref
    pool = ctx.kv_pool(3, 1)
    view, alive = pool.tensor()[1:], weakref.ref(pool)
    del pool
    gc.collect()
    assert alive() is not None
    del view
    gc.collect()
    assert alive() is None
