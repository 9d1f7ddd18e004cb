"""What the serving operators of qeng are measured on: the page planner (block tables and slot maps from request lengths), the rotary
append through a slot map, and the attention of rows that share leading pages.

`run` computes them in plain torch operations, or through the framework's entry points where `own` is set.  Lengths follow from a case
alone (their order from the seed), so that `work` knows them; values, page ids and token order come from the seed."""
import math

import torch

own = False
HD, PAGE = 128, 16
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_ctx = []


def _context():
    """The engine context of this process (a server keeps one per GPU)."""
    from cyb_b200 import qeng
    if not _ctx:
        _ctx.append(qeng.Context(torch.cuda.current_device()))
    return _ctx[0]


# ---- cases ----------------------------------------------------------------------------------------------------------
def listed():
    def attn(name, **kw):
        return {"name": name, "op": "attn", "heads": 32, "kv_heads": 8, "groups": 1, "batch": 1, "prefix": 0, "own": 0, "cached": 0, "prompts": 0,
                "tokens": 0, "softcap": 0.0, "window": 0, "out": "bf16", **kw}

    def append(name, **kw):
        return {"name": name, "op": "append", "heads": 32, "kv_heads": 8, "tokens": 1, "dtype": "f32", "norm": False, "base": 10000.0, "far": 4096, **kw}

    def plan(name, **kw):
        return {"name": name, "op": "plan", "requests": 1, "chunk": 0, "chunked": 0, "released": 0, "idle": 0, "cached": 4096, "capacity": 1, **kw}

    return [
        # a decode step of a full server: every request gets one token
        plan("plan-decode64", requests=64, capacity=64),
        # a mixed step in a buffer of fixed size: 12 prompt chunks, 20 requests that end, 9 that wait, the others decode
        plan("plan-mixed300", requests=300, chunk=512, chunked=12, released=20, idle=9, capacity=8192),
        # many prompts at once
        plan("plan-prompts1000", requests=1000, chunk=128, chunked=1000, cached=2048, capacity=131072),
        # one token of one sequence: latency
        append("append-decode1"),
        # a chunk of an odd size, normed heads, positions far out, 16-bit rows
        append("append-chunk777", heads=12, kv_heads=4, tokens=777, dtype="bf16", norm=True, base=1000000.0, far=200000),
        # a long prompt straight from the f32 matmul
        append("append-prompt8192", tokens=8192),
        # few sequences behind a short system prompt: latency
        attn("shared-4x512", batch=4, prefix=512, own=64, out="f32"),
        # a small batch behind a long document, f32 results
        attn("shared-16x4096", batch=16, prefix=4096, own=512, out="f32"),
        # three system prompts, soft-capped scores, a window that ends inside the prefix, an odd number of pages and heads
        attn("shared-37x1000-window", batch=37, groups=3, heads=12, kv_heads=4, prefix=1000, own=700, softcap=50.0, window=1100, out="f16"),
        # a busy server: memory and tensor cores in balance
        attn("shared-64x16384", batch=64, prefix=16384, own=1024),
        # the largest: 256 answers about one long document
        attn("shared-256x16384", batch=256, prefix=16384, own=256),
        # prompts of one to 2048 tokens behind cached ones: each a group whose rows share all pages
        attn("prompts-7x2048", prompts=7, tokens=2048, cached=1500, out="f16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = max((_attn_work(c)["flops"], _attn_work(c)["bytes"]) for c in listed() if c["op"] == "attn")
    op = rng.choice(["plan", "append", "attn", "attn", "attn", "prompt"])
    if op == "plan":
        n = _log(rng, 1, 1000)
        chunked = rng.randint(0, n) if rng.random() < 0.5 else rng.randint(0, min(n, 16))
        rest = n - chunked
        released = rng.randint(0, rest // 3)
        idle = rng.randint(0, (rest - released) // 3)
        return {"op": "plan", "requests": n, "chunk": _log(rng, 1, 128 if chunked > 64 else 1024), "chunked": chunked, "released": released, "idle": idle,
                "cached": _log(rng, 1, 4096), "capacity": _log(rng, n, 131072)}
    heads, kv_heads = rng.choice([(32, 8), (32, 8), (32, 32), (12, 4), (8, 1), (28, 4), (5, 5)])
    if op == "append":
        return {"op": "append", "heads": heads, "kv_heads": kv_heads, "tokens": _log(rng, 1, 8192 if heads + 2 * kv_heads <= 48 else 4096),
                "dtype": rng.choice(["f32", "f16", "bf16"]), "norm": rng.random() < 0.5, "base": rng.choice([10000.0, 1000000.0]), "far": _log(rng, 16, 1000000)}
    while True:
        c = {"op": "attn", "heads": heads, "kv_heads": kv_heads, "groups": 1, "batch": 1, "prefix": 0, "own": 0, "cached": 0, "prompts": 0, "tokens": 0,
             "softcap": rng.choice([0.0, 0.0, 0.0, 50.0]), "window": rng.choice([0, 0, 0, _log(rng, 16, 8192)]), "out": rng.choice(["f32", "f16", "bf16"])}
        if op == "prompt":
            c.update(prompts=rng.randint(1, 8), tokens=_log(rng, 1, 2048), cached=rng.choice([0, _log(rng, 1, 4096)]))
        else:
            c.update(batch=_log(rng, 1, 256), prefix=_log(rng, 1, 16384), own=_log(rng, 1, 1024))
            c.update(groups=rng.choice([1, 1, rng.randint(1, min(4, c["batch"]))]))
        w = _attn_work(c)
        if w["flops"] <= most[0] and w["bytes"] <= most[1]:
            return c


def _spread(n, top):
    """n lengths from 1 to `top`, spread evenly and out of order, `top` among them."""
    return [1 + int((top - 1) * (((i + 1) * 0.6180339887498949) % 1.0)) if i else top for i in range(n)] if top > 0 else [0] * n


def _attn_shape(case):
    """Groups of a case: (rows' lengths, shared pages) of each."""
    if case["prompts"]:
        got = []
        for t, c in zip(_spread(case["prompts"], case["tokens"]), _spread(case["prompts"], case["cached"])):
            got.append(([c + i + 1 for i in range(t)], (c + t + PAGE - 1) // PAGE))
        return got
    own_lens, pre = _spread(case["batch"], case["own"]), _spread(case["groups"], case["prefix"])
    got = []
    for g in range(case["groups"]):
        pages = pre[g] // PAGE
        got.append(([pages * PAGE + n for n in own_lens[g::case["groups"]]], pages))
    return got


def _attn_work(case):
    seen = read = rows = 0
    for lens, pages in _attn_shape(case):
        lo = [max(0, n - case["window"]) if case["window"] else 0 for n in lens]
        seen += sum(n - a for n, a in zip(lens, lo))
        end = min(pages * PAGE, max(lens))
        read += max(0, end - min(lo)) + sum(max(0, n - max(a, pages * PAGE)) for n, a in zip(lens, lo))
        rows += len(lens)
    size = 4 if case["out"] == "f32" else 2
    return {"bytes": read * case["kv_heads"] * 2 * HD * 2 + rows * case["heads"] * HD * (2 + size), "flops": 4 * HD * case["heads"] * seen}


def _plan_shape(case):
    """(cached tokens, tokens to add) of the requests."""
    n, c = case["requests"], case["chunked"]
    lens = [x - 1 if i % 7 == 0 else x for i, x in enumerate(_spread(n, case["cached"]))]
    add = _spread(c, case["chunk"]) + [-1] * case["released"] + [0] * case["idle"]
    return lens, add + [1] * (n - len(add))


def work(case):
    if case["op"] == "attn":
        return _attn_work(case)
    if case["op"] == "append":
        values = case["tokens"] * (case["heads"] + 2 * case["kv_heads"]) * HD
        return {"bytes": values * ((4 if case["dtype"] == "f32" else 2) + 2) + 8 * case["tokens"], "flops": 4 * values}
    lens, add = _plan_shape(case)
    pages = sum(-(-(n + a) // PAGE) - -(-n // PAGE) for n, a in zip(lens, add) if a > 0) + sum(-(-n // PAGE) for n, a in zip(lens, add) if a < 0)
    return {"bytes": 4 * (4 * case["capacity"] + 4 * case["requests"] + 1 + 2 * pages) + 32, "flops": 16 * case["capacity"]}


# ---- what a server holds before the call -------------------------------------------------------------------------------
def _pool(gen, pages, kv_heads, fill):
    """A cache of `pages` pages as the framework keeps it, or as a plain tensor; normal values where it is to be read."""
    if own:
        handle = _context().kv_pool(pages, kv_heads)
        data = handle.tensor()
    else:
        handle = None
        data = torch.zeros((pages, kv_heads, 2, PAGE, HD), dtype=torch.float16, device="cuda")
    if fill:
        flat = data.view(-1)
        for at in range(0, flat.numel(), 1 << 28):
            part = flat[at:at + (1 << 28)]
            part.copy_(torch.randn(part.shape, generator=gen, device="cuda", dtype=torch.float16))
    return handle, data


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = {"case": case}
    if case["op"] == "attn":
        shape = _attn_shape(case)
        pages = [(p, max(-(-n // PAGE) for n in lens)) for lens, p in shape]
        width = max(1, max(m for _, m in pages))
        prompt = bool(case["prompts"])
        count = sum(p if prompt else p + sum(max(0, -(-n // PAGE) - p) for n in lens) for lens, p in shape)
        s["handle"], s["pool"] = _pool(gen, max(1, count), case["kv_heads"], True)
        ids = torch.randperm(max(1, count), generator=gen, device="cuda").to(torch.int32)
        tables, all_lens, rows, at = [], [], [], 0
        for g, (lens, p) in enumerate(shape):
            order = list(range(len(lens))) if prompt else torch.randperm(len(lens), generator=gen, device="cuda").tolist()
            lens = [lens[i] for i in order]
            shape[g] = (lens, p)
            all_lens += lens
            t = torch.zeros((1 if prompt else len(lens), width), dtype=torch.int32)
            t[:, :p] = torch.arange(at, at + p)
            at += p
            if not prompt:
                for i, n in enumerate(lens):
                    m = max(0, -(-n // PAGE) - p)
                    t[i, p:p + m] = torch.arange(at, at + m)
                    at += m
            rows += [g] * len(lens)
            tables.append(t)
        s["table"] = ids[torch.cat(tables).cuda().long()].contiguous()
        s["rows"] = _ints(rows) if prompt else None
        s["lens"] = _ints(all_lens)
        first = [0]
        for lens, _ in shape:
            first.append(first[-1] + len(lens))
        s["first"], s["shared"] = _ints(first), _ints([p for _, p in shape])
        s["shape"] = [(len(lens), p, 0 if prompt else max(0, max(-(-n // PAGE) for n in lens) - p)) for lens, p in shape]
        s["q"] = torch.randn((len(all_lens), case["heads"], HD), generator=gen, device="cuda", dtype=torch.float32).half()
    elif case["op"] == "append":
        n = case["tokens"]
        width = (case["heads"] + 2 * case["kv_heads"]) * HD
        s["x"] = torch.randn((n, width), generator=gen, device="cuda").to(DTYPES[case["dtype"]])
        # tokens of one sequence that ends at position `far` or later, in scattered pages
        p0 = max(0, case["far"] - n)
        pos = torch.arange(p0, p0 + n, device="cuda")
        count = (p0 + n - 1) // PAGE - p0 // PAGE + 1
        s["handle"], s["pool"] = _pool(gen, count, case["kv_heads"], False)
        ids = torch.randperm(count, generator=gen, device="cuda")
        s["pos"] = pos.to(torch.int32)
        s["slots"] = (ids[pos // PAGE - p0 // PAGE] * PAGE + pos % PAGE).to(torch.int32)
        s["gains"] = [1 + 0.1 * torch.randn(HD, generator=gen, device="cuda") for _ in range(2)] if case["norm"] else [None, None]
    else:
        lens, add = _plan_shape(case)
        n = len(lens)
        order = torch.randperm(n, generator=gen, device="cuda").tolist()
        lens, add = [lens[i] for i in order], [add[i] for i in order]
        width = max(max(-(-(a + max(b, 0)) // PAGE) for a, b in zip(lens, add)), 1)
        held = [-(-a // PAGE) for a in lens]
        spare = sum(-(-(a + max(b, 0)) // PAGE) for a, b in zip(lens, add)) - sum(held) + 17
        count = sum(held) + spare
        ids = torch.randperm(count, generator=gen, device="cuda").to(torch.int32)
        t = torch.zeros((n, width), dtype=torch.int64)
        at = 0
        for i, h in enumerate(held):
            t[i, :h] = torch.arange(at, at + h)
            at += h
        s["table"] = ids[t.cuda()].contiguous()
        s["lens"], s["add"] = _ints(lens), _ints(add)
        # the free pages lie across the ring's end
        head = count - spare // 2
        ring = torch.full((count,), -1, dtype=torch.int32, device="cuda")
        ring[(head + torch.arange(spare, device="cuda")) % count] = ids[at:]
        s["ring"], s["ends"] = ring, torch.tensor([head, head + spare], dtype=torch.int64, device="cuda")
        s["handle"] = None
        if own:
            s["handle"] = _context().kv_pool(count, 1)
            s["out"] = _context().kv_plan_buffers(n, case["capacity"])
    return s


# ---- one pass ------------------------------------------------------------------------------------------------------------
def run(s):
    op = s["case"]["op"]
    return _run_attn(s) if op == "attn" else _run_append(s) if op == "append" else _run_plan(s)


def _run_plan(s):
    lens, add, table, ring, ends, cap = s["lens"], s["add"], s["table"], s["ring"], s["ends"], s["case"]["capacity"]
    if own:
        p = _context().kv_plan(s["handle"], lens, add, table, ring, ends, cap, out=s["out"])
        return {"starts": p.starts, "slots": p.slots, "pos": p.pos, "seen": p.seen, "rows": p.rows, "lens": p.lens, "ends": p.ends, "table": table, "ring": ring}
    n, width, size = lens.numel(), table.shape[1], ring.numel()
    held = (lens + PAGE - 1) // PAGE
    wish = torch.where((add > 0) & (lens + add <= width * PAGE), add, 0)
    need = (lens + wish + PAGE - 1) // PAGE - held
    fits = (wish.cumsum(0) <= cap) & (need.cumsum(0) <= ends[1] - ends[0])
    wish, need = torch.where(fits, wish, 0), torch.where(fits, need, 0)
    after = wish.cumsum(0)
    starts = torch.cat([after.new_zeros(1), after])
    taken = need.cumsum(0) - need
    gone = torch.where(add < 0, held, 0)
    freed = gone.cumsum(0) - gone
    # pages: new ones from the ring's head, those of ended requests behind its tail
    j = torch.arange(width, device=lens.device)
    k = j - held[:, None]
    table = torch.where((k >= 0) & (k < need[:, None]), ring[(ends[0] + taken[:, None] + k) % size], table)
    to = torch.where(j < gone[:, None], (ends[1] + freed[:, None] + j) % size, size)
    ring = torch.cat([ring, ring.new_zeros(1)]).scatter(0, to.reshape(-1), table.reshape(-1))[:size]
    # tokens
    t = torch.arange(cap, device=lens.device)
    live = t < starts[n]
    r = torch.searchsorted(after, t, right=True).clamp(max=n - 1)
    p = torch.where(live, lens[r] + t - starts[r], 0)
    slots = torch.where(live, table[r, p // PAGE] * PAGE + p % PAGE, -1)
    i32 = torch.int32
    return {"starts": starts.to(i32), "slots": slots.to(i32), "pos": p.to(i32), "seen": torch.where(live, p + 1, 0).to(i32), "rows": torch.where(live, r, -1).to(i32),
            "lens": torch.where(add < 0, 0, lens + wish).to(i32), "ends": ends + torch.stack([need.sum(), gone.sum()]), "table": table, "ring": ring}


def _run_append(s):
    c, x, pool, gains = s["case"], s["x"], s["pool"], s["gains"]
    if own:
        q = _context().rope_append(s["handle"], x, s["pos"], s["slots"], c["base"], q_gain=gains[0], k_gain=gains[1], eps=1e-6)
        return {"q": q, "pool": pool}
    n, hq, hkv = c["tokens"], c["heads"], c["kv_heads"]
    x = x.float().view(n, hq + 2 * hkv, HD)
    freq = c["base"] ** (-torch.arange(0, HD, 2, device="cuda", dtype=torch.float64) / HD)
    angle = s["pos"].double()[:, None] * freq
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turned(h, gain):
        if gain is not None:
            h = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + 1e-6) * gain
        a, b = h[..., :HD // 2], h[..., HD // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).half()

    q, k, v = turned(x[:, :hq], gains[0]), turned(x[:, hq:hq + hkv], gains[1]), x[:, hq + hkv:].half()
    slots = s["slots"].long()
    pool[slots // PAGE, :, 0, slots % PAGE] = k
    pool[slots // PAGE, :, 1, slots % PAGE] = v
    return {"q": q, "pool": pool}


def _run_attn(s):
    c = s["case"]
    if own:
        return _context().attn_shared(s["handle"], s["q"], s["table"], s["lens"], s["first"], s["shared"], rows=s["rows"], softcap=c["softcap"],
                                      window=c["window"], dtype=DTYPES[c["out"]])
    hkv, grp = c["kv_heads"], c["heads"] // c["kv_heads"]
    out, at = [], 0
    for n, pages, more in s["shape"]:
        q = s["q"][at:at + n].float().view(n, hkv, grp, HD) * HD ** -0.5
        lens = s["lens"][at:at + n, None]
        r = at if s["rows"] is None else s["rows"][at].long()
        kv = s["pool"][s["table"][r, :pages].long()]  # [pages, kv heads, 2, 16, dims]
        k, v = (kv[:, :, i].transpose(0, 1).reshape(hkv, pages * PAGE, HD).float() for i in range(2))
        scores = torch.einsum("nhgd,hld->nhgl", q, k)
        if more:  # every row's own pages
            kv = s["pool"][s["table"][at:at + n, pages:pages + more].long()]
            ko, vo = (kv[:, :, :, i].transpose(1, 2).reshape(n, hkv, more * PAGE, HD).float() for i in range(2))
            scores = torch.cat([scores, torch.einsum("nhgd,nhld->nhgl", q, ko)], -1)
        if c["softcap"]:
            scores = c["softcap"] * torch.tanh(scores / c["softcap"])
        j = torch.arange(scores.shape[-1], device="cuda")
        keep = j < lens
        if c["window"]:
            keep &= j >= lens - c["window"]
        scores.masked_fill_(~keep[:, None, None], -math.inf)
        p = torch.exp(scores - scores.amax(-1, keepdim=True))
        o = torch.einsum("nhgl,hld->nhgd", p[..., :pages * PAGE], v)
        if more:
            o += torch.einsum("nhgl,nhld->nhgd", p[..., pages * PAGE:], vo)
        out.append((o / p.sum(-1, keepdim=True)).reshape(n, hkv * grp, HD))
        at += n
    return torch.cat(out).to(DTYPES[c["out"]])


# ---- 64 bits -------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers
    s = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "append":
        hq, hkv = case["heads"], case["kv_heads"]
        q = torch.empty((case["tokens"], hq, HD), dtype=f64, device="cuda")
        pool = s["pool"].double()
        for h in range(hq + 2 * hkv):
            x = s["x"][:, h * HD:(h + 1) * HD].to(f64)
            if h < hq + hkv:
                g = s["gains"][0 if h < hq else 1]
                if g is not None:
                    x = x / (x.pow(2).sum(1, keepdim=True) / HD + 1e-6).sqrt() * g.to(f64)
                z = torch.polar(torch.ones((), dtype=f64, device="cuda"), torch.outer(s["pos"].to(f64), torch.exp(-math.log(case["base"]) / 64 * torch.arange(64, dtype=f64, device="cuda"))))
                z = torch.complex(x[:, :64].contiguous(), x[:, 64:].contiguous()) * z
                x = torch.cat([z.real, z.imag], 1)
            if h < hq:
                q[:, h] = x
            else:
                page, at = s["slots"].long() // PAGE, s["slots"].long() % PAGE
                pool[page, (h - hq) % hkv, 0 if h < hq + hkv else 1, at] = x
        return {"q": q, "pool": pool}
    out = torch.empty(s["q"].shape, dtype=f64, device="cuda")
    hkv, grp = case["kv_heads"], case["heads"] // case["kv_heads"]
    rows = s["rows"].tolist() if s["rows"] is not None else range(len(out))
    kept = {}
    for t, (row, n) in enumerate(zip(rows, s["lens"].tolist())):
        a = max(0, n - case["window"]) if case["window"] else 0
        if row not in kept or s["rows"] is None:
            kv = s["pool"][s["table"][row].long()].to(f64).permute(2, 1, 0, 3, 4).reshape(2, hkv, -1, HD)
            kept = {row: kv}
        k, v = kept[row][0, :, a:n], kept[row][1, :, a:n]
        x = torch.bmm(s["q"][t].to(f64).view(hkv, grp, HD), k.transpose(1, 2)) / math.sqrt(HD)
        if case["softcap"]:
            x = torch.tanh(x / case["softcap"]) * case["softcap"]
        out[t] = torch.bmm(torch.softmax(x, -1), v).view(hkv * grp, HD)
    return out
