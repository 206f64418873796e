"""The paged KV-cache operators (tb2_paged_*, through toy_b200.paged) against
plain implementations: page accounting against host lists (whole numbers,
equal), appended rows against the f32 arithmetic they are defined by (equal
bits), attention against 64-bit sums within a bound derived from its
arithmetic (paged_ref.attend_bounds), and a run of all four as a serving loop
makes it."""
import math
import os
import sys

import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import paged_ref as R  # noqa: E402

pytestmark = pytest.mark.gpu


def i32(x, dev):
    import torch
    return torch.tensor(x, dtype=torch.int32, device=dev)


def no_error():
    from toy_b200._lib import lib
    assert lib().tb2_device_error() == 0


# ------------------------------------------------------------------ plan, release
def host_plan(lens, add, table, free, count, P, n_tokens):
    """(status, lens, table, count, taken, cu, slots, positions, requests) by lists."""
    n, width = len(lens), len(table[0])
    table = [list(r) for r in table]
    bad = 0
    for a, b in zip(lens, add):
        if a < 0 or b < 0:
            bad = max(bad, 4)
        elif -(-(a + b) // P) > width:
            bad = max(bad, 2)
    need = [0 if bad else -(-(a + b) // P) - -(-a // P) for a, b in zip(lens, add)]
    status = 4 if not 0 <= count <= len(free) else bad
    if not status and sum(add) > n_tokens:
        status = 3
    if not status and sum(need) > count:
        status = 1
    slots, pos, req = [-1] * n_tokens, [0] * n_tokens, [-1] * n_tokens
    if status:
        return status, lens, table, count, 0, [0] * (n + 1), slots, pos, req
    top, t, cu = count, 0, [0]
    for b in range(n):
        for i in range(need[b]):
            top -= 1
            table[b][-(-lens[b] // P) + i] = free[top]
        for i in range(add[b]):
            p = lens[b] + i
            slots[t], pos[t], req[t] = table[b][p // P] * P + p % P, p, b
            t += 1
        cu.append(t)
    return 0, [a + b for a, b in zip(lens, add)], table, top, count - top, cu, slots, pos, req


def scenario(seed, n, P, width, kind):
    import random
    r = random.Random(seed)
    most = width * P
    lens = [r.choice([0, r.randrange(0, most + 1), min(most, P * r.randrange(0, width + 1))]) for _ in range(n)]
    if kind == "decode":
        add = [1 if x < most else 0 for x in lens]
    elif kind == "none":
        add = [0] * n
    else:
        add = [r.choice([0, min(1, most - x), r.randrange(0, most - x + 1)]) for x in lens]
    n_pages = n * width + 3
    ids = list(range(n_pages))
    r.shuffle(ids)
    table, at = [], 0
    for x in lens:
        h = -(-x // P)
        table.append(ids[at:at + h] + [-7] * (width - h))
        at += h
    free = ids[at:]
    return lens, add, table, free, n_pages


@pytest.mark.parametrize("n,P,width,kind,room", [
    (1, 16, 4, "mixed", 0), (1, 1, 9, "decode", 3), (3, 7, 5, "mixed", 1), (16, 16, 8, "decode", 0),
    (33, 64, 3, "none", 5), (257, 16, 12, "mixed", 100), (1024, 8, 6, "mixed", 0), (1500, 24, 30, "mixed", 17),
    (5000, 16, 2, "decode", 0), (16384, 32, 1, "mixed", 9)])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan(cuda, n, P, width, kind, room, in_place):
    import torch
    from toy_b200 import paged
    lens, add, table, free, n_pages = scenario(n * 31 + P, n, P, width, kind)
    n_tokens = sum(add) + room
    want = host_plan(lens, add, table, free, len(free), P, n_tokens)
    assert want[0] == 0
    L, A, F = i32(lens, cuda), i32(add, cuda), i32(free, cuda)
    # a table with a wider stride, whose other columns stay
    wide = torch.full((n, width + 3), 99, dtype=torch.int32, device=cuda)
    wide[:, :width] = i32(table, cuda)
    T = wide[:, :width]
    S = i32([len(free), 55, 55, 55], cuda)
    out = None
    if in_place:
        e = lambda k, t=torch.int32: torch.full((k,), 123, dtype=t, device=cuda)  # noqa: E731
        out = paged.Plan(L, S, e(n + 1), e(n_tokens, torch.int64), e(n_tokens), e(n_tokens))
    p = paged.plan(L, A, T, F, S, page_size=P, n_pages=n_pages, n_tokens=n_tokens, out=out)
    assert p.state.tolist() == [want[3], 0, sum(add), want[4]]
    assert p.lens.tolist() == want[1] and T.tolist() == want[2] and p.cu_tokens.tolist() == want[5]
    assert p.slots.tolist() == want[6] and p.positions.tolist() == want[7] and p.requests.tolist() == want[8]
    assert bool((wide[:, width:] == 99).all()) and F.tolist() == free
    if not in_place:
        assert L.tolist() == lens and S.tolist() == [len(free), 55, 55, 55]
    no_error()


@pytest.mark.parametrize("what,status", [("pages", 1), ("row", 2), ("room", 3), ("negative", 4), ("add", 4),
                                         ("count", 4)])
@pytest.mark.parametrize("n", [5, 700])
def test_plan_all_or_nothing(cuda, what, status, n):
    import torch
    from toy_b200 import paged
    P, width = 16, 40
    lens, add, table, free, n_pages = scenario(9, n, P, width, "mixed")
    lens[2], add[2], lens[4] = 10, 30, 100
    n_tokens, count = sum(add), len(free)
    if what == "pages":
        count = 1
    elif what == "row":
        add[4] = width * P - 99
        n_tokens = sum(add)
    elif what == "room":
        n_tokens -= 1
    elif what == "negative":
        lens[1] = -1
    elif what == "add":
        add[3] = -2
    else:
        count = len(free) + 1
    L, A, F, T, S = i32(lens, cuda), i32(add, cuda), i32(free, cuda), i32(table, cuda), i32([count, 0, 0, 0], cuda)
    p = paged.plan(L, A, T, F, S, page_size=P, n_pages=n_pages, n_tokens=n_tokens)
    assert p.state.tolist() == [count, status, 0, 0]
    assert p.lens.tolist() == lens and T.tolist() == table and F.tolist() == free
    assert p.cu_tokens.tolist() == [0] * (n + 1)
    assert bool((p.slots == -1).all()) and bool((p.positions == 0).all()) and bool((p.requests == -1).all())
    torch.cuda.synchronize()
    no_error()


def test_plan_bad_page_ids(cuda):
    """A page id that is no page: its tokens get slot -1 and the error word says so; the others are right."""
    from toy_b200 import paged
    from toy_b200._lib import lib
    P = 4
    F = i32([2, -3, 5], cuda)                            # free[1], the second page taken, is none
    T = i32([[0, -1, -1], [77, -1, -1], [1, -1, -1]], cuda)   # nor is request 1's open page
    # request 2: position 3 in page 1, 4..7 in free[2] = 5, 8 in free[1]
    p = paged.plan(i32([2, 2, 3], cuda), i32([1, 1, 6], cuda), T, F, i32([3, 0, 0, 0], cuda), page_size=P, n_pages=6,
                   n_tokens=8)
    assert p.slots.tolist() == [2, -1, 7, 20, 21, 22, 23, -1] and p.state.tolist() == [1, 0, 8, 2]
    assert lib().tb2_device_error() == 0x5001
    no_error()


@pytest.mark.parametrize("n,P,width", [(1, 16, 3), (40, 8, 5), (900, 16, 40), (16384, 4, 2)])
@pytest.mark.parametrize("in_place", [False, True])
def test_release(cuda, n, P, width, in_place):
    import random
    from toy_b200 import paged
    lens, _, table, free, n_pages = scenario(n + 5, n, P, width, "none")
    r = random.Random(n)
    done = [r.choice([0, 0, 1, 7, -1]) for _ in range(n)]
    cap = free + [-9] * (n_pages - len(free))
    want_free, want_table, want_lens = list(free), [list(t) for t in table], list(lens)
    for b in range(n):
        if done[b]:
            h = -(-lens[b] // P)
            want_free += table[b][:h]
            want_table[b][:h] = [-1] * h
            want_lens[b] = 0
    pushed = len(want_free) - len(free)
    L, D, T, F, S = i32(lens, cuda), i32(done, cuda), i32(table, cuda), i32(cap, cuda), i32([len(free), 0, 0, 0], cuda)
    Lo, So = (L, S) if in_place else (i32([5] * n, cuda), i32([5] * 4, cuda))
    paged.release(L, D, T, F, S, page_size=P, n_pages=n_pages, lens_out=Lo, state_out=So)
    assert So.tolist() == [len(want_free), 0, 0, pushed]
    assert Lo.tolist() == want_lens and T.tolist() == want_table
    assert F.tolist() == want_free + cap[len(want_free):]
    no_error()


@pytest.mark.parametrize("what,status", [("stack", 1), ("negative", 4), ("long", 4), ("count", 4)])
def test_release_all_or_nothing(cuda, what, status):
    from toy_b200 import paged
    P, n, width = 8, 20, 6
    lens, _, table, free, n_pages = scenario(3, n, P, width, "none")
    lens[4], count = 30, len(free)
    cap = free + [-9] * 4
    if what == "stack":
        cap = free
    elif what == "negative":
        lens[0] = -5
    elif what == "long":
        lens[0] = width * P + 1
    else:
        count = -1
    L, T, F, S = i32(lens, cuda), i32(table, cuda), i32(cap, cuda), i32([count, 0, 0, 0], cuda)
    paged.release(L, i32([1] * n, cuda), T, F, S, page_size=P, n_pages=n_pages)
    assert S.tolist() == [count, status, 0, 0]
    assert L.tolist() == lens and T.tolist() == table and F.tolist() == cap
    no_error()


# ------------------------------------------------------------------ append
def rope_table(rows, dh, dev):
    import torch
    a = torch.arange(rows, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, dh, 2).double() / dh)
    return torch.stack([a.cos(), a.sin()], -1).float().contiguous().to(dev)


@pytest.mark.parametrize("row", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("cache", ["f32", "f16", "bf16", "q8_0"])
@pytest.mark.parametrize("n,H,KV,dh,P,layout", [
    (1, 9, 3, 64, 16, "heads"), (7, 4, 4, 32, 1, "tokens"), (37, 28, 4, 128, 16, "layers"),
    (64, 6, 2, 96, 24, "tokens"), (300, 8, 1, 128, 100, "heads"), (5, 5, 5, 64, 3, "layers")])
def test_append(cuda, row, cache, n, H, KV, dh, P, layout):
    import torch
    from toy_b200 import paged
    g = torch.Generator(device=cuda).manual_seed(n * 7 + dh)
    n_pages = (n + P - 1) // P + 2
    k, v, ks, vs = R.make_pools(n_pages, KV, P, dh, cache, layout, g, cuda)
    before = [x.clone() if x is not None else None for x in (k, v, ks, vs)]
    c = paged.PagedCache(k, v, ks, vs)
    qkv = torch.randn((n, (H + 2 * KV) * dh + 16), generator=g, device=cuda).to(R.TORCH[row])
    qkv[0, :] = 0                                       # zero rows: a Q8_0 scale of 0
    q, kn, vn = (qkv[:, a * dh:b * dh].view(n, b - a, dh) for a, b in
                 ((0, H), (H, H + KV), (H + KV, H + 2 * KV)))
    slots = torch.randperm(n_pages * P, generator=g, device=cuda)[:n]
    slots[n // 3:n // 3 + n // 4] = -1                  # padded rows
    pos = torch.randint(0, 500, (n,), generator=g, device=cuda, dtype=torch.int32)
    rope = rope_table(500, dh, cuda)
    bias = torch.randn((H + 2 * KV) * dh, generator=g, device=cuda) if n % 2 else None
    f = [q.float(), kn.float(), vn.float()]
    if bias is not None:
        b = bias.view(-1, dh)
        f = [f[0] + b[:H], f[1] + b[H:H + KV], f[2] + b[H + KV:]]
    cs = rope[pos.long()]
    want_q, want_k, want_v = R.rotate(f[0], cs), R.rotate(f[1], cs), f[2]
    got = paged.append(c, slots, kn, vn, q=q, positions=pos, rope=rope, bias=bias)
    assert torch.equal(got, want_q.to(q.dtype))
    live = slots >= 0
    pg, off = slots[live] // P, slots[live] % P
    for pool, scale, x, old, olds in ((k, ks, want_k, before[0], before[2]), (v, vs, want_v, before[1], before[3])):
        if cache == "q8_0":
            qx, dx = R.q8_0(x[live])
            old[pg, :, off], olds[pg, :, off] = qx, dx
            assert torch.equal(scale.view(torch.int16), olds.view(torch.int16))
        else:
            old[pg, :, off] = x[live].to(pool.dtype)
        assert torch.equal(pool, old)                   # the other rows as they were
    # q in place, without rope or bias k and v alone are the plain rows
    q2 = q.clone()
    paged.append(c, torch.full_like(slots, -1), kn, vn, q=q2, q_out=q2, positions=pos, rope=rope, bias=bias)
    assert torch.equal(q2, got)
    paged.append(c, slots, kn, vn)
    for pool, scale, x in ((k, ks, kn), (v, vs, vn)):
        rows = R.values(pool, scale)[pg, :, off]
        x = x[live].float()
        ref = x.to(pool.dtype).double() if cache != "q8_0" else R.values(*R.q8_0(x))
        assert torch.equal(rows, ref)
    no_error()


def test_append_out_of_range(cuda):
    """A slot past the pool and a position past the table write nothing and are reported; the rest is written."""
    import torch
    from toy_b200 import paged
    from toy_b200._lib import lib
    z = lambda: torch.zeros((3, 2, 4, 32), device=cuda)  # noqa: E731
    for bad, code in (("slot", 0x5002), ("position", 0x5003), ("negative position", 0x5003)):
        k, v = z(), z()
        c = paged.PagedCache(k, v)
        x = torch.ones((3, 2, 32), device=cuda)
        slots = torch.tensor([1, 12 if bad == "slot" else 2, 11], device=cuda)
        pos = i32([0, {"slot": 1, "position": 8, "negative position": -1}[bad], 2], cuda)
        paged.append(c, slots, x, x, positions=pos, rope=rope_table(8, 32, cuda))
        want = z()
        for s in (1, 11):
            want[s // 4, :, s % 4] = 1
        assert lib().tb2_device_error() == code
        assert torch.equal(v, want)


# ------------------------------------------------------------------ attend
def run_attend(cuda, lens, H, KV, dh, P, row, cache, layout="heads", seed=0, mag=1.0, qmag=1.0, width=None, scale=None,
               poison=True, extra=0):
    import torch
    from toy_b200 import paged
    g = torch.Generator(device=cuda).manual_seed(seed + dh + H)
    n = len(lens)
    need = [(max(0, x) + P - 1) // P for x in lens]
    width = width or max(1, max(need))
    n_pages = sum(need) + 2 + extra
    k, v, ks, vs = R.make_pools(n_pages, KV, P, dh, cache, layout, g, cuda, mag)
    perm = torch.randperm(n_pages, generator=g, device=cuda).int()
    table = torch.full((n, width + 2), 10 ** 9, dtype=torch.int32, device=cuda)     # unused entries: no page
    at, dead = 0, torch.ones((n_pages, P), dtype=torch.bool, device=cuda)
    for b in range(n):
        table[b, :need[b]] = perm[at:at + need[b]]
        dead[perm[at:at + need[b]].long()] = False
        if need[b] and lens[b] % P:
            dead[int(perm[at + need[b] - 1]), lens[b] % P:] = True
        at += need[b]
    kd, vd = R.values(k, ks), R.values(v, vs)
    if poison:                                          # what no request holds may be anything
        if cache == "q8_0":
            for s in (ks, vs):
                s.masked_fill_(dead[:, None, :, None], math.nan)
        else:
            k.masked_fill_(dead[:, None, :, None], math.nan)
            v.masked_fill_(dead[:, None, :, None], math.inf)
    qkv = (torch.randn((n, (H + 2) * dh), generator=g, device=cuda) * qmag).to(R.TORCH[row])
    q = qkv[:, dh:(H + 1) * dh].view(n, H, dh)          # a view with a wider stride
    lt = i32(lens, cuda)
    sc = dh ** -0.5 if scale is None else scale
    lse = torch.zeros((n, H), device=cuda)
    ws = paged.attend_workspace(cuda)
    cache_ = paged.PagedCache(k, v, ks, vs)
    out = paged.attend(cache_, q, table[:, :width], lt, lse=lse, scale=sc, workspace=ws)
    o, l, av, ds = R.attend(kd, vd, q, table, lens, sc)
    bo, bl = R.attend_bounds(o, l, av, ds, lt, dh, q.dtype)
    empty = lt <= 0
    assert bool((out[empty] == 0).all()) and bool((lse[empty] == -math.inf).all())
    err = (out.double() - o).abs()
    assert bool((err <= bo).all()), (float((err / bo).max()), float(err.max()))
    assert bool(((lse.double() - l).abs()[~empty] <= bl[~empty]).all()), float(((lse.double() - l).abs()[~empty] / bl[~empty]).max())
    # the same bits again, with the workspace the last call left
    out2, lse2 = torch.full_like(out, 7), torch.full_like(lse, 7)
    paged.attend(cache_, q, table[:, :width], lt, out=out2, lse=lse2, scale=sc, workspace=ws)
    assert torch.equal(out, out2) and torch.equal(lse, lse2)
    no_error()
    return out, o


EDGES = [0, 1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 255, 257, 300]


@pytest.mark.parametrize("row", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("cache", ["f32", "f16", "bf16", "q8_0"])
@pytest.mark.parametrize("H,KV,dh,P,layout", [
    (9, 3, 64, 16, "heads"), (28, 4, 128, 16, "tokens"), (4, 4, 32, 1, "heads"), (6, 2, 96, 24, "layers"),
    (16, 1, 128, 100, "heads"), (8, 1, 64, 32, "tokens"), (40, 2, 64, 8, "heads"), (18, 2, 96, 64, "heads"),
    (12, 1, 32, 128, "layers")])
def test_attend_edges(cuda, row, cache, H, KV, dh, P, layout):
    run_attend(cuda, EDGES, H, KV, dh, P, row, cache, layout)


@pytest.mark.parametrize("cache", ["f32", "f16", "bf16", "q8_0"])
@pytest.mark.parametrize("lens,H,KV,dh,P", [
    ([1], 1, 1, 64, 16), ([5000], 8, 1, 128, 16), ([20011], 9, 3, 64, 24), ([0, 0, 0], 4, 2, 64, 16),
    ([3000, 1, 0, 17, 4097], 28, 4, 128, 128), ([1024] * 3, 16, 16, 128, 1024), ([700] * 40, 32, 8, 64, 16),
    ([-3, 5], 4, 2, 32, 16), ([2500] * 2, 4, 4, 96, 7)])
def test_attend_lengths(cuda, cache, lens, H, KV, dh, P):
    run_attend(cuda, lens, H, KV, dh, P, "f32", cache, seed=3)


@pytest.mark.parametrize("cache", ["f32", "f16", "bf16", "q8_0"])
@pytest.mark.parametrize("mag,qmag,scale", [(1e-4, 1e3, 0.3), (30.0, 3.0, 0.5), (1.0, 1e-6, 1.0), (2e-3, 2e4, -0.1),
                                            (1.0, 1.0, 0.0)])
def test_attend_magnitudes(cuda, cache, mag, qmag, scale):
    """Tiny and large keys, queries and scores (one key takes all the weight, or all the same)."""
    run_attend(cuda, [1, 50, 333, 1000], 12, 3, 64, 16, "f32", cache, seed=5, mag=mag, qmag=qmag, scale=scale)


@pytest.mark.parametrize("n", [1, 3, 500, 5000])
def test_attend_many_requests(cuda, n):
    import random
    r = random.Random(n)
    run_attend(cuda, [r.choice([0, 1, 5, 16, 40, 90]) for _ in range(n)], 4, 2, 32, 16, "f32", "bf16", seed=n)


def test_attend_growing_values(cuda):
    """Keys whose scores rise along the history (the running maximum moves at every tile), one of them far above the
    rest in the middle, and values of very different sizes along it."""
    import torch
    from toy_b200 import paged
    for cache in ("f32", "f16", "bf16", "q8_0"):
        L, P, dh = 900, 16, 64
        ramp = torch.linspace(-8, 8, L, device=cuda)
        ramp[L // 2] = 60.0
        rows = torch.zeros((1024, dh), device=cuda)
        rows[:L, 0] = ramp
        rows[:, 40] = 0.5
        vals = torch.randn((1024, dh), generator=torch.Generator(device=cuda).manual_seed(1), device=cuda)
        vals *= (10.0 ** torch.linspace(-3, 3, 1024, device=cuda))[:, None]
        for flip in (False, True):
            if flip:
                vals = vals.flip(0)
            pools = []
            for x in (rows, vals):
                x = x.view(64, 1, P, dh)
                pools.append(R.q8_0(x) if cache == "q8_0" else (x.to(R.TORCH[cache]), None))
            (k, ks), (v, vs) = pools
            q = torch.zeros((1, 3, dh), device=cuda)
            q[0, :, 0] = torch.tensor([8.0, -8.0, 0.1], device=cuda)
            table = torch.arange(64, dtype=torch.int32, device=cuda)[None, :]
            lens = i32([L], cuda)
            out = paged.attend(paged.PagedCache(k, v, ks, vs), q, table, lens, scale=0.25)
            o, l, av, ds = R.attend(R.values(k, ks), R.values(v, vs), q, table, [L], 0.25)
            bo, _ = R.attend_bounds(o, l, av, ds, lens, dh, q.dtype)
            assert bool(((out.double() - o).abs() <= bo).all()), (cache, flip)
    no_error()


def test_attend_bad_pages(cuda):
    """Pages that are none are skipped: the request attends to the rest, and the error word says so."""
    import torch
    from toy_b200 import paged
    from toy_b200._lib import lib
    g = torch.Generator(device=cuda).manual_seed(0)
    k, v, _, _ = R.make_pools(8, 2, 16, 64, "bf16", "heads", g, cuda)
    q = torch.randn((2, 6, 64), generator=g, device=cuda)
    for bad in (8, -1, 2 ** 31 - 1, -2 ** 31):
        out = paged.attend(paged.PagedCache(k, v), q, i32([[0, bad, 2, 3], [4, 5, 6, bad]], cuda), i32([60, 40], cuda))
        assert lib().tb2_device_error() == 0x5001
        good = paged.attend(paged.PagedCache(k, v), q, i32([[0, 2, 3, 0], [4, 5, 6, 7]], cuda), i32([44, 40], cuda))
        no_error()
        assert float((out - good).abs().max()) < 1e-5      # the same keys, other tiles
    bad = paged.attend(paged.PagedCache(k, v), q[:1], i32([[9, 9, 9]], cuda), i32([33], cuda))
    assert lib().tb2_device_error() == 0x5001 and bool((bad == 0).all())


def test_attend_lengths_past_the_table(cuda):
    """A length beyond what the table row spans is cut to it."""
    import torch
    from toy_b200 import paged
    g = torch.Generator(device=cuda).manual_seed(0)
    k, v, _, _ = R.make_pools(12, 2, 16, 64, "f16", "heads", g, cuda)
    q = torch.randn((2, 6, 64), generator=g, device=cuda)
    table = torch.arange(12, dtype=torch.int32, device=cuda).view(2, 6)
    c = paged.PagedCache(k, v)
    want = paged.attend(c, q, table, i32([96, 40], cuda))
    for long in (97, 1000, 2 ** 31 - 1):
        assert torch.equal(paged.attend(c, q, table, i32([long, 40], cuda)), want)
    no_error()


def test_attend_huge_queries(cuda):
    """Queries near the end of the f32 range still pick the key of the largest score."""
    import torch
    from toy_b200 import paged
    for cache in ("f32", "f16", "bf16", "q8_0"):
        g = torch.Generator(device=cuda).manual_seed(0)
        k, v, ks, vs = R.make_pools(4, 1, 16, 64, cache, "heads", g, cuda)
        q = torch.randn((1, 2, 64), generator=g, device=cuda) * torch.tensor([1e35, 1e-30], device=cuda)[:, None]
        table = torch.arange(4, dtype=torch.int32, device=cuda)[None, :]
        out = paged.attend(paged.PagedCache(k, v, ks, vs), q, table, i32([60], cuda))
        kd, vd = (R.values(a, b).reshape(-1, 64)[:60] for a, b in ((k, ks), (v, vs)))
        top = vd[(kd @ q[0, 0].double()).argmax()]
        assert float((out[0, 0].double() - top).abs().max()) <= 2e-6 * float(top.abs().max())
        mean = vd.mean(0)      # all scores are 0
        assert float((out[0, 1].double() - mean).abs().max()) <= 2e-6 * float(vd.abs().mean())
    no_error()


def test_own_workspace_in_a_graph(cuda):
    """Without a workspace the call makes its own, in a captured graph too."""
    import torch
    from toy_b200 import paged
    g = torch.Generator(device=cuda).manual_seed(3)
    k, v, _, _ = R.make_pools(200, 2, 16, 64, "bf16", "heads", g, cuda)
    c = paged.PagedCache(k, v)
    q = torch.randn((2, 8, 64), generator=g, device=cuda)
    table, lens = torch.arange(200, dtype=torch.int32, device=cuda).view(2, 100), i32([1600, 900], cuda)
    want = paged.attend(c, q, table, lens)
    out = torch.empty_like(want)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        paged.attend(c, q, table, lens, out=out)
    for _ in range(3):
        out.fill_(7)
        gr.replay()
        assert torch.equal(out, want)
    no_error()


def test_attend_past_32_bits(cuda):
    """A pool of more than 2^31 elements: pages at its far end."""
    import torch
    from toy_b200 import paged
    KV, P, dh = 4, 64, 128
    n_pages = 2 ** 31 // (KV * P * dh) + 40
    for cache in ("q8_0", "bf16"):
        shape = (n_pages, KV, P, dh)
        t = torch.int8 if cache == "q8_0" else torch.bfloat16
        k, v = torch.empty(shape, dtype=t, device=cuda), torch.empty(shape, dtype=t, device=cuda)
        ks = vs = None
        if cache == "q8_0":
            ks, vs = (torch.empty(shape[:3] + (dh // 32,), dtype=torch.float16, device=cuda) for _ in range(2))
        ids = torch.tensor([n_pages - 1, 3, n_pages - 20, n_pages - 39], device=cuda)
        g = torch.Generator(device=cuda).manual_seed(2)
        small = R.make_pools(4, KV, P, dh, cache, "heads", g, cuda)
        for big, s in zip((k, v, ks, vs), small):
            if s is not None:
                big[ids] = s
        q = torch.randn((1, 8, dh), generator=g, device=cuda)
        a = paged.attend(paged.PagedCache(k, v, ks, vs), q, ids.int()[None, :], i32([250], cuda))
        b = paged.attend(paged.PagedCache(*small), q, i32([[0, 1, 2, 3]], cuda), i32([250], cuda))
        assert torch.equal(a, b)
        # and a row appended there
        row = torch.randn((1, KV, dh), generator=g, device=cuda)
        slot = torch.tensor([(n_pages - 1) * P + 5], device=cuda)
        paged.append(paged.PagedCache(k, v, ks, vs), slot, row, row)
        want = R.q8_0(row)[0] if cache == "q8_0" else row.to(t)
        assert torch.equal(k[n_pages - 1, :, 5], want[0]) and torch.equal(v[n_pages - 1, :, 5], want[0])
        del k, v, ks, vs
        torch.cuda.empty_cache()
    no_error()


def test_nonfinite_stays_in_its_request(cuda):
    """A NaN key of one request and a NaN query head of another reach no other request or head."""
    import torch
    from toy_b200 import paged
    g = torch.Generator(device=cuda).manual_seed(4)
    for cache in ("f32", "f16", "bf16"):
        k, v, _, _ = R.make_pools(9, 2, 16, 64, cache, "heads", g, cuda)
        q = torch.randn((3, 6, 64), generator=g, device=cuda)
        table = torch.arange(9, dtype=torch.int32, device=cuda).view(3, 3)
        lens = i32([40, 48, 33], cuda)
        c = paged.PagedCache(k, v)
        base = paged.attend(c, q, table, lens)
        k[0, 0, 3] = math.nan
        q[2, 4] = math.nan
        got = paged.attend(c, q, table, lens)
        assert bool(got[0, :3].isnan().all()) and bool(got[2, 4].isnan().all())
        keep = torch.ones((3, 6), dtype=torch.bool, device=cuda)
        keep[0, :3] = False
        keep[2, 4] = False
        assert torch.equal(got[keep], base[keep])
    no_error()


# ------------------------------------------------------------------ streams, graphs, refusals with GPU tensors
def test_python_refusals(cuda):
    import torch
    from toy_b200 import paged
    k = torch.zeros((4, 2, 16, 64), device=cuda)
    c = paged.PagedCache(k, k.clone())
    q, t, n = torch.zeros((2, 4, 64), device=cuda), i32([[0], [1]], cuda), i32([1, 1], cuda)
    bad = [lambda: paged.PagedCache(k, k[:3]), lambda: paged.PagedCache(k, k.bfloat16()),
           lambda: paged.PagedCache(k.to(torch.int8), k.to(torch.int8)), lambda: paged.PagedCache(k, k.cpu()),
           lambda: paged.PagedCache(k.transpose(2, 3), k.transpose(2, 3)),
           lambda: paged.PagedCache(k, k.clone(), k, k), lambda: paged.attend(c, q[:, :3], t, n),
           lambda: paged.attend(c, q[..., :32], t, n), lambda: paged.attend(c, q.double(), t, n),
           lambda: paged.attend(c, q, t.long(), n), lambda: paged.attend(c, q, t[:1], n),
           lambda: paged.attend(c, q, t, n[:1]), lambda: paged.attend(c, q, t, n.cpu()),
           lambda: paged.attend(c, q, t, n, out=q.bfloat16()), lambda: paged.attend(c, q, t, n, lse=q),
           lambda: paged.attend(c, q, t, n, workspace=q), lambda: paged.attend(c, q.transpose(0, 1), t, n),
           lambda: paged.append(c, n, q[:, :2], q[:, :2]),
           lambda: paged.append(c, n.long(), q[:, :2], q[:, :2].bfloat16()),
           lambda: paged.append(c, n.long(), q, q), lambda: paged.append(c, n.long(), q[:, :2], q[:, :2], rope=k),
           lambda: paged.append(c, n.long(), q[:, :2], q[:, :2], q=q, bias=torch.zeros(64, device=cuda)),
           lambda: paged.plan(n, n, t, n, n, page_size=16, n_pages=4, n_tokens=2),
           lambda: paged.plan(n, n[:1], t, n, i32([0] * 4, cuda), page_size=16, n_pages=4, n_tokens=2)]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was not refused")
    with pytest.raises(RuntimeError):
        paged.attend(c, q, t, n, workspace=torch.zeros(16, dtype=torch.uint8, device=cuda)[:8])
    with pytest.raises(RuntimeError):
        paged.plan(n, n, t, n, i32([0] * 4, cuda), page_size=0, n_pages=4, n_tokens=2)
    assert paged.append(c, n.long()[:0], q[:0, :2], q[:0, :2]) is None
    assert paged.attend(c, q[:0], t, n).shape == (0, 4, 64)


def test_side_stream_and_graph(cuda):
    """plan, append and attend captured on a side stream and replayed on grown lengths, against eager calls; a second
    graph with its own workspace replays beside it."""
    import torch
    from toy_b200 import paged
    n, H, KV, dh, P, width = 5, 9, 3, 64, 16, 20
    n_pages = n * width

    class World:
        def __init__(self):
            g = torch.Generator(device=cuda).manual_seed(11)
            self.k, self.v, self.ks, self.vs = R.make_pools(n_pages, KV, P, dh, "q8_0", "heads", g, cuda)
            self.c = paged.PagedCache(self.k, self.v, self.ks, self.vs)
            self.lens, self.add = i32([0] * n, cuda), i32([1, 1, 0, 1, 1], cuda)
            self.table = torch.full((n, width), -1, dtype=torch.int32, device=cuda)
            self.free, self.state = torch.arange(n_pages, dtype=torch.int32, device=cuda), i32([n_pages, 0, 0, 0], cuda)
            e = lambda t: torch.empty(n, dtype=t, device=cuda)  # noqa: E731
            self.out = paged.Plan(self.lens, self.state, torch.empty(n + 1, dtype=torch.int32, device=cuda),
                                  e(torch.int64), e(torch.int32), e(torch.int32))
            self.x = torch.zeros((n, (H + 2 * KV) * dh), device=cuda)
            self.q_out, self.o = torch.empty((n, H, dh), device=cuda), torch.empty((n, H, dh), device=cuda)
            self.rope, self.ws = rope_table(width * P, dh, cuda), paged.attend_workspace(cuda)

        def step(self):
            p = paged.plan(self.lens, self.add, self.table, self.free, self.state, page_size=P, n_pages=n_pages,
                           n_tokens=n, out=self.out)
            q, k, v = (self.x[:, a * dh:b * dh].view(n, b - a, dh) for a, b in
                       ((0, H), (H, H + KV), (H + KV, H + 2 * KV)))
            # token i of the step belongs to request requests[i]; here rows are kept per request: row i -> slots[i]
            paged.append(self.c, p.slots, k, v, q=q, q_out=self.q_out, positions=p.positions, rope=self.rope)
            paged.attend(self.c, self.q_out, self.table, self.lens, out=self.o, workspace=self.ws)

    eager, one, two = World(), World(), World()
    side = torch.cuda.Stream()
    graphs = []
    torch.cuda.synchronize()
    for w in (one, two):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=side):
            w.step()
        graphs.append(gr)
    other = torch.cuda.Stream()
    for i in range(40):
        x = torch.randn((n, (H + 2 * KV) * dh), generator=torch.Generator(device=cuda).manual_seed(i), device=cuda)
        for w in (eager, one, two):
            w.x.copy_(x)
        eager.step()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[0].replay()
        with torch.cuda.stream(other):
            graphs[1].replay()
        torch.cuda.synchronize()
        for w in (one, two):
            assert torch.equal(w.o, eager.o) and torch.equal(w.q_out, eager.q_out)
            assert torch.equal(w.table, eager.table) and torch.equal(w.lens, eager.lens)
            assert torch.equal(w.k, eager.k) and torch.equal(w.v, eager.v)
    assert eager.lens.tolist() == [40, 40, 0, 40, 40]
    no_error()


# ------------------------------------------------------------------ a run of them together
@pytest.mark.parametrize("cache,row", [("bf16", "bf16"), ("f32", "f32"), ("q8_0", "f32"), ("f16", "f32")])
def test_serving_loop(cuda, cache, row):
    """Requests come, append prompts or single tokens, attend, finish and give their pages back, 25 steps, against
    host-side lists of every request's rows."""
    import random
    import torch
    from toy_b200 import paged
    r = random.Random(6)
    n, H, KV, dh, P, width = 6, 8, 2, 64, 8, 10
    n_pages = 20                                        # too few at times: some steps find no room
    g = torch.Generator(device=cuda).manual_seed(1)
    k, v, ks, vs = R.make_pools(n_pages, KV, P, dh, cache, "tokens", g, cuda)
    c = paged.PagedCache(k, v, ks, vs)
    rope = rope_table(width * P, dh, cuda)
    ws = paged.attend_workspace(cuda)
    lens, table = i32([0] * n, cuda), torch.full((n, width), -1, dtype=torch.int32, device=cuda)
    free, state = torch.randperm(n_pages, generator=g, device=cuda).int(), i32([n_pages, 0, 0, 0], cuda)
    rows = [([], []) for _ in range(n)]
    refused = 0
    for step in range(25):
        add = [r.choice([0, 1, 1, 1, 3, 20]) for _ in range(n)]
        n_tokens = sum(add) + r.choice([0, 2])
        x = torch.randn((n_tokens, (H + 2 * KV) * dh), generator=g, device=cuda).to(R.TORCH[row])
        p = paged.plan(lens, i32(add, cuda), table, free, state, page_size=P, n_pages=n_pages, n_tokens=n_tokens)
        ql, kl, vl = (x[:, a * dh:b * dh].view(n_tokens, b - a, dh) for a, b in
                      ((0, H), (H, H + KV), (H + KV, H + 2 * KV)))
        qo = paged.append(c, p.slots, kl, vl, q=ql, positions=p.positions, rope=rope)
        assert torch.equal(p.lens - lens, i32(add, cuda)) or int(p.state[1]) != 0
        lens, state = p.lens, p.state
        if int(state[1]):                               # no room: the step did nothing
            refused += 1
            add = [0] * n
        kr = R.rotate(kl.float(), rope[p.positions.long()])
        for t in range(sum(add)):
            b = int(p.requests[t])
            for w, y in ((0, kr[t]), (1, vl[t].float())):
                rows[b][w].append(R.values(*R.q8_0(y)) if cache == "q8_0" else y.to(k.dtype).double())
        # the requests' last token of the step attends (a request that appended none repeats its first row)
        last = [max(0, int(p.cu_tokens[b + 1]) - 1) for b in range(n)]
        q = qo[torch.tensor(last, device=cuda)] if n_tokens else torch.zeros((n, H, dh), device=cuda, dtype=x.dtype)
        out = paged.attend(c, q, table, lens, workspace=ws)
        hist = [len(a) for a, _ in rows]
        assert lens.tolist() == hist
        most = max(1, max(hist))
        kd, vd = (torch.zeros((n, KV, most, dh), dtype=torch.float64, device=cuda) for _ in range(2))
        for b in range(n):
            for w, d in ((0, kd), (1, vd)):
                for t, y in enumerate(rows[b][w]):
                    d[b, :, t] = y
        o, l, av, ds = R.attend(kd, vd, q, torch.arange(n, device=cuda)[:, None], hist, dh ** -0.5)
        bo, _ = R.attend_bounds(o, l, av, ds, lens, dh, q.dtype)
        assert bool(((out.double() - o).abs() <= bo).all())
        done = [int(h > 50 or r.random() < 0.1) for h in hist]
        paged.release(lens, i32(done, cuda), table, free, state, page_size=P, n_pages=n_pages)
        for b in range(n):
            if done[b]:
                rows[b] = ([], [])
        held = sum(-(-len(a) // P) for a, _ in rows)
        assert state.tolist()[:2] == [n_pages - held, 0]
        ids = free[:n_pages - held].tolist() + [int(table[b, i]) for b in range(n)
                                                for i in range(-(-len(rows[b][0]) // P))]
        assert sorted(ids) == list(range(n_pages))
    assert refused
    no_error()
