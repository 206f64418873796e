"""The paged KV-cache operators at the ends of their ranges: scores far from 0
against the values that a single key leaves, and the calls the other paged
tests do not make."""
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


def pools(x, cache):
    """(pool, scale) of f32 rows x in the cache's type."""
    return R.q8_0(x) if cache == "q8_0" else (x.to(R.TORCH[cache]), None)


# ------------------------------------------------------------------ attend
@pytest.mark.parametrize("cache", ["f32", "f16", "bf16", "q8_0"])
@pytest.mark.parametrize("G,dh", [(3, 64), (12, 64), (7, 128), (2, 32)])
def test_attend_far_scores(cuda, cache, G, dh):
    """Largest scores of 2^18 to 2^31 (in powers of two), above and below 0, histories of one key, of one tile and of
    many: the key of the largest score takes all the weight, so the output is its value row and lse its score.

    The keys' scores differ by 1 / 64 of 2^18 at least, so every other weight is 0 in 32 bits. What is left: the
    weight's planes (2^-23 of it), the value's (f32: 2^-22), sums, the quotient and its rounding (4 u), 2^-20 together
    with room for a factor of two; a score's are its operands' (2^-22 each at most), 3 roundings on the way in and 3
    out: 2^-20 as well."""
    import torch
    from toy_b200 import paged
    g = torch.Generator(device=cuda).manual_seed(dh + G)
    P, lens = 16, [1, 40, 700]
    width = 44
    n = len(lens)
    rows = torch.zeros((n, width * P, dh), device=cuda)
    vals = torch.randn((n, width * P, dh), generator=g, device=cuda)
    if cache == "q8_0":                             # (scales of unlike sizes: from 2^-9 to 2^4 times the usual)
        vals *= 2.0 ** torch.randint(-9, 5, (n, width * P, 1), generator=g, device=cuda)
    for b, L in enumerate(lens):
        order = torch.randperm(L, generator=g, device=cuda)
        rows[b, :L, 0] = 1 + order % 64 / 64.0      # the largest of many keys is met more than once
        top = int((order % 64).max())
        keep = (order % 64 == top).nonzero()[0]
        rows[b, :L, 0][order % 64 == top] -= 1 / 64.0
        rows[b, keep, 0] += 1 / 64.0
    for sign in (1.0, -1.0):                        # below 0: the smallest |score| is the largest, made one as well
        shape = rows if sign > 0 else torch.where(rows > 0, 3.0 - rows, rows)
        (k, ks), (v, vs) = (pools(x.view(n * width, 1, P, dh), cache) for x in (shape, vals))
        kd, vd = R.values(k, ks).view(n, -1, dh), R.values(v, vs).view(n, -1, dh)
        c = paged.PagedCache(k, v, ks, vs)
        table = torch.arange(n * width, dtype=torch.int32, device=cuda).view(n, width)
        for e in range(18, 32):
            for mant in (1.0, 1.3, 1.7):
                q = torch.zeros((n, G, dh), device=cuda)
                q[:, :, 0] = sign * mant * 2.0 ** e / 1.4427 * (1 + torch.arange(G, device=cuda) / 64.0)
                lse = torch.empty((n, G), device=cuda)
                out = paged.attend(c, q, table, i32(lens, cuda), lse=lse, scale=0.5)
                for b, L in enumerate(lens):
                    s = q[b, :, :1].double() * kd[b, :L, 0] * 0.5
                    top, at = s.max(-1)
                    assert bool((s.topk(min(2, L), -1).values.diff().abs() > 300).all())   # (the case's own promise)
                    want = vd[b, at]
                    err = (out[b].double() - want).abs()
                    assert bool((err <= 2.0 ** -20 * want.abs()).all()), (sign, e, mant, L, float(err.max()))
                    assert bool(((lse[b].double() - top).abs() <= 2.0 ** -20 * top.abs()).all()), (sign, e, mant, L)
    no_error()


def finite(x):
    import torch
    return torch.nan_to_num(x, nan=0.0, posinf=0.0, neginf=0.0)


@pytest.mark.parametrize("row", ["f32", "bf16"])
@pytest.mark.parametrize("cache", ["f32", "f16", "bf16", "q8_0"])
@pytest.mark.parametrize("H,KV,dh,P,lens", [
    (6, 2, 64, 16, [3, 40, 0, 700]), (12, 1, 128, 16, [1, 20000]), (3, 3, 32, 5, [9, 300, 2000]),
    (40, 2, 64, 8, [5, 333]),
    (10, 1, 96, 32, [70, 5000])])
def test_attend_infinities(cuda, row, cache, H, KV, dh, P, lens):
    """Keys and values with infinities in a live history, against the formula in 64 bits: a key whose score is -inf
    weighs nothing, one of +inf makes its head NaN, an infinite value of positive weight its column infinite, values of
    both signs NaN. Over Q8_0 an infinity is a block's scale. What stays finite is held to paged_ref's bounds with the
    finite keys' scores and values: parts with infinities are summed key by key, at most 512 roundings here, where the
    bounds have room for 2 (len / 16 + 256)."""
    import torch
    from toy_b200 import paged
    g = torch.Generator(device=cuda).manual_seed(dh)
    n, G = len(lens), H // KV
    width = max(-(-x // P) for x in lens)
    x, y = (torch.randn((n * width, KV, P, dh), generator=g, device=cuda) for _ in range(2))
    q = (torch.randn((n, H, dh), generator=g, device=cuda)).to(R.TORCH[row])
    q[:, :, :32] = q[:, :, :32].abs() + 0.5           # block 0: all of one sign, by the head
    q[:, 1::3, :32] *= -1
    (k, ks), (v, vs) = (pools(t, cache) for t in (x, y))
    table = torch.randperm(n * width, generator=g, device=cuda).int().view(n, width)
    for what in ("minus key", "plus key", "value", "values", "mixed key"):
        pk, pv, pks, pvs = (None if t is None else t.clone() for t in (k, v, ks, vs))
        for b, L in enumerate(lens):
            for at in {L // 3, max(0, L - 1)} if L > 2 else ():
                page, off = int(table[b, at // P]), at % P
                if what == "mixed key":               # products of both signs: NaN
                    if cache == "q8_0":
                        pk[page, :, off, :2] = torch.tensor([5, -5], dtype=torch.int8, device=cuda)
                        pk[page, :, off, 2:32] = 3
                        pks[page, :, off, 0] = math.inf
                    else:
                        pk[page, :, off, 0], pk[page, :, off, 1] = math.inf, -math.inf
                elif "key" in what:
                    sign = -1 if what == "minus key" else 1
                    if cache == "q8_0":
                        pk[page, :, off, :32] = pk[page, :, off, :32].abs().clamp(min=1) * sign
                        pks[page, :, off, 0] = math.inf
                    else:
                        pk[page, :, off, 3] = sign * math.inf
                else:
                    sign = -1 if what == "values" and at == L // 3 else 1
                    if cache == "q8_0":
                        pv[page, :, off, :32] = pv[page, :, off, :32].abs().clamp(min=1) * sign
                        pvs[page, :, off, 0] = math.inf
                    else:
                        pv[page, :, off, 5] = sign * math.inf
        lt = i32(lens, cuda)
        lse = torch.empty((n, H), device=cuda)
        out = paged.attend(paged.PagedCache(pk, pv, pks, pvs), q, table, lt, lse=lse, scale=0.1)
        kd, vd = R.values(pk, pks), R.values(pv, pvs)
        o, l, (absv, _), _ = R.attend(kd, vd, q, table, lens, 0.1)
        _, _, (_, vmax), ds = R.attend(finite(kd), finite(vd), q, table, lens, 0.1)
        bo, bl = R.attend_bounds(finite(o), finite(l), (finite(absv), vmax), ds, lt, dh, q.dtype)
        assert torch.equal(out.isnan(), o.isnan()), what
        assert torch.equal(out.isinf(), o.isinf()) and torch.equal(out[o.isinf()].double(), o[o.isinf()]), what
        ok = o.isfinite()
        assert bool(((out.double() - o).abs()[ok] <= bo[ok]).all()), what
        assert torch.equal(lse.isfinite(), l.isfinite()), what
        ok = l.isfinite()
        assert bool(((lse.double() - l).abs()[ok] <= bl[ok]).all()), what
        again = paged.attend(paged.PagedCache(pk, pv, pks, pvs), q, table, lt, scale=0.1)
        assert torch.equal(torch.nan_to_num(again, nan=7.0), torch.nan_to_num(out, nan=7.0))
    no_error()


# ------------------------------------------------------------------ release
@pytest.mark.parametrize("n,P,width", [(1, 16, 3), (40, 8, 5), (300, 4, 24), (900, 16, 40), (16384, 4, 2)])
@pytest.mark.parametrize("share", [0.02, 0.5, 1.0])
@pytest.mark.parametrize("in_place", [False, True])
def test_release_bad_pages(cuda, n, P, width, share, in_place):
    """Table entries that are no page are cleared and reported, and do not reach the stack; the others do, in order."""
    import random
    from toy_b200 import paged
    from toy_b200._lib import lib
    r = random.Random(n * 7 + int(share * 100))
    lens = [r.choice([0, 1, r.randrange(0, width * P + 1), width * P]) for _ in range(n)]
    lens[0] = width * P
    done = [int(r.random() < 0.7) for _ in range(n)]
    done[0] = 1
    n_pages = n * width + 1
    held = [-(-x // P) for x in lens]
    ids = r.sample(range(n_pages), sum(held))
    table, at, bad = [], 0, 0
    for b in range(n):
        row = ids[at:at + held[b]]
        at += held[b]
        for i in range(held[b]):
            if done[b] and (r.random() < share or (b == 0 and i == 1)):
                row[i] = r.choice([-1, n_pages, 2 ** 31 - 1, -2 ** 31])
                bad += 1
        table.append(row + [-3] * (width - held[b]))
    free = [5, 6]
    cap = free + [-9] * (n_pages - len(free))
    want = list(free)
    for b in range(n):
        if done[b]:
            want += [p for p in table[b][:held[b]] if 0 <= p < n_pages]
    L, D, T, F, S = i32(lens, cuda), i32(done, cuda), i32(table, cuda), i32(cap, cuda), i32([len(free), 9, 9, 9], cuda)
    Lo, So = (L, S) if in_place else (i32([5] * n, cuda), i32([5] * 4, cuda))
    paged.release(L, D, T, F, S, page_size=P, n_pages=n_pages, lens_out=Lo, state_out=So)
    if len(free) + sum(h for h, d in zip(held, done) if d) > len(cap):     # the stack could pass its end: nothing done
        assert So.tolist() == [len(free), 1, 0, 0] and F.tolist() == cap and T.tolist() == table
        return no_error()
    assert bad and lib().tb2_device_error() == 0x5001
    assert So.tolist() == [len(want), 0, 0, len(want) - len(free)]
    assert F[:len(want)].tolist() == want
    assert Lo.tolist() == [0 if d else x for x, d in zip(lens, done)]
    assert T.tolist() == [[-1] * h + row[h:] if d else row for row, h, d in zip(table, held, done)]
    no_error()


# ------------------------------------------------------------------ set-up
FIRST_CALLS = """
import ctypes, sys, time
sys.path[:0] = [{root!r}, {tests!r}]
import torch
import paged_ref as R
from toy_b200 import paged
from toy_b200._lib import lib
dev = torch.device("cuda:0")
g = torch.Generator(device=dev).manual_seed(0)
i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
H, KV, dh, P, n = {H}, {KV}, {dh}, 16, 3
k, v, ks, vs = R.make_pools(12, KV, P, dh, {cache!r}, "heads", g, dev)
qkv = torch.randn((n, (H + 2 * KV) * dh), generator=g, device=dev).to(R.TORCH[{row!r}])
q, kn, vn = (qkv[:, a * dh:b * dh].view(n, b - a, dh) for a, b in ((0, H), (H, H + KV), (H + KV, H + 2 * KV)))
lens, add, done = i32([0, 20, 5]), i32([1, 1, 1]), i32([1, 1, 1])
table = torch.full((n, 4), -1, dtype=torch.int32, device=dev)
table[1, :2], table[2, 0] = i32([7, 3]), 9
free, state = i32([0, 1, 2, 4, 5, 6, 8, 10, 11, 0, 0, 0]), i32([9, 0, 0, 0])
e = lambda m, t=torch.int32: torch.empty(m, dtype=t, device=dev)
out = paged.Plan(e(n), e(4), e(n + 1), e(n, torch.int64), e(n), e(n))
o, qo, tab2, free2, after = torch.empty_like(q.contiguous()), torch.empty_like(q.contiguous()), e((n, 4)), e(12), e(4)
c = paged.PagedCache(k, v, ks, vs)
ws = paged.attend_workspace(dev)
lse = torch.empty((n, H), device=dev)
torch.cuda.synchronize()
gr = torch.cuda.CUDAGraph()
with torch.cuda.graph(gr):
    p = paged.plan(lens, add, table, free, state, page_size=P, n_pages=12, n_tokens=n, out=out)
    paged.append(c, p.slots, kn, vn, q=q, q_out=qo)
    paged.attend(c, qo, table, p.lens, out=o, lse=lse, workspace=ws)
    tab2.copy_(table)
    free2.copy_(free)
    paged.release(p.lens, done, tab2, free2, p.state, page_size=P, n_pages=12, lens_out=e(n), state_out=after)
gr.replay()
torch.cuda.synchronize()
assert out.lens.tolist() == [1, 21, 6] and out.state.tolist() == [8, 0, 3, 1]
assert out.slots.tolist() == [11 * P, 3 * P + 4, 9 * P + 5]
assert after.tolist() == [12, 0, 0, 4] and free2.tolist()[8:] == [11, 7, 3, 9]
w, _, sums, ds = R.attend(R.values(k, ks), R.values(v, vs), q, table, [1, 21, 6], dh ** -0.5)
b, _ = R.attend_bounds(w, w[..., 0], sums, ds, out.lens, dh, q.dtype)
assert bool(((o.double() - w).abs() <= b).all()), float((o.double() - w).abs().max())
assert lib().tb2_device_error() == 0
print("captured first")
"""


@pytest.mark.parametrize("H,KV,dh,row,cache", [(4, 2, 128, "bf16", "bf16"), (12, 1, 96, "f32", "q8_0")])
def test_first_calls_in_a_capture(cuda, H, KV, dh, row, cache):
    """A process whose first calls of the operators are captured: tb2_paged_prepare (PagedCache calls it) has loaded
    and set up what they launch."""
    import subprocess
    tests = os.path.dirname(os.path.abspath(__file__))
    code = FIRST_CALLS.format(root=os.path.dirname(tests), tests=tests, H=H, KV=KV, dh=dh, row=row, cache=cache)
    p = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert p.returncode == 0 and "captured first" in p.stdout, p.stderr[-2000:]


# ------------------------------------------------------------------ unaligned rows, repeats
@pytest.mark.parametrize("row", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("cache", ["f32", "bf16", "q8_0"])
@pytest.mark.parametrize("H,KV,dh,P,lens", [
    (9, 3, 64, 16, [5, 0, 130, 900]), (12, 1, 32, 8, [33, 3000]), (4, 2, 96, 24, [1, 2000, 77]),
    (20, 2, 128, 16, [64, 9000])])
def test_attend_unaligned_rows(cuda, row, cache, H, KV, dh, P, lens):
    """q and out that start at odd elements with odd row strides: the aligned call's results to the bit, nothing around
    out touched; histories of one CTA and split ones."""
    import torch
    from toy_b200 import paged
    g = torch.Generator(device=cuda).manual_seed(H)
    n, width = len(lens), max(-(-x // P) for x in lens)
    k, v, ks, vs = R.make_pools(n * width, KV, P, dh, cache, "heads", g, cuda)
    c = paged.PagedCache(k, v, ks, vs)
    table = torch.randperm(n * width, generator=g, device=cuda).int().view(n, width)
    q = torch.randn((n, H, dh), generator=g, device=cuda).to(R.TORCH[row])
    lt = i32(lens, cuda)
    lse, lse2 = torch.empty((n, H), device=cuda), torch.empty((n, H), device=cuda)
    want = paged.attend(c, q, table, lt, lse=lse)
    W = H * dh
    for at, pad in ((1, 2), (3, 1), (7, 5)):
        qf = torch.zeros(n * (W + pad) + 16, device=cuda, dtype=q.dtype)
        of = torch.full((n * (W + pad) + 16,), 5.0, device=cuda, dtype=q.dtype)
        qv = qf.as_strided((n, H, dh), (W + pad, dh, 1), at)
        ov = of.as_strided((n, H, dh), (W + pad, dh, 1), at)
        qv.copy_(q)
        paged.attend(c, qv, table, lt, out=ov, lse=lse2)
        assert torch.equal(ov, want) and torch.equal(lse2, lse)
        ov.fill_(5.0)
        assert bool((of == 5.0).all())
        # one side aligned, the other not
        got = paged.attend(c, qv, table, lt)
        paged.attend(c, q, table, lt, out=ov)
        assert torch.equal(got, want) and torch.equal(ov, want)
    no_error()


@pytest.mark.parametrize("cache", ["f32", "bf16", "q8_0"])
@pytest.mark.parametrize("lens,H,KV,dh", [([20000], 32, 8, 128), ([5000, 1, 777, 0, 4096], 9, 3, 64),
                                          ([600] * 40, 28, 4, 128)])
def test_attend_repeats_itself(cuda, cache, lens, H, KV, dh):
    """The same inputs in new tensors, with another call between and other work on a second stream: the same bits."""
    import torch
    from toy_b200 import paged
    P, n = 16, len(lens)
    width = max(-(-x // P) for x in lens)

    def state(seed):
        g = torch.Generator(device=cuda).manual_seed(seed)
        k, v, ks, vs = R.make_pools(n * width, KV, P, dh, cache, "heads", g, cuda)
        return (paged.PagedCache(k, v, ks, vs), torch.randn((n, H, dh), generator=g, device=cuda),
                torch.randperm(n * width, generator=g, device=cuda).int().view(n, width), i32(lens, cuda))

    first = paged.attend(*state(1))
    ws, busy = paged.attend_workspace(cuda), torch.randn((4096, 4096), device=cuda)
    side = torch.cuda.Stream()
    for _ in range(4):
        a, b = state(1), state(2)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for _ in range(4):
                busy = busy @ busy * 1e-3
        paged.attend(*b, workspace=ws)
        got = paged.attend(*a, workspace=ws)
        torch.cuda.synchronize()
        assert torch.equal(got, first)
    no_error()


# ------------------------------------------------------------------ gradients
def test_gradients_are_refused(cuda):
    """An input that requires a gradient would get none: refused, but not under torch.no_grad()."""
    import torch
    from toy_b200 import paged
    k = torch.zeros((4, 2, 16, 64), device=cuda)
    c = paged.PagedCache(k, k.clone())
    x = lambda h, g=False: torch.ones((2, h, 64), device=cuda, requires_grad=g)  # noqa: E731
    table, lens, slots = i32([[0], [1]], cuda), i32([1, 1], cuda), torch.tensor([0, 16], device=cuda)
    bias = torch.zeros(8 * 64, device=cuda, requires_grad=True)
    calls = [lambda: paged.attend(c, x(4, True), table, lens), lambda: paged.append(c, slots, x(2, True), x(2)),
             lambda: paged.append(c, slots, x(2), x(2, True)), lambda: paged.append(c, slots, x(2), x(2), q=x(4, True)),
             lambda: paged.append(c, slots, x(2), x(2), q=x(4), bias=bias),
             lambda: paged.attend(c, x(4, True) * 2, table, lens),
             lambda: paged.attend(c, x(4), table, lens, out=x(4, True))]
    for f in calls:
        with pytest.raises(ValueError, match="gradient"):
            f()
        with torch.no_grad():
            f()
    assert not paged.attend(c, x(4), table, lens).requires_grad
    no_error()


# ------------------------------------------------------------------ operands of an f32 cache
@pytest.mark.parametrize("H,KV,dh", [(3, 1, 64), (8, 2, 128), (12, 1, 32), (16, 1, 96)])
def test_attend_f32_values(cuda, H, KV, dh):
    """A request of one key gives that key's value row: its weight is 1, so all that is lost is what the value's two
    halves leave out, at most a unit of its last place (2^-23 of it)."""
    import torch
    from toy_b200 import paged
    g = torch.Generator(device=cuda).manual_seed(dh)
    n = 64
    k, v, _, _ = R.make_pools(n, KV, 16, dh, "f32", "heads", g, cuda)
    v *= 10.0 ** torch.randint(-30, 31, v.shape, generator=g, device=cuda)
    v[0, 0, 0, 0], v[1, 0, 0, 0] = 3.4028234e38, -3.4028234e38       # (the ends of f32: `hi` rounds to infinity)
    q = torch.randn((n, H, dh), generator=g, device=cuda)
    out = paged.attend(paged.PagedCache(k, v), q, torch.arange(n, dtype=torch.int32, device=cuda)[:, None],
                       i32([1] * n, cuda))
    want = v[:, :, 0].repeat_interleave(H // KV, 1).double()
    assert bool(((out.double() - want).abs() <= 2.0 ** -23 * want.abs()).all())
    no_error()


def test_sizes_past_32_bits_are_refused(cuda):
    """Counts that the entry points' 32 bits would cut are refused (they would have been taken modulo 2^32)."""
    import torch
    from toy_b200 import paged
    big = torch.empty(2 ** 32 + 4, dtype=torch.int32, device=cuda)
    i, t = i32([0] * 4, cuda), i32([[0, 0]] * 4, cuda)
    with pytest.raises(ValueError, match="2\\^31"):
        paged.plan(i, i, t, big, i, page_size=16, n_pages=4, n_tokens=0)
    with pytest.raises(ValueError, match="2\\^31"):
        paged.release(i, i, t, big, i, page_size=16, n_pages=4)
    with pytest.raises(ValueError, match="2\\^31"):
        paged.plan(big, i, t, i, i, page_size=16, n_pages=4, n_tokens=0)
    with pytest.raises(ValueError, match="2\\^31"):
        paged.plan(i[:1], i, big[None, :], i, i, page_size=16, n_pages=4, n_tokens=0)
    del big
    torch.cuda.empty_cache()
    no_error()


@pytest.mark.parametrize("cache", ["f32", "f16", "bf16", "q8_0"])
@pytest.mark.parametrize("L", [1, 40, 3000])
def test_attend_all_minus_infinity(cuda, cache, L):
    """A request whose scores are all -inf counts as an empty one; the heads beside it and the next request do not."""
    import torch
    from toy_b200 import paged
    P, dh, width = 16, 64, -(-3000 // 16)
    g = torch.Generator(device=cuda).manual_seed(L)
    k, v, ks, vs = R.make_pools(2 * width, 1, P, dh, cache, "heads", g, cuda)
    c = paged.PagedCache(k, v, ks, vs)
    q = torch.randn((2, 5, dh), generator=g, device=cuda)
    q[:, :2, :32] = q[:, :2, :32].abs() + 0.1
    table = torch.arange(2 * width, dtype=torch.int32, device=cuda).view(2, width)
    lens, lse, base = i32([L, 70], cuda), torch.empty((2, 5), device=cuda), torch.empty((2, 5), device=cuda)
    want = paged.attend(c, q, table, lens, lse=base)
    if cache == "q8_0":
        k[:width, 0, :, :32] = -k[:width, 0, :, :32].abs().clamp(min=1)
        ks[:width, 0, :, 0] = math.inf
    else:
        k[:width, 0, :, 0] = -math.inf
    out = paged.attend(c, q, table, lens, lse=lse)
    assert bool((out[0, :2] == 0).all()) and bool((lse[0, :2] == -math.inf).all())
    assert torch.equal(out[1], want[1]) and torch.equal(lse[1], base[1])
    neg = q[0, :, 0] < 0
    if cache != "q8_0":                                 # scores of +inf
        assert bool(out[0, neg].isnan().all()) and bool(lse[0, neg].isnan().all())
    no_error()


# ------------------------------------------------------------------ captured release
@pytest.mark.parametrize("n,P,width", [(6, 16, 5), (900, 16, 40)])
def test_release_captured(cuda, n, P, width):
    """A release of one CTA and of several in a graph, twice in a row, replayed with other requests done and with an
    entry that is no page, against the eager call."""
    import torch
    from toy_b200 import paged
    from toy_b200._lib import lib
    n_pages = n * width
    gen = torch.Generator(device=cuda).manual_seed(n)
    table0 = torch.randperm(n_pages, generator=gen, device=cuda).int().view(n, width).contiguous()
    lens0 = torch.full((n,), width * P, dtype=torch.int32, device=cuda)

    def world():
        return {"lens": lens0.clone(), "table": table0.clone(), "state": i32([0] * 4, cuda),
                "free": torch.full((n_pages,), -9, dtype=torch.int32, device=cuda),
                "a": torch.zeros(n, dtype=torch.int32, device=cuda), "b": torch.zeros(n, dtype=torch.int32, device=cuda)}

    def step(w):
        for done in ("a", "b"):
            paged.release(w["lens"], w[done], w["table"], w["free"], w["state"], page_size=P, n_pages=n_pages)

    graphed, eager = world(), world()
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        step(graphed)
    for i in range(4):
        for w in (graphed, eager):
            w["lens"].copy_(lens0)
            w["table"].copy_(table0)
            if i == 2:
                w["table"][n // 2, 1], w["table"][0, 0] = n_pages, -5
            w["state"].zero_()
            pick = torch.arange(n, device=cuda) * 2654435761 % 4
            w["a"].copy_(pick == i)
            w["b"].copy_(pick == (i + 1) % 4)
            if i == 2:
                w["a"][n // 2] = w["b"][0] = 1
        gr.replay()
        step(eager)
        for key in ("lens", "table", "state"):
            assert torch.equal(graphed[key], eager[key]), (i, key)
        top = int(eager["state"][0])
        done = int(((eager["a"] != 0) | (eager["b"] != 0)).sum())
        assert top == done * width - (2 if i == 2 else 0)
        free = graphed["free"][:top]
        assert torch.equal(free, eager["free"][:top]) and free.unique().numel() == top and int(free.min()) >= 0
        assert lib().tb2_device_error() == (0x5001 if i == 2 else 0)
