"""Token log probabilities (toy_b200.logprobs) against their definition in 64
bits, within bounds that count the roundings; their gradient against the
formula, against differences, and through autograd; refusals that need a GPU."""
import math

import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24          # half a step of f32, relative


def half(dtype):
    import torch
    return torch.finfo(dtype).eps / 2


def dt(name):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def make(n, V, dtype, seed=0, pad=0, shift=0, spread=3.0):
    """Logits [n, V] inside rows of V + pad values, `shift` values behind the buffer's start."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    buf = torch.zeros(n * (V + pad) + shift, device="cuda", dtype=dtype)
    x = buf[shift:].view(n, V + pad)[:, :V]
    x.copy_(torch.randn((n, V), device="cuda", generator=g) * spread)
    t = torch.randint(0, V, (n,), device="cuda", generator=g)
    return x, t


def reference(x, t, scale, top):
    """ln p [n, V], logprob, entropy, ids and the sums' mean |scale (x - max)|, in 64 bits on the host."""
    import torch
    x64 = x.double().cpu()
    z = x64 * scale
    m = z.amax(-1, keepdim=True)
    d = torch.where(m == -math.inf, torch.full_like(z, -math.inf), z - m)
    e = torch.where(d == -math.inf, torch.zeros_like(d), d.exp())
    s = e.sum(-1, keepdim=True)
    lp = torch.where(s > 0, d - s.log(), torch.full_like(d, -math.inf))
    p = torch.where(s > 0, e / s, torch.zeros_like(e))
    plp = torch.where(p > 0, p * lp, torch.zeros_like(p))
    tok = t.cpu()
    got = lp.gather(1, tok.clamp(min=0)[:, None])[:, 0]
    order = (x64 + 0.0).sort(dim=-1, descending=True, stable=True).indices[:, :top]
    mean = torch.where(p > 0, p * d.abs(), torch.zeros_like(p)).sum(-1)
    return {"lp": lp, "p": p, "logprob": torch.where(tok < 0, torch.zeros_like(got), got), "entropy": -plp.sum(-1),
            "ids": order, "mean": mean, "lns": torch.where(s > 0, s.log(), torch.zeros_like(s))[:, 0], "d": d}


def sum_error(r, V):
    """Bound of ln s's error: every term is off by its exponent's three roundings (difference, constant, product) and
    by ex2's 2^-22, the sum by a thread's chain and the tree behind it. (A thread has two chains of every second value,
    of V / 256 where a row has 128 threads, and of at most 64, V / 256 + 32, where one of 8192 or fewer has 64.)"""
    return U * (3 * r["mean"] + 4 + V / 256 + 80 + 2 * r["lns"])


def bound(r, d, V):
    """Of ln p at a logit d below the maximum: ln s's, and the roundings of scale d, of ln s and of their difference."""
    return sum_error(r, V) + U * 3 * (d.abs() + r["lns"])


def close(got, want, tol):
    import torch
    got = got.double().cpu()
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf])
    off = (got - want).abs()[~inf]
    assert (off <= tol.expand_as(want)[~inf]).all(), (off.max(), off / tol.expand_as(want)[~inf])


def taken(res, rows):
    return type(res)(*(None if a is None else a[rows] for a in res))


def check(x, t, scale=1.0, top=0, r=None, rows=slice(None)):
    """A call on all of x, whose `rows` are looked at."""
    import torch
    from toy_b200 import logprobs as L
    V = x.shape[1]
    got = L.token_logprobs(x, t, scale=scale, entropy=True, top=top)
    again = L.token_logprobs(x, t, scale=scale, entropy=True, top=top)
    for a, b in zip(got, again):
        assert a is None or torch.equal(a, b)
    got, x, t = taken(got, rows), x[rows], t[rows]
    scale = torch.tensor(scale, dtype=torch.float32).double().item()
    r = r or reference(x, t, scale, top)
    live = t.cpu() >= 0
    dt_ = torch.where(live, r["d"].gather(1, t.cpu().clamp(min=0)[:, None])[:, 0], torch.zeros(len(live)).double())
    close(got.logprob, r["logprob"], bound(r, torch.where(dt_.isinf(), torch.zeros_like(dt_), dt_), V))
    # H = ln s - scale u / s: u's terms round as s's do, and twice more
    close(got.entropy, r["entropy"], sum_error(r, V) * (1 + r["mean"]) + U * (6 * r["mean"] + 4 * r["lns"]))
    if top:
        assert torch.equal(got.top_ids.cpu(), r["ids"])
        d = r["d"].gather(1, r["ids"])
        d0 = torch.where(d.isinf(), torch.zeros_like(d), d)
        tol = bound({k: r[k][:, None] for k in ("mean", "lns")}, d0, V)
        close(got.top_logprobs, r["lp"].gather(1, r["ids"]), tol)
    return got


SIZES = [(1, 1), (1, 2), (3, 7), (2, 8), (5, 31), (19, 257), (700, 300), (18, 1000), (40, 4099), (1, 50303),
         (19, 50303), (160, 20001), (300, 9000), (1300, 2048), (1300, 33), (1185, 100), (1190, 4097), (700, 20001)]


@pytest.mark.parametrize("name", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,V", SIZES)
def test_sizes(cuda, n, V, name):
    x, t = make(n, V, dt(name), seed=V + n)
    check(x, t, top=min(V, 20))


@pytest.mark.parametrize("name,V", [("f32", 28001), ("bf16", 56005), ("f16", 60001)])
@pytest.mark.parametrize("n", [591, 593, 600, 888, 889, 1185])
def test_rounds_with_a_rest(cuda, n, V, name):
    """More rows than run at once: those of the last round may be split."""
    x, t = make(n, V, dt(name), seed=n)
    x[n - 1] = -math.inf
    t[n - 2] = -1
    rows = [0, 1, 295, 590, n - 2, n - 1] + [i for i in (591, 592, 593, 887, 888, 1183, 1184) if i < n]
    check(x, t, scale=0.7, top=7 if n % 2 else 0, rows=rows)
    check_grad(x, t, scale=0.7, top=3 if n % 2 else 0, entropy=n % 2 == 0, rows=rows)


@pytest.mark.parametrize("name", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("pad,shift", [(0, 1), (1, 0), (3, 5), (8, 0), (5, 8)])
@pytest.mark.parametrize("n,V", [(3, 1003), (700, 515), (2, 6), (1200, 1003), (600, 9001)])
def test_rows_off_their_boundaries(cuda, n, V, pad, shift, name):
    x, t = make(n, V, dt(name), seed=7, pad=pad, shift=shift)
    check(x, t, scale=0.7, top=min(V, 32))


@pytest.mark.parametrize("top", [1, 2, 31, 32])
@pytest.mark.parametrize("scale", [1e-3, 0.5, 1.0, 3.0])
def test_top_and_scale(cuda, top, scale):
    import torch
    x, t = make(30, 3001, torch.float32, seed=top)
    t[::3] = -1 - t[::3]
    check(x, t, scale=scale, top=top)


@pytest.mark.parametrize("name", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,V", [(2, 70), (3, 30001), (900, 8003), (1200, 2003)])
def test_equal_logits(cuda, n, V, name):
    """Flat rows, rows of two values, rows that rise or fall: ties go to the lower index."""
    import torch
    x, t = make(n, V, dt(name))
    x[0] = 0.5
    x[1] = (torch.arange(V, device="cuda") % 3 == 1).to(x.dtype)
    if n > 2:
        x[2] = torch.arange(V, device="cuda").to(x.dtype) * 2.0 ** -9
    if n > 5:
        x[3] = -torch.arange(V, device="cuda").to(x.dtype) * 2.0 ** -9
        x[4] = 0.0
        x[4, ::2] = -0.0
        x[5] = -1.0
        x[5, V - 5:] = 1.0            # five stand out, at the end; the rest ties
    check(x, t, top=32)


@pytest.mark.parametrize("name", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,V", [(12, 90), (12, 9001), (900, 2003), (1200, 2003), (600, 20003)])
def test_masks(cuda, n, V, name):
    """-inf and the type's lowest value; rows that they leave one word, few words or none."""
    import torch
    x, t = make(n, V, dt(name), seed=3)
    low = torch.finfo(x.dtype).min
    x[0] = -math.inf
    x[1] = low
    x[2] = -math.inf
    x[2, V // 2] = 1.25
    x[3] = low
    x[3, V - 1] = -2.0
    x[4, 7:] = -math.inf
    x[5, :-7] = -math.inf
    x[6] = -math.inf
    x[6, 3::5] = torch.arange(len(range(3, V, 5)), device="cuda").to(x.dtype) * 2.0 ** -8
    x[7] = torch.finfo(x.dtype).max
    x[8] = -math.inf
    x[8, :: V // 4] = low
    t[2], t[4], t[5] = V // 2, 80, 3
    x[9, t[9]] = -math.inf
    t[10] = -5
    check(x, t, top=32)


def test_not_a_number(cuda):
    """A NaN or +inf makes its row's probabilities NaN, and no other's; NaN counts as the largest."""
    import torch
    from toy_b200 import logprobs as L
    for n, V in ((6, 5000), (700, 5000), (1200, 4000)):
        x, t = make(n, V, torch.float32, seed=1)
        want = reference(x, t, 1.0, 8)
        x[1, 40], x[2, V - 1], x[4, 7], x[4, 9] = math.nan, math.inf, math.nan, -math.nan
        got = L.token_logprobs(x, t, entropy=True, top=8)
        for r in (1, 2, 4):
            assert got.logprob[r].isnan() and got.entropy[r].isnan() and got.top_logprobs[r].isnan().all()
        assert got.top_ids[1, 0] == 40 and got.top_ids[2, 0] == V - 1 and got.top_ids[4, :2].tolist() == [7, 9]
        ok = [r for r in range(n) if r not in (1, 2, 4)]
        assert got.logprob[ok].isfinite().all() and torch.equal(got.top_ids[ok].cpu(), want["ids"][ok])
        d = L.token_logprobs_grad(x, t, got, torch.ones(n, device="cuda"))
        assert d[1].isnan().any() and d[ok].isfinite().all()


def grad_reference(x, t, scale, r, gl, gh, ids, gt):
    import torch
    p, lp = r["p"], r["lp"]
    some = (p.sum(-1) > 0)[:, None]
    g = torch.zeros(x.shape[0], dtype=torch.float64) if gl is None else gl.double().cpu()
    g = torch.where(t.cpu() >= 0, g, torch.zeros_like(g))
    own = torch.zeros_like(p).scatter_add_(1, t.cpu().clamp(min=0)[:, None], g[:, None])
    a = g.clone()
    if gt is not None:
        own.scatter_add_(1, ids.cpu(), gt.double().cpu())
        a += gt.double().cpu().sum(-1)
    d = own - a[:, None] * p
    if gh is not None:
        plp = torch.where(p > 0, p * lp, torch.zeros_like(p))
        d -= gh.double().cpu()[:, None] * (plp + p * r["entropy"][:, None])
    return torch.where(some, d * scale, torch.zeros_like(d)), a


def check_grad(x, t, scale=1.0, top=0, entropy=True, out=None, seed=5, token=True, rows=None):
    import torch
    from toy_b200 import logprobs as L
    n, V = x.shape
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    gl, gh, gt = rnd(n) if token else None, rnd(n) if entropy else None, rnd(n, top) if top else None
    res = L.token_logprobs(x, t, scale=scale, entropy=entropy, top=top)
    s64 = torch.tensor(scale, dtype=torch.float32).double().item()
    got = L.token_logprobs_grad(x, t, res, gl, grad_entropy=gh, grad_top=gt, scale=scale, out=out)
    if rows is not None:
        res, x, t, got = taken(res, rows), x[rows], t[rows], got[rows]
        gl, gh, gt = (None if a is None else a[rows] for a in (gl, gh, gt))
    r = reference(x, t, s64, top)
    want, a = grad_reference(x, t, s64, r, gl, gh, res.top_ids, gt)
    # p is off by its exponent's roundings, ex2's and ln s's error; the words' own gradients are sums of a few terms
    lp = torch.where(r["lp"].isinf(), torch.zeros_like(r["lp"]), r["lp"]).abs()
    rel = sum_error(r, V)[:, None] + U * (4 * lp + 2 * r["lns"][:, None] + 8)
    coef = a.abs()[:, None] + (gh.abs().double().cpu()[:, None] * (lp + r["entropy"][:, None]) if entropy else 0)
    own = torch.zeros_like(want)
    if token:
        own.scatter_add_(1, t.cpu().clamp(min=0)[:, None], gl.abs().double().cpu()[:, None])
    if top:
        own.scatter_add_(1, res.top_ids.cpu(), gt.abs().double().cpu())
    sums = (gl.abs().double().cpu() if token else 0) + (gt.abs().double().cpu().sum(-1) if top else 0)
    tol = s64 * (r["p"] * (rel * coef + U * 40 * (sums[:, None] if token or top else 0)) + U * 40 * own)
    if entropy:   # the entropy read is off itself
        tol = tol + s64 * r["p"] * gh.abs().double().cpu()[:, None] * \
            (sum_error(r, V) * (2 + r["mean"]) + U * 8 * (r["mean"] + r["lns"]))[:, None]
    tiny = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}[x.dtype]
    tol = tol * (1 + half(x.dtype)) + half(x.dtype) * want.abs() + tiny * (1 + s64 * coef.max().item())
    off = (got.double().cpu() - want).abs()
    assert (off <= tol).all(), ((off / tol).max(), off.max())
    return got


@pytest.mark.parametrize("name", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,V", SIZES)
def test_grad_sizes(cuda, n, V, name):
    x, t = make(n, V, dt(name), seed=V + n)
    t[n // 2] = -1
    check_grad(x, t, top=min(V, 4))
    check_grad(x, t, scale=1.5, entropy=False)


@pytest.mark.parametrize("name", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("pad,shift,opad,oshift", [(0, 1, 0, 0), (1, 0, 0, 0), (3, 5, 2, 1), (0, 0, 3, 3),
                                                  (8, 8, 1, 0)])
def test_grad_rows_off_their_boundaries(cuda, pad, shift, opad, oshift, name):
    import torch
    for n, V in ((3, 1003), (700, 515), (2, 6), (1, 40001), (600, 9001)):
        x, t = make(n, V, dt(name), seed=7, pad=pad, shift=shift)
        buf = torch.full((n * (V + opad) + oshift + 32,), 7.0, device="cuda", dtype=x.dtype)
        out = buf[oshift:oshift + n * (V + opad)].view(n, V + opad)[:, :V]
        check_grad(x, t, top=min(V, 5), out=out)
        whole = buf.clone()
        whole[oshift:oshift + n * (V + opad)].view(n, V + opad)[:, :V] = 7.0
        assert (whole == 7.0).all()          # nothing beside the rows is written


@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_grad_in_place(cuda, name):
    import torch
    from toy_b200 import logprobs as L
    for n, V, pad in ((5, 70001, 0), (900, 1003, 5), (1, 300, 0), (600, 9001, 3), (600, 30001, 0)):
        x, t = make(n, V, dt(name), seed=2, pad=pad)
        res = L.token_logprobs(x, t, entropy=True, top=16)
        g = torch.randn(n, device="cuda")
        gt = torch.randn((n, 16), device="cuda")
        want = L.token_logprobs_grad(x, t, res, g, grad_entropy=g, grad_top=gt)
        got = L.token_logprobs_grad(x, t, res, g, grad_entropy=g, grad_top=gt, out=x)
        assert got.data_ptr() == x.data_ptr() and torch.equal(got, want)


def test_grad_masks_and_repeats(cuda):
    """Masked words and rows, padding, the same word several times among the alternatives."""
    import torch
    from toy_b200 import logprobs as L
    x, t = make(8, 5003, torch.float32, seed=9)
    x[0] = -math.inf
    x[1] = torch.finfo(torch.float32).min
    x[2, 5:] = -math.inf
    x[3, ::2] = -math.inf
    t[2], t[3], t[4] = 3, 1, -9
    check_grad(x, t, top=5)
    ids = torch.zeros((8, 6), dtype=torch.int64, device="cuda") + torch.arange(8, device="cuda")[:, None]
    ids[:, 3:] += 4000
    t = torch.arange(8, device="cuda")          # the token among them too
    res = L.token_logprobs(x, t, entropy=True)._replace(top_ids=ids)
    gl, gt = torch.randn(8, device="cuda"), torch.randn((8, 6), device="cuda")
    got = L.token_logprobs_grad(x, t, res, gl, grad_top=gt)
    r = reference(x, t, 1.0, 0)
    want, _ = grad_reference(x, t, 1.0, r, gl, None, ids, gt)
    assert (got.double().cpu() - want).abs().max() <= 1e-5      # sums of seven terms of a few units: 2^-17 at most
    # (word 4002 is an alternative of row 2, and has a gradient of its own at probability 0 too)
    assert (got[0] == 0).all() and (got[2, 5:4002] == 0).all() and (got[2, 4003:] == 0).all()


def test_grad_against_differences(cuda):
    import torch
    from toy_b200 import logprobs as L
    x, t = make(6, 700, torch.float32, seed=4)
    gl, gh, gt = (torch.randn(s, device="cuda") for s in ((6,), (6,), (6, 3)))
    res = L.token_logprobs(x, t, scale=0.75, entropy=True, top=3)
    d = L.token_logprobs_grad(x, t, res, gl, grad_entropy=gh, grad_top=gt, scale=0.75).double().cpu()
    ids = res.top_ids.cpu()

    def f(z):
        lp = torch.log_softmax(z * 0.75, -1)
        h = -(lp.exp() * lp).sum(-1)
        return (lp.gather(1, t.cpu()[:, None])[:, 0] * gl.double().cpu() + h * gh.double().cpu()).sum() + \
            (lp.gather(1, ids) * gt.double().cpu()).sum()

    x64 = x.double().cpu()
    for k in range(5):
        v = torch.randn(x.shape, dtype=torch.float64, generator=torch.Generator().manual_seed(k))
        h = 1e-5
        num = (f(x64 + h * v) - f(x64 - h * v)) / (2 * h)
        # differences are off by h^2 of third derivatives of order 1, the gradient by some 2^-20 of its terms
        assert abs((d * v).sum() - num) <= 1e-4 * (d.abs() * v.abs()).sum()


def test_autograd(cuda):
    import torch
    from toy_b200 import logprobs as L
    x, t = make(9, 4001, torch.float32, seed=6)
    t[4] = -1
    w = torch.randn((9, 4), device="cuda")
    a = x.clone().requires_grad_()
    r = L.token_logprobs(a, t, scale=1.25, entropy=True, top=4)
    assert not r.stats.requires_grad and not r.top_ids.requires_grad
    (r.logprob.sum() * 0.5 + (r.entropy * w[:, 0]).mean() + (r.top_logprobs * w).sum()).backward()
    res = L.token_logprobs(x, t, scale=1.25, entropy=True, top=4)
    want = L.token_logprobs_grad(x, t, res, torch.full((9,), 0.5, device="cuda"),
                                 grad_entropy=(w[:, 0] * (torch.ones((), device="cuda") / 9)).contiguous(), grad_top=w,
                                 scale=1.25)
    # (the same kernel; w / 9 may be rounded otherwise on the way back)
    assert torch.allclose(a.grad, want, rtol=1e-5, atol=1e-9)
    # only one of the outputs used, another not asked for; the gradient of a broadcast logit row is refused
    b = x.clone().requires_grad_()
    L.token_logprobs(b, t).logprob.sum().backward()
    want = L.token_logprobs_grad(x, t, L.token_logprobs(x, t), torch.ones(9, device="cuda"))
    assert torch.equal(b.grad, want)
    with pytest.raises(ValueError):
        L.token_logprobs(x[:1].expand(9, -1).requires_grad_(), t)
    with torch.no_grad():
        assert not L.token_logprobs(b, t).logprob.requires_grad


def test_written_tensors_are_noted(cuda):
    """What autograd saved of logits that a gradient was written over is refused, not used."""
    import torch
    from toy_b200 import logprobs as L
    x, t = make(4, 100, torch.float32)
    a = x.clone().requires_grad_()
    z = a * 2.0
    r = L.token_logprobs(z, t)
    with torch.no_grad():
        L.token_logprobs_grad(z, t, r, torch.ones(4, device="cuda"), out=z)
    with pytest.raises(RuntimeError):
        r.logprob.sum().backward()


def test_streams_and_graphs(cuda):
    import torch
    from toy_b200 import logprobs as L
    L.prepare()
    x, t = make(20, 30011, torch.bfloat16, seed=8)
    g = torch.randn(20, device="cuda")
    want = L.token_logprobs(x, t, entropy=True, top=5)
    want_d = L.token_logprobs_grad(x, t, want, g, grad_entropy=g)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = L.token_logprobs(x, t, entropy=True, top=5)
    torch.cuda.current_stream().wait_stream(st)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = L.token_logprobs(x, t, entropy=True, top=5)
            d = L.token_logprobs_grad(x, t, got, g, grad_entropy=g)
        graphs.append((graph, got, d))
    y, t2 = make(20, 30011, torch.bfloat16, seed=18)
    x.copy_(y)
    t.copy_(t2)
    for graph, _, _ in graphs:
        graph.replay()
    want = L.token_logprobs(y, t2, entropy=True, top=5)
    want_d = L.token_logprobs_grad(y, t2, want, g, grad_entropy=g)
    for _, got, d in graphs:
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(d, want_d)


def test_tokens_outside_the_vocabulary(cuda):
    import torch
    from toy_b200 import logprobs as L
    from toy_b200._lib import lib
    assert lib().tb2_device_error() == 0
    x, t = make(40, 900, torch.float32)
    t[3] = 900
    got = L.token_logprobs(x, t)
    assert got.logprob[3].isnan() and got.logprob[[0, 1, 2, 4]].isfinite().all()
    assert lib().tb2_device_error() == 0x5101
    d = L.token_logprobs_grad(x, t, got, torch.ones(40, device="cuda"))
    assert (d[3] == 0).all() and lib().tb2_device_error() == 0x5101
    t[3] = 2 ** 40
    ids = torch.zeros((40, 2), dtype=torch.int64, device="cuda")
    ids[5, 1] = -1
    got = L.token_logprobs(x, t)._replace(top_ids=ids)
    assert lib().tb2_device_error() == 0x5101
    L.token_logprobs_grad(x, t, got, None, grad_top=torch.ones((40, 2), device="cuda"))
    assert lib().tb2_device_error() == 0x5101


def test_offsets_past_32_bits(cuda):
    """Rows that lie more than 2^31 values behind the first."""
    import torch
    from toy_b200 import logprobs as L
    V, n = 50000, 3
    buf = torch.zeros((n, 1100 * 10 ** 6), device="cuda", dtype=torch.float16)
    x = buf[:, 1000 * 10 ** 6: 1000 * 10 ** 6 + V]
    y, t = make(n, V, torch.float16)
    x.copy_(y)
    a, b = L.token_logprobs(x, t, entropy=True, top=7), L.token_logprobs(y.contiguous(), t, entropy=True, top=7)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    g = torch.ones(n, device="cuda")
    want = L.token_logprobs_grad(y, t, b, g)
    assert torch.equal(L.token_logprobs_grad(x, t, a, g, out=x), want)
    assert (buf[:, 1000 * 10 ** 6 - 64:1000 * 10 ** 6] == 0).all()


def test_refusals(cuda):
    import torch
    from toy_b200 import logprobs as L
    x, t = make(4, 100, torch.float32)
    res = L.token_logprobs(x, t)
    g = torch.ones(4, device="cuda")
    for bad in (lambda: L.token_logprobs(x[0], t), lambda: L.token_logprobs(x.double(), t),
                lambda: L.token_logprobs(x, t.int()), lambda: L.token_logprobs(x, t[:3]),
                lambda: L.token_logprobs(x, t.cpu()), lambda: L.token_logprobs(x.t().contiguous().t(), t),
                lambda: L.token_logprobs(x, t, scale=0.0), lambda: L.token_logprobs(x, t, scale=math.inf),
                lambda: L.token_logprobs(x, t, scale=-1.0), lambda: L.token_logprobs(x, t, scale=1e-60),
                lambda: L.token_logprobs(x, t, top=33), lambda: L.token_logprobs(x[:, :3], t, top=4),
                lambda: L.token_logprobs(x, t, top=-1), lambda: L.token_logprobs(x[:1].expand(4, -1), t),
                lambda: L.token_logprobs_grad(x, t, res, g, grad_entropy=g),
                lambda: L.token_logprobs_grad(x, t, res, g.double()), lambda: L.token_logprobs_grad(x, t, res, g[:3]),
                lambda: L.token_logprobs_grad(x, t, res, g, grad_top=torch.ones((4, 2), device="cuda")),
                lambda: L.token_logprobs_grad(x, t, res, g, out=torch.empty((4, 100), device="cuda").half()),
                lambda: L.token_logprobs_grad(x.clone().requires_grad_(), t, res, g)):
        with pytest.raises(ValueError):
            bad()
    assert L.token_logprobs(x[:0], t[:0], entropy=True, top=3).top_ids.shape == (0, 3)
    assert L.token_logprobs_grad(x[:0], t[:0], L.token_logprobs(x[:0], t[:0]), g[:0]).shape == (0, 100)
