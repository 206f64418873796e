"""Tokens sorted by expert and back (toy_b200.experts): the sort against a host
list (whole numbers, equal), rows moved without a change, sums against 64 bits
within a bound that counts their roundings, gradients against the formula,
differences and autograd."""
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def dt(name):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def choices(T, K, E, seed=0, dropped=0.2, wide=False, same=False):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    ids = torch.randint(0, E, (T, K), device="cuda", generator=g)
    if same:
        ids[:] = E - 1
    ids[torch.rand((T, K), device="cuda", generator=g) < dropped] = -1
    return ids if wide else ids.int()


def host_sort(ids, E):
    flat = ids.flatten().tolist()
    order = [i for e in range(E) for i, x in enumerate(flat) if x == e]
    offsets = [0]
    for e in range(E):
        offsets.append(offsets[-1] + flat.count(e))
    pos = [-1] * len(flat)
    for at, i in enumerate(order):
        pos[i] = at
    return offsets, order + [-1] * (len(flat) - len(order)), pos


def check_sort(r, ids, E):
    import torch
    flat = ids.flatten().long().cpu()
    live = (flat >= 0) & (flat < E)
    n = int(live.sum())
    counts = torch.bincount(flat[live], minlength=E)
    assert r.offsets.tolist() == [0] + counts.cumsum(0).tolist()
    order = torch.where(live, flat, E).sort(stable=True).indices
    order[n:] = -1
    assert torch.equal(r.order.cpu().long(), order)
    pos = torch.full((flat.numel(),), -1)
    pos[order[:n]] = torch.arange(n)
    assert torch.equal(r.pos.cpu().long().flatten(), pos)


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("T,K,E", [(1, 1, 1), (1, 8, 64), (3, 2, 5), (16, 8, 64), (33, 3, 1024), (128, 8, 2),
                                   (129, 8, 31), (4096, 8, 64), (1000, 7, 160), (30011, 3, 7), (40000, 8, 1000)])
def test_sort(cuda, T, K, E, wide):
    from toy_b200 import experts as X
    for dropped, same in ((0.0, False), (0.3, False), (1.0, False), (0.1, True)):
        ids = choices(T, K, E, seed=T + E, dropped=dropped, wide=wide, same=same)
        r = X.sort(ids, E)
        check_sort(r, ids, E)
        if T * K <= 400:
            assert (r.offsets.tolist(), r.order.tolist(), r.pos.flatten().tolist()) == host_sort(ids, E)


def rows_in(n, d, dtype, seed, pad=0, shift=0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    buf = torch.zeros(n * (d + pad) + shift + 16, device="cuda", dtype=dtype)
    x = buf[shift:shift + n * (d + pad)].view(n, d + pad)[:, :d]
    x.copy_(torch.randn((n, d), device="cuda", generator=g))
    return x


SHAPES = [(1, 1, 1, 1, 0, 0), (5, 2, 4, 7, 0, 0), (16, 8, 64, 2048, 0, 0), (300, 3, 8, 1000, 0, 0),
          (300, 3, 8, 1001, 0, 0), (70, 8, 16, 256, 8, 8), (70, 8, 16, 250, 3, 1), (40, 16, 64, 72, 0, 0),
          (1000, 5, 128, 64, 0, 0), (2500, 1, 3, 96, 0, 0), (1501, 2, 16, 136, 0, 0), (111, 4, 8, 520, 8, 8),
          (67, 6, 64, 1032, 0, 0), (130, 7, 9, 64, 0, 0), (50, 9, 32, 256, 0, 0), (1, 1, 8, 72, 0, 0)]


@pytest.mark.parametrize("name", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("T,K,E,d,pad,shift", SHAPES)
def test_rows(cuda, T, K, E, d, pad, shift, name):
    """dispatch, combine and their gradients, at odd widths, strides and starts."""
    import torch
    from toy_b200 import experts as X
    t = dt(name)
    h = torch.finfo(t).eps / 2
    ids = choices(T, K, E, seed=d)
    r = X.sort(ids, E)
    n, order, pos = int(r.offsets[-1]), r.order.cpu().long(), r.pos.cpu().long()
    x, z, dy = rows_in(T, d, t, 1, pad, shift), rows_in(T * K, d, t, 2, pad, shift), rows_in(T, d, t, 3, pad, shift)
    w = torch.randn((T, K), device="cuda")
    w[pos.cuda() < 0] = float("nan")                  # a slot of no expert takes no part, whatever its weight
    z[n:] = float("nan")                              # nor does a row of none
    keep = rows_in(T * K, d, t, 4, pad, shift)
    xs = X.dispatch(x, r, out=keep.clone())
    assert torch.equal(xs[:n].cpu(), x.cpu()[order[:n] // K])
    assert torch.equal(xs[n:], keep[n:])
    assert (X.dispatch(x, r)[n:] == 0).all()
    on = pos >= 0
    z64, w64, at = z.double().cpu(), torch.where(on, w.double().cpu(), 0.0), pos.clamp(min=0)
    z64[n:] = 0
    terms = torch.stack([w64[:, k, None] * torch.where(on[:, k, None], z64[at[:, k]], 0.0) for k in range(K)])
    for res in (None, dy):
        base = torch.zeros((T, d), dtype=torch.float64) if res is None else res.double().cpu()
        y = X.combine(z, r, w, residual=res)
        want, size = base + terms.sum(0), base.abs() + terms.abs().sum(0)
        # K products summed one by one: K roundings of at most the terms' sum; then the result's own
        tol = (K + 1) * U * size * (1 + h) + h * want.abs() + 2.0 ** -25 * (name == "f16")
        assert ((y.double().cpu() - want).abs() <= tol).all()
    buf = dy.clone()
    assert torch.equal(X.combine(z, r, w, residual=buf, out=buf), X.combine(z, r, w, residual=dy))
    dz, dw = X.combine_grad(dy, z, r, w)
    dys, ws = dy.double().cpu()[order[:n] // K], w.double().cpu().flatten()[order[:n], None]
    assert ((dz[:n].double().cpu() - dys * ws).abs() <= (h + U) * (dys * ws).abs() + 2.0 ** -25 * (name == "f16")).all()
    assert (dz[n:] == 0).all()
    got = X.combine_grad(dy, z, r, w, out=keep.clone())[0]
    assert torch.equal(got[:n], dz[:n]) and torch.equal(got[n:], keep[n:])
    prod = dys * z64[:n]
    want = torch.zeros(T * K, dtype=torch.float64)
    want[order[:n]] = prod.sum(-1)
    size = torch.zeros(T * K, dtype=torch.float64)
    size[order[:n]] = prod.abs().sum(-1)
    # a lane sums at most d / 32 + 8 products in a row, then five halvings
    tol = (d / 32 + 14) * U * size
    assert ((dw.double().cpu().flatten() - want).abs() <= tol).all()
    assert torch.equal(dw.cpu()[~on], torch.zeros(int((~on).sum())))
    inplace = z.clone()
    assert torch.equal(X.combine_grad(dy, inplace, r, w, out=inplace)[0][:n], dz[:n])
    dx = X.dispatch_grad(z, r)
    terms = torch.stack([torch.where(on[:, k, None], z64[at[:, k]], 0.0) for k in range(K)])
    tol = (K * U * terms.abs().sum(0)) * (1 + h) + h * terms.sum(0).abs() + 2.0 ** -25 * (name == "f16")
    assert ((dx.double().cpu() - terms.sum(0)).abs() <= tol).all()


def test_autograd_and_differences(cuda):
    import torch
    from toy_b200 import experts as X
    T, K, E, d = 40, 3, 8, 33
    r = X.sort(choices(T, K, E, seed=1), E)
    mix = torch.randn((d, d), device="cuda") / d ** 0.5
    x, w, res = (torch.randn(s, device="cuda", requires_grad=True) for s in ((T, d), (T, K), (T, d)))
    g = torch.randn((T, d), device="cuda")
    y = X.combine(torch.tanh(X.dispatch(x, r) @ mix), r, w, residual=res)
    (y * g).sum().backward()
    pos = r.pos.cpu().long()

    def f(x, w, res):
        z = torch.tanh(x @ mix.double().cpu())
        return ((res + (torch.where(pos >= 0, w, 0.0).sum(-1)[:, None] * z)) * g.double().cpu()).sum()

    at = [t.detach().double().cpu() for t in (x, w, res)]
    for i, t in enumerate((x, w, res)):
        v = torch.randn(t.shape, dtype=torch.float64)
        lo, hi = list(at), list(at)
        lo[i], hi[i] = at[i] - 1e-5 * v, at[i] + 1e-5 * v
        num = (f(*hi) - f(*lo)) / 2e-5
        # f32 sums of 33 terms through a product of f32: 2^-18 of the terms
        assert abs((t.grad.double().cpu() * v).sum() - num) <= 1e-4 * (t.grad.double().cpu().abs() * v.abs()).sum()
    # a broadcast gradient, and only the weights' gradient wanted
    w2 = w.detach().clone().requires_grad_()
    z = torch.randn((T * K, d), device="cuda")
    X.combine(z, r, w2).sum().backward()
    want = X.combine_grad(torch.ones((T, d), device="cuda"), z, r, w2.detach())[1]
    assert torch.equal(w2.grad, want)
    z2 = z.clone().requires_grad_()
    X.combine(z2, r).sum().backward()
    assert torch.equal(z2.grad[int(r.offsets[-1]):], torch.zeros_like(z2.grad[int(r.offsets[-1]):]))
    with pytest.raises(ValueError):
        X.combine_grad(g, z2, r, w)


def test_streams_and_graphs(cuda):
    import torch
    from toy_b200 import experts as X
    X.prepare()
    T, K, E, d = 600, 4, 16, 128
    ids, x = choices(T, K, E), rows_in(T, d, torch.bfloat16, 1)
    w = torch.rand((T, K), device="cuda")
    outs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            r = X.sort(ids, E)
            y = X.combine(X.dispatch(x, r), r, w)
        outs.append((graph, r, y))
    ids.copy_(choices(T, K, E, seed=5))
    for graph, _, _ in outs:
        graph.replay()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        want = X.sort(ids, E)
        y = X.combine(X.dispatch(x, want), want, w)
    torch.cuda.current_stream().wait_stream(st)
    check_sort(want, ids, E)
    for _, r, got in outs:
        assert all(torch.equal(a, b) for a, b in zip(r, want)) and torch.equal(got, y)


def test_values_out_of_range(cuda):
    import torch
    from toy_b200 import experts as X
    from toy_b200._lib import lib
    assert lib().tb2_device_error() == 0
    for wide in (False, True):
        ids = choices(50, 4, 9, wide=wide)
        ids[7, 2] = 9 if not wide else 2 ** 40
        r = X.sort(ids, 9)
        assert lib().tb2_device_error() == 0x5102
        ids[7, 2] = -1
        assert all(torch.equal(a, b) for a, b in zip(r, X.sort(ids, 9)))
    x = torch.randn((50, 16), device="cuda")
    short = X.dispatch(x, r, out=torch.zeros((100, 16), device="cuda"))
    assert lib().tb2_device_error() == 0x5103
    assert torch.equal(short, X.dispatch(x, r)[:100])
    assert lib().tb2_device_error() == 0


def test_refusals(cuda):
    import torch
    from toy_b200 import experts as X
    ids = choices(6, 2, 4)
    r = X.sort(ids, 4)
    x, z, w = (torch.randn(s, device="cuda") for s in ((6, 32), (12, 32), (6, 2)))
    for bad in (lambda: X.sort(ids.float(), 4), lambda: X.sort(ids, 0), lambda: X.sort(ids, 1025),
                lambda: X.sort(ids.t(), 4), lambda: X.sort(ids.flatten(), 4), lambda: X.sort(ids.cpu(), 4),
                lambda: X.dispatch(x[:5], r), lambda: X.dispatch(x.double(), r), lambda: X.dispatch(x.cpu(), r),
                lambda: X.dispatch(x[:, :1].expand(6, 32), r), lambda: X.dispatch(x, r, out=z.half()),
                lambda: X.dispatch(x, r, out=z[:, :31]), lambda: X.combine(z, r, w.half()),
                lambda: X.combine(z, r, w[:, :1]), lambda: X.combine(z, r, w, residual=x.half()),
                lambda: X.combine(z, r, w, out=x[:5]), lambda: X.combine(z, r._replace(pos=r.pos.long()), w),
                lambda: X.dispatch(x.requires_grad_(), r, out=z), lambda: X.combine_grad(x[:, :16], z, r, w)):
        with pytest.raises(ValueError):
            bad()
    e = torch.empty((0, 2), dtype=torch.int32, device="cuda")
    r0 = X.sort(e, 4)
    assert r0.offsets.tolist() == [0] * 5 and X.dispatch(x.detach()[:0], r0).shape == (0, 32)
    assert X.combine(z[:0], r0, w[:0]).shape == (0, 32)
