"""AdamW over many tensors (toy_b200.multi_adamw) against the step's definition
in 64 bits: weights within a bound that counts the roundings, f32 moments too,
8-bit moments equal to the exact values rounded once."""
import math

import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
BLOCK = 256


def dt(name):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def hp_row(step=7, lr=1e-2, wd=0.1):
    from toy_b200 import AdamW
    a = AdamW.for_lora()
    a.lr, a.weight_decay = lr, wd
    return a.hp(step)


def held(x, floor):
    """The values that x [n] f64 is held as, by lists of blocks: powers of two and e4m3 roundings."""
    import torch
    out = torch.empty_like(x)
    for a in range(0, x.numel(), BLOCK):
        b = x[a:a + BLOCK]
        top = b.abs().max().item()
        e = -100
        while top > 448.0 * 2.0 ** e:
            e += 1
        t = b / 2.0 ** e
        step = 2.0 ** (torch.floor(torch.log2(t.abs().clamp(min=2.0 ** -6))) - 3)
        q = (t / step).round() * step
        if floor:
            q = torch.where((t > 0) & (q == 0), 2.0 ** -9, q)
        out[a:a + BLOCK] = q * 2.0 ** e
    return out


def make(shapes, ptype, gtype, seed=0, shift=0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)

    def one(s, t, f):
        n = math.prod(s)
        buf = torch.zeros(n + shift, device="cuda", dtype=t)
        buf[shift:] = torch.randn(n, device="cuda", generator=g) * f
        return buf[shift:].view(s)
    return [one(s, ptype, 0.5) for s in shapes], [one(s, gtype, 0.1) for s in shapes]


SHAPES = [(1,), (3, 5), (256,), (17, 33), (2, 512), (255,), (1000, 7), (4, 256), (0, 3), (40000,)]


def run_steps(shapes, ptype, gtype, bits, steps=3, copies=None, shift=0, factor=0.5):
    import torch
    from toy_b200.multi_adamw import MultiAdamW
    ps, _ = make(shapes, ptype, gtype, 0, shift)
    cp = [torch.zeros(p.shape, device="cuda", dtype=copies) for p in ps] if copies else None
    opt = MultiAdamW(ps, bits=bits, copies=cp)
    scale = torch.tensor(factor, device="cuda") if factor != 1 else None
    for k in range(steps):
        _, gs = make(shapes, ptype, gtype, k + 1, shift)
        if k == 1:
            gs[0] = None                      # this weight rests
        hp = torch.tensor(hp_row(k + 1), dtype=torch.float32, device="cuda")
        lr, b1, b2, eps, wd, c1, c2 = hp.double().tolist()
        before = [p.double().cpu() for p in ps]
        m0, v0 = ([x.double().cpu() for x in y] for y in opt.moments())
        opt.step(gs, hp if k else hp.tolist(), grad_scale=scale)
        m1, v1 = opt.moments()
        for i, p in enumerate(ps):
            if gs[i] is None or not p.numel():
                assert torch.equal(p.double().cpu(), before[i])
                continue
            g = gs[i].double().cpu() * factor
            m, v = m0[i] * b1 + g * (1 - b1), v0[i] * b2 + g * g * (1 - b2)
            root = v.sqrt()
            w = before[i] * (1 - lr * wd) - lr * c1 * m / (root * math.sqrt(c2) + eps)
            # m: a product, a factor and a sum, their errors within the terms; the update as much and the root's eight,
            # the quotient's and the factor's; keep and the difference
            size_m = (m0[i] * b1).abs() + (g * (1 - b1)).abs()
            upd = lr * c1 / (root * math.sqrt(c2) + eps)
            tol_m = 4 * U * size_m + 2.0 ** -149
            tol = U * (3 * before[i].abs() + upd * (4 * size_m + 16 * m.abs())) + U * w.abs()
            if ptype != torch.float32:
                tol = tol + torch.finfo(ptype).eps / 2 * (w.abs() + tol) + 2.0 ** -25
            assert ((p.double().cpu() - w).abs() <= tol).all()
            if copies:
                assert torch.equal(cp[i], p.to(copies))
            if bits == 8:
                assert torch.equal(m1[i].double().cpu().flatten(), held(m.flatten(), False))
                r = held(root.flatten(), True)
                assert torch.equal(v1[i].double().cpu().flatten(), r * r)
            else:
                assert ((m1[i].double().cpu() - m).abs() <= tol_m).all()
                assert ((v1[i].double().cpu() - v).abs() <= 8 * U * v).all()
    return opt


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("pn", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("gn", ["f32", "bf16", "f16"])
def test_types(cuda, pn, gn, bits):
    import torch
    run_steps(SHAPES, dt(pn), dt(gn), bits, copies=torch.bfloat16 if pn == "f32" else None)


@pytest.mark.parametrize("bits", [8, 32])
def test_tensors_off_their_boundaries_and_copies(cuda, bits):
    import torch
    run_steps(SHAPES, torch.float32, torch.bfloat16, bits, shift=1)
    run_steps(SHAPES, torch.bfloat16, torch.float32, bits, shift=3, copies=torch.float16, factor=1)


def test_more_tensors_than_a_launch(cuda):
    import torch
    run_steps([(5 + i % 70, 9) for i in range(1000)], torch.float32, torch.float32, 8, steps=2)
    run_steps([(3, 100)] * 449, torch.float32, torch.bfloat16, 32, steps=2)


def test_many_values(cuda):
    """20 million values: codes next to a border among them, all equal to the exact values' roundings."""
    import torch
    from toy_b200.multi_adamw import MultiAdamW
    g = torch.Generator(device="cuda").manual_seed(1)
    n = 20 * 2 ** 20
    p = torch.zeros(n, device="cuda")
    opt = MultiAdamW([p], bits=8)
    for k in range(3):
        gr = (torch.randn(n, device="cuda", generator=g) * 10.0 ** (-6 * torch.rand(n, device="cuda", generator=g)))
        hp = torch.tensor(hp_row(k + 1), dtype=torch.float32, device="cuda")
        b1, b2 = hp[1].double(), hp[2].double()
        m0, v0 = (x[0].double() for x in opt.moments())
        opt.step([gr], hp)
        m1, v1 = (x[0] for x in opt.moments())
        for x, got, floor in ((m0 * b1 + gr.double() * (1 - b1), m1, False),
                              ((v0 * b2 + gr.double() ** 2 * (1 - b2)).sqrt(), v1, True)):
            b = x.view(-1, BLOCK)
            f, e = torch.frexp(b.abs().amax(-1, keepdim=True) / 448)
            scale = torch.ldexp(torch.ones_like(f), torch.where(f == 0.5, e - 1, e).clamp(min=-100))
            t = b / scale
            step = torch.ldexp(torch.ones_like(t), torch.frexp(t.abs().clamp(min=2.0 ** -6)).exponent - 4)
            q = (t / step).round() * step
            if floor:
                q = torch.where((t > 0) & (q == 0), 2.0 ** -9, q)
            want = (q * scale).flatten()
            assert torch.equal(got.double(), want * want if floor else want)


def test_rounding_at_random(cuda):
    """Each held value is a code next to the exact one, the upper one as often as its place between them says; the same
    seed gives the same bits, another seed others; nothing else of the step changes."""
    import torch
    from toy_b200.multi_adamw import MultiAdamW
    g = torch.Generator(device="cuda").manual_seed(3)
    n = 1 << 20
    gr = torch.randn(n, device="cuda", generator=g)
    # one value of 448 in each block, so that codes are of the values themselves
    gr.view(-1, 256)[:, 0] = 1.0
    size = torch.exp2(-18 * torch.rand(n, device="cuda", generator=g))
    start = torch.rand(n, device="cuda", generator=g) * 400 * size
    start.view(-1, 256)[:, 0] = 448.0
    hp = torch.tensor([1e-3, 0.5, 0.5, 1e-8, 0.0, 1.0, 1.0], device="cuda")

    def run(seed):
        p = [torch.zeros(n, device="cuda")]
        opt = MultiAdamW(p)
        opt.set_moments([start], [start * start])
        held_m, held_v = (x[0].double() for x in opt.moments())
        opt.step([gr], hp, seed=seed)
        return p[0], opt.moments()[0][0].double(), opt.moments()[1][0].double().sqrt(), held_m, held_v
    p, m, r, m0, v0 = run(5)
    assert all(torch.equal(a, b) for a, b in zip((p, m, r), run(torch.tensor([5], device="cuda"))))
    other = run(6)
    assert torch.equal(p, other[0]) and not torch.equal(m, other[1]) and not torch.equal(r, other[2])
    exact_m = 0.5 * m0 + 0.5 * gr.double()
    exact_r = (0.5 * v0 + 0.5 * gr.double() ** 2).sqrt()
    for got, want in ((m, exact_m), (r, exact_r)):
        top = want.abs().view(-1, 256).amax(-1, keepdim=True)
        f, e = torch.frexp(top / 448)
        scale = torch.ldexp(torch.ones_like(f), torch.where(f == 0.5, e - 1, e))
        t, q = want.view(-1, 256) / scale, got.view(-1, 256) / scale
        step = torch.ldexp(torch.ones_like(t), torch.frexp(t.abs().clamp(min=2.0 ** -6)).exponent - 4)
        assert ((q - t).abs() <= step * (1 + 1e-5)).all()      # (f32: off by some 2^-22 of the value)
        ok = t.abs() > 2.0 ** -9 if got is r else torch.ones_like(t, dtype=torch.bool)   # (a root keeps the first code)
        off = ((q - t) / step)[ok]
        # places are uniform or not, the mean of the errors is 0 with a deviation of at most half a step each
        assert off.mean().abs() <= 5 * 0.5 / off.numel() ** 0.5 + 2.0 ** -16
        place = ((t / step) - torch.floor(t / step))[ok]
        up = (off > 0).double()
        for lo in (0.1, 0.4, 0.8):                              # of those a tenth above a code, four tenths, ...
            at = (place > lo) & (place < lo + 0.02)
            rate = up[at].mean()
            assert (rate - (lo + 0.01)).abs() <= 5 * 0.5 / at.sum().item() ** 0.5 + 0.01


def test_moments_follow_at_random(cuda):
    """300 steps of the same gradients, beta2 = 0.999: v comes to 1 - 0.999^300 of their squares on average. (Rounded to
    nearest it stops after a dozen steps.)"""
    import torch
    from toy_b200.multi_adamw import MultiAdamW
    n = 1 << 16
    g = [torch.ones(n, device="cuda").view(256, 256) * (1 + torch.arange(256, device="cuda") / 256.0)]
    got = {}
    for seeded in (False, True):
        opt = MultiAdamW([torch.zeros((256, 256), device="cuda")])
        for k in range(300):
            opt.step(g, [0.0, 0.9, 0.999, 1e-8, 0.0, 1.0, 1.0], seed=k if seeded else None)
        m, v = (x[0] for x in opt.moments())
        got[seeded] = (v / g[0] ** 2).mean().item() / (1 - 0.999 ** 300)
        # (to nearest m stops too: at 0.75 a step moves it by 0.1 (1 - 0.75) = 0.025, less than half its codes' 0.0625)
        assert not seeded or ((m / g[0]).mean() - 1).abs() <= 0.1
    # the square of a root that is right on average is above by its variance, a few per cent
    assert abs(got[True] - 1) <= 0.1 and got[False] < 0.2, got


def test_moments_there_and_back(cuda):
    import torch
    from toy_b200.multi_adamw import MultiAdamW
    for shift in (0, 1):
        ps, gs = make(SHAPES, torch.float32, torch.float32, 3, shift)
        a, b = (MultiAdamW([p.clone() for p in ps], bits=8) for _ in range(2))
        a.step(gs, hp_row())
        ms, vs = a.moments()
        b.set_moments(ms, vs)
        again = b.moments(out=([torch.empty_like(x) for x in ms], [torch.empty_like(x) for x in vs]))
        for x, y in zip(ms + vs, again[0] + again[1]):
            assert torch.equal(x, y)
        rnd = [torch.randn(p.shape, device="cuda") for p in ps]
        b.set_moments(rnd, [r * r for r in rnd])
        got = b.moments()
        for r, m, v in zip(rnd, *got):
            if r.numel():
                assert torch.equal(m.double().cpu().flatten(), held(r.double().cpu().flatten(), False))
                want = held((r * r).double().sqrt().cpu().flatten(), True)
                assert torch.equal(v.double().cpu().flatten(), want * want)
    c = MultiAdamW([torch.zeros(9, device="cuda")], bits=32)
    c.set_moments([torch.ones(9, device="cuda")], [torch.full((9,), 2.0, device="cuda")])
    assert c.m[0].sum() == 9 and c.moments()[1][0].sum() == 18


def test_edges(cuda):
    """Zero gradients, one value that dwarfs its block, values that are not finite."""
    import torch
    from toy_b200.multi_adamw import MultiAdamW
    p = [torch.ones(600, device="cuda")]
    opt = MultiAdamW(p, bits=8)
    opt.step([torch.zeros(600, device="cuda")], hp_row(wd=0.0))
    assert (p[0] == 1).all() and all((x[0] == 0).all() for x in opt.moments())
    g = torch.full((600,), 1e-9, device="cuda")
    g[300] = 1e6
    opt.step([g], hp_row())
    m, v = (x[0] for x in opt.moments())
    assert (v > 0).all() and p[0].isfinite().all()       # small roots beside a large one stay above 0
    opt.step([g * 1e-9], hp_row())
    assert (p[0] - 1).abs().max() < 1                    # and no step is boundless
    g = torch.ones(600, device="cuda")
    g[5], g[520] = math.nan, math.inf
    opt.step([g], hp_row())
    m = opt.moments()[0][0]
    assert m[:256].isnan().all() and m[256:512].isfinite().all() and m[512:].isnan().all()


def test_streams_and_graphs(cuda):
    import torch
    from toy_b200.multi_adamw import MultiAdamW, prepare
    prepare()
    ps, gs = make(SHAPES, torch.float32, torch.bfloat16, 5)
    hp = torch.tensor(hp_row(), dtype=torch.float32, device="cuda")
    a, b = (MultiAdamW([p.clone() for p in ps], bits=8) for _ in range(2))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step(gs, hp)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    for k in range(3):
        for g in gs:
            g.mul_(0.5)
        hp[0] *= 0.5
        graph.replay()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            b.step(gs, hp)
        torch.cuda.current_stream().wait_stream(st)
    for x, y in zip(a.params + a.m_scale, b.params + b.m_scale):
        assert torch.equal(x, y)


def test_written_weights_are_noted(cuda):
    import torch
    from toy_b200.multi_adamw import MultiAdamW
    w = torch.ones(300, device="cuda", requires_grad=True)
    opt = MultiAdamW([w])
    y = (w * w).sum()
    opt.step([torch.ones(300, device="cuda")], hp_row())
    with pytest.raises(RuntimeError):
        y.backward()


def test_refusals(cuda):
    import torch
    from toy_b200.multi_adamw import MultiAdamW
    p = [torch.zeros((4, 6), device="cuda"), torch.zeros(300, device="cuda")]
    g = [torch.zeros((4, 6), device="cuda"), torch.zeros(300, device="cuda")]
    opt = MultiAdamW(p)
    hp = hp_row()
    z8 = [torch.zeros(24, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn),
          torch.zeros(300, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn)]
    sc = [torch.zeros(1, device="cuda"), torch.zeros(2, device="cuda")]
    for bad in (lambda: MultiAdamW([]), lambda: MultiAdamW([p[0].cpu()]), lambda: MultiAdamW(p, bits=16),
                lambda: MultiAdamW([p[0], p[1].half()]), lambda: MultiAdamW([p[0].t()]),
                lambda: MultiAdamW(p, copies=[p[0].half()]), lambda: MultiAdamW(p, copies=p),
                lambda: MultiAdamW(p, copies=[p[0].half(), p[0].half()]), lambda: MultiAdamW([p[0], p[0]]),
                lambda: MultiAdamW([p[1][:200], p[1][100:]]), lambda: MultiAdamW(p, state=(z8, z8, sc, sc)),
                lambda: MultiAdamW(p, state=(z8, z8, None, None)),
                lambda: MultiAdamW(p, state=(z8, z8, sc, sc[:1])), lambda: MultiAdamW(p, state=(z8, z8, sc, sc[::-1])),
                lambda: MultiAdamW(p, bits=32, state=(z8, z8, None, None)),
                lambda: opt.step(g[:1], hp), lambda: opt.step([g[0], g[0]], hp),
                lambda: opt.step([g[0].t().contiguous(), g[1]], hp), lambda: opt.step([g[0], g[1].half()], hp),
                lambda: opt.step([g[0], g[1].double()], hp), lambda: opt.step([g[0].cpu(), g[1]], hp),
                lambda: opt.step([g[0], g[1].repeat(2)[::2]], hp), lambda: opt.step(g, hp[:6]),
                lambda: opt.step(g, hp, grad_scale=torch.ones(2, device="cuda")),
                lambda: opt.step(g, torch.zeros(7, device="cuda").double()), lambda: opt.moments(out=(g, g[:1])),
                lambda: opt.set_moments(g, [g[0], g[0]])):
        with pytest.raises(ValueError):
            bad()
    MultiAdamW(p, state=(z8, [t.clone() for t in z8], sc, [t.clone() for t in sc])).step([None, None], hp)
