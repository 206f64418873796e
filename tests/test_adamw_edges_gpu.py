"""Where AdamW over many tensors goes wrong easily: weights whose storage moves,
writes that autograd has to know of, block scales at a power of two's border,
second moments below f32's normal numbers, lists that are too short."""
import math

import pytest

pytestmark = pytest.mark.gpu
HP = [1e-2, 0.9, 0.999, 1e-8, 0.0, 10.0, 1000.0]


def ones(*shape, dtype=None):
    import torch
    return torch.ones(shape, device="cuda", dtype=dtype or torch.float32)


@pytest.mark.parametrize("bits", [8, 32])
def test_weights_whose_storage_moves(cuda, bits):
    """A parameter keeps its identity when `p.data = ...` gives it other memory: the step is made there, and what the
    old memory holds stays; a parameter that no longer fits is refused before anything runs."""
    import torch
    from toy_b200.multi_adamw import MultiAdamW
    a, b = torch.nn.Parameter(ones(300)), torch.nn.Parameter(ones(4, 6))
    ca, cb = ones(300, dtype=torch.bfloat16), ones(4, 6, dtype=torch.bfloat16)
    opt = MultiAdamW([a, b], bits=bits, copies=[ca, cb])
    want = MultiAdamW([ones(300), ones(4, 6)], bits=bits)
    gs = [ones(300), ones(4, 6)]
    for o in (opt, want):
        o.step(gs, HP, seed=1)
    old, old_copy = a.data, ca.data         # (kept alive: nothing here is written out of range, mended or not)
    a.data, ca.data = old.clone(), old_copy.clone()
    before, before_copy = old.clone(), old_copy.clone()
    for k in range(2):
        for o in (opt, want):
            o.step(gs, HP, seed=2 + k)
    assert torch.equal(old, before) and torch.equal(old_copy, before_copy)
    for p, q, c in zip(opt.params, want.params, opt.copies):
        assert torch.equal(p.detach(), q) and torch.equal(c, q.bfloat16())
    kept = a.data
    for other in (kept.double(), kept.half(), kept.cpu(), ones(600)[::2], ones(299), b.data.view(-1)):
        a.data = other
        was = b.detach().clone()
        with pytest.raises(ValueError):
            opt.step(gs, HP, seed=9)
        assert torch.equal(b.detach(), was)
    a.data = kept
    opt.step(gs, HP, seed=4)
    want.step(gs, HP, seed=4)
    assert torch.equal(a.detach(), want.params[0]) and torch.equal(b.detach(), want.params[1])


@pytest.mark.parametrize("what", ["detached", "frozen", "copy", "later", "moments", "state"])
def test_every_written_tensor_is_noted(cuda, what):
    """What autograd saved of a tensor that a step (or moments(out=)) has written since is refused, not used: weights
    given detached, weights saved for another tensor's gradient, 16-bit copies, weights that require a gradient only
    later, f32 moments."""
    import torch
    from toy_b200.multi_adamw import MultiAdamW
    w = ones(16, 16)
    c = ones(16, 16, dtype=torch.bfloat16)
    x = torch.randn((4, 16), device="cuda", requires_grad=True)
    leaf = w.requires_grad_() if what == "detached" else w
    opt = MultiAdamW([leaf.detach() if what == "detached" else w], copies=[c], bits=32 if what == "state" else 8)
    out = ([ones(16, 16)], [ones(16, 16)])
    if what == "later":
        w.requires_grad_()
    y = {"detached": lambda: (leaf * leaf).sum(), "frozen": lambda: (x @ w).sum(),
         "copy": lambda: (x.bfloat16() @ c).sum(), "later": lambda: (w * w).sum(),
         "moments": lambda: (x @ out[0][0]).sum(), "state": lambda: (x @ opt.moments()[1][0]).sum()}[what]()
    if what == "moments":
        opt.moments(out=out)
    else:
        opt.step([ones(16, 16)], HP, seed=0)
    with pytest.raises(RuntimeError):
        y.backward()


def test_resting_weights_are_not_noted(cuda):
    """A weight whose gradient is None is not written, and a backward through it stands."""
    import torch
    from toy_b200.multi_adamw import MultiAdamW
    w, v = (ones(300).requires_grad_() for _ in range(2))
    opt = MultiAdamW([w, v])
    y = (w * w).sum()
    opt.step([None, ones(300)], HP, seed=0)
    y.backward()
    assert (w.grad == 2).all()


def check_roots(opt, root):
    """The first weight's held roots and their scales are those of the exact ones, root [blocks, 256] f64."""
    import torch
    top = root.amax(-1, keepdim=True)
    e = torch.floor(torch.log2(top / 448)) - 1
    for _ in range(3):
        e = torch.where(top > 448 * torch.exp2(e), e + 1, e)
    scale = torch.exp2(e.clamp(min=-100))
    assert torch.equal(opt.v_scale[0].double(), scale[:, 0])
    t = root / scale
    step = torch.ldexp(torch.ones_like(t), torch.frexp(t.clamp(min=2.0 ** -6)).exponent - 4)
    q = (t / step).round() * step
    q = torch.where((t > 0) & (q == 0), 2.0 ** -9, q) * scale
    assert torch.equal(opt.moments()[1][0].double(), q * q)


def test_block_scales_at_the_border(cuda):
    """A block's largest root at 448 times a power of two and a few f32 steps to either side of it: the scale is the
    smallest power of two that brings the block within 448, and the small roots beside it are the exact ones'
    roundings. From an empty state with beta2 = 0.75, so that the root is half the gradient, exactly; and on from held
    roots, with gradients that bring the largest within some 2^-23 of the border."""
    import torch
    from toy_b200.multi_adamw import MultiAdamW
    gen = torch.Generator(device="cuda").manual_seed(0)
    rows = [(e, k) for e in range(-16, 30) for k in range(-8, 9)]
    g = torch.rand((len(rows), 256), device="cuda", generator=gen) * \
        torch.exp2(-17 * torch.rand((len(rows), 256), device="cuda", generator=gen))
    for i, (e, k) in enumerate(rows):
        g[i] *= 2.0 ** e
        g[i, 7 + i % 200] = 896.0 * 2.0 ** e * (1 + k * 2.0 ** -23 if k >= 0 else 1 + k * 2.0 ** -24)
    opt = MultiAdamW([torch.zeros_like(g)])
    opt.step([g], [0.0, 0.5, 0.75, 1e-8, 0.0, 1.0, 1.0])
    check_roots(opt, g.double() / 2)
    n = 1 << 14
    for b2 in (0.75, 0.9, 0.999):
        opt = MultiAdamW([torch.zeros((n, 256), device="cuda")])
        start = torch.rand((n, 256), device="cuda", generator=gen)
        start[:, 9] = 300 + 100 * torch.rand(n, device="cuda", generator=gen)
        opt.set_moments([start], [start * start])
        v0 = opt.moments()[1][0].double()
        hp = torch.tensor([0.0, 0.5, b2, 1e-8, 0.0, 1.0, 1.0], device="cuda")
        b2 = hp[2].double()
        g = torch.zeros((n, 256), device="cuda")
        near = 1 + (torch.rand(n, device="cuda", generator=gen).double() - 0.5) * 2.0 ** -21
        g[:, 9] = (((448.0 * near) ** 2 - b2 * v0[:, 9]) / (1 - b2)).sqrt().float()
        opt.step([g], hp)
        check_roots(opt, (b2 * v0 + (1 - b2) * g.double() ** 2).sqrt())


def test_second_moments_below_the_normal_numbers(cuda):
    """f32 moments: roots of second moments below 2^-126 count, as in the framework's other AdamW."""
    import torch
    from toy_b200.multi_adamw import MultiAdamW
    g = torch.logspace(-22, -17, 1000, device="cuda")
    p = [torch.zeros(1000, device="cuda")]
    opt = MultiAdamW(p, bits=32)
    opt.step([g], [1.0, 0.9, 0.5, 1e-30, 0.0, 1.0, 1.0])
    m, v = (x[0].double() for x in opt.moments())
    assert (v < 2.0 ** -126).any() and (v[v > 0] > 0).any()
    want = -m / (v.sqrt() + 1e-30)
    on = v > 0
    # the root and the sum within half a step each, the quotient and the difference too; eps itself rounded
    assert ((p[0].double() - want)[on].abs() <= 8 * 2.0 ** -24 * want[on].abs()).all()


@pytest.mark.parametrize("bits", [8, 32])
def test_moments_lists_that_do_not_fit(cuda, bits):
    import torch
    from toy_b200.multi_adamw import MultiAdamW
    opt = MultiAdamW([ones(9), ones(2, 3)], bits=bits)

    def both():
        return [ones(9), ones(2, 3)]
    for ms, vs in ((both()[:1], both()), (both(), both()[:1]), (both() + [ones(1)], both()),
                   ([ones(9), ones(3)], both()), (both(), [ones(9), ones(2, 4)]), (both(), [ones(1), ones(2, 3)])):
        with pytest.raises(ValueError):
            opt.set_moments(ms, vs)
        with pytest.raises(ValueError):
            opt.moments(out=(ms, vs))
    assert all((x == 0).all() for y in opt.moments() for x in y)       # nothing was set
    opt.set_moments(both(), both())
    got = opt.moments(out=(both(), both()))
    assert all((x == 1).all() for y in got for x in y)


def test_a_captured_step_takes_its_seed_as_a_tensor(cuda):
    """A number would be the same in each replay, and so the random bits."""
    import torch
    from toy_b200.multi_adamw import MultiAdamW, prepare
    prepare()
    opt, g, hp = MultiAdamW([ones(300)]), [ones(300)], torch.tensor(HP, device="cuda")
    seed = torch.zeros(1, device="cuda", dtype=torch.int64)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        torch.zeros(1, device="cuda")
        with pytest.raises(ValueError):
            opt.step(g, hp, seed=3)
        with pytest.raises(ValueError):
            opt.step(g, HP, seed=seed)
        opt.step(g, hp, seed=seed)
    want = MultiAdamW([ones(300)])
    for k in range(3):
        seed.fill_(k)
        graph.replay()
        want.step(g, HP, seed=k)
        assert all(torch.equal(a, b) for a, b in zip(opt.m_scale + opt.params, want.m_scale + want.params))
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(opt.m + opt.v,
                                                                                         want.m + want.v))


def test_steps_to_nearest_are_warned_of(cuda):
    """8-bit moments do not follow small steps without a seed: said once for each optimizer, and nowhere else."""
    import warnings
    from toy_b200.multi_adamw import MultiAdamW

    def heard(*steps, **kw):
        opt = MultiAdamW([ones(300)], **kw)
        with warnings.catch_warnings(record=True) as w:
            warnings.simplefilter("always")
            for seed in steps:
                opt.step([ones(300)], HP, seed=seed)
        return len(w)
    assert heard(None, None, None) == 1 and heard(1, 2) == 0 and heard(None, None, bits=32) == 0
