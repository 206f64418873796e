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
