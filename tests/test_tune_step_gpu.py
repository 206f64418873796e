"""The operators as a fine-tune step uses them together: tokens to experts and
back, log probabilities with an entropy bonus and a distillation term, the
gradient through all of it, and an AdamW step with 8-bit moments. The gradients
against the same step in 64 bits by autograd on the host; the step as a user's
loop makes it, for running."""
import pytest

pytestmark = pytest.mark.gpu

T, D, E, K, V, FF = 96, 64, 6, 2, 1003, 48


def weights(seed, device, dtype):
    import torch
    g = torch.Generator().manual_seed(seed)
    w = {"emb": (V, D), "router": (E, D), "up": (E, D, FF), "down": (E, FF, D), "head": (V, D)}
    return {k: (torch.randn(s, generator=g, dtype=torch.float64) / (D ** 0.5)).to(device=device, dtype=dtype)
            for k, s in w.items()}


def routed(x, w, ids):
    """Softmax weights of the chosen experts, renormalised."""
    import torch
    p = torch.softmax(x @ w["router"].T, -1).gather(1, ids.long())
    return p / p.sum(-1, keepdim=True)


def loss_on_gpu(w, tokens, targets, adv, teacher):
    import torch
    from toy_b200 import experts, logprobs
    x = w["emb"][tokens]
    ids = (x @ w["router"].T).detach().topk(K, -1).indices
    r = experts.sort(ids, E)
    xs = experts.dispatch(x, r)
    at = r.offsets.tolist()
    z = torch.cat([torch.tanh(xs[at[e]:at[e + 1]] @ w["up"][e]) @ w["down"][e] for e in range(E)])
    y = experts.combine(z, r, routed(x, w, ids), residual=x)
    s = logprobs.token_logprobs(y @ w["head"].T, targets, scale=0.8, entropy=True, top=4)
    loss = -(adv * s.logprob).sum() - 0.05 * s.entropy.mean() - (teacher * s.top_logprobs).sum() * 0.1
    return loss, ids, s.top_ids


def loss_on_host(w, tokens, targets, adv, teacher, ids, top_ids):
    import torch
    x = w["emb"][tokens]
    wt = routed(x, w, ids)
    y = x
    for k in range(K):
        e = ids[:, k].long()
        h = torch.tanh(torch.einsum("td,tdf->tf", x, w["up"][e]))
        y = y + wt[:, k, None] * torch.einsum("tf,tfd->td", h, w["down"][e])
    lp = torch.log_softmax(0.8 * (y @ w["head"].T), -1)
    got = torch.where(targets >= 0, lp.gather(1, targets.clamp(min=0)[:, None])[:, 0], 0.0)
    return -(adv * got).sum() + 0.05 * (lp.exp() * lp).sum(-1).mean() - (teacher * lp.gather(1, top_ids)).sum() * 0.1


def test_gradients_and_steps(cuda):
    import torch
    from toy_b200 import AdamW
    from toy_b200.multi_adamw import MultiAdamW
    g = torch.Generator().manual_seed(1)
    tokens, targets = torch.randint(0, V, (T,), generator=g), torch.randint(0, V, (T,), generator=g)
    targets[::7] = -1
    adv, teacher = torch.randn(T, generator=g), torch.rand((T, 4), generator=g)
    w = {k: v.requires_grad_() for k, v in weights(0, "cuda", torch.float32).items()}
    dev = [t.cuda() for t in (tokens, targets, adv, teacher)]
    loss, ids, top_ids = loss_on_gpu(w, *dev)
    loss.backward()
    h = {k: v.requires_grad_() for k, v in weights(0, "cpu", torch.float64).items()}
    want = loss_on_host(h, tokens, targets, adv.double(), teacher.double(), ids.cpu(), top_ids.cpu())
    want.backward()
    # f32 products of 64 to 1003 terms between them: errors of some 2^-24 times the square root of the terms' number,
    # against gradients whose own terms cancel to a tenth
    assert abs(loss.item() - want.item()) <= 1e-5 * abs(want.item()) + 1e-4
    for k in w:
        a, b = w[k].grad.double().cpu(), h[k].grad
        assert (a - b).norm() <= 2e-5 * b.norm(), (k, (a - b).norm() / b.norm())
    names = list(w)
    copies = [w[k].detach().bfloat16() for k in names]
    opt = MultiAdamW([w[k].detach() for k in names], bits=8, copies=copies)
    hp = AdamW.for_lora()
    hp.lr = 1e-3
    before = {k: w[k].detach().clone() for k in names}
    for step in range(3):
        if step:
            for k in names:
                w[k].grad = None
            loss_on_gpu(w, *dev)[0].backward()
        norm = torch.stack([w[k].grad.norm() for k in names]).norm()
        opt.step([w[k].grad for k in names], hp.hp(step + 1), grad_scale=(1.0 / norm.clamp(min=1.0)).view(1),
                 seed=step)
    for k, c in zip(names, copies):
        d = (w[k].detach() - before[k]).abs()
        assert d.max() > 0 and d.max() <= 3.5e-3          # three steps of at most the rate each, but for roundings
        assert torch.equal(c, w[k].detach().bfloat16())
    m, v = opt.moments()
    assert all(x.isfinite().all() for x in m + v)


def test_captured_without_autograd(cuda):
    """The same chain of calls in a CUDA graph, gradients by their own calls; a leaf's autograd there is refused."""
    import torch
    from toy_b200 import experts, logprobs
    from toy_b200.multi_adamw import MultiAdamW
    logprobs.prepare()
    x = torch.randn((T, D), device="cuda")
    ids = torch.randint(0, E, (T, K), device="cuda", dtype=torch.int32)
    wt = torch.rand((T, K), device="cuda")
    head = torch.randn((V, D), device="cuda")
    t = torch.randint(0, V, (T,), device="cuda")
    ones = torch.ones(T, device="cuda")
    hp = torch.tensor([1e-3, 0.9, 0.999, 1e-8, 0.0, 1.0, 1.0], device="cuda")

    def chain(head, opt):
        r = experts.sort(ids, E)
        z = experts.dispatch(x, r)
        y = experts.combine(z, r, wt, residual=x)
        logits = y @ head.T
        s = logprobs.token_logprobs(logits, t, entropy=True)
        d = logprobs.token_logprobs_grad(logits, t, s, ones, grad_entropy=ones, out=logits)
        dz, dw = experts.combine_grad(d @ head, z, r, wt)
        opt.step([d.T @ y], hp)
        return experts.dispatch_grad(dz, r), dw

    h1, h2 = head.clone(), head.clone()
    o1, o2 = MultiAdamW([h1]), MultiAdamW([h2])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        chain(head.clone(), MultiAdamW([head.clone()]))        # (the library behind @ sets itself up)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = chain(h1, o1)
    for _ in range(2):
        graph.replay()
        want = chain(h2, o2)
        assert torch.equal(h1, h2) and all(torch.equal(a, b) for a, b in zip(got, want))
    leaf = torch.randn((4, 50), device="cuda", requires_grad=True)
    eager = logprobs.token_logprobs(leaf, t[:4] % 50)          # an eager graph of the leaf lives
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        torch.zeros(1, device="cuda")
        with pytest.raises(RuntimeError):
            logprobs.token_logprobs(leaf, t[:4])
        with pytest.raises(RuntimeError):
            experts.combine(leaf, experts.Routing(ids, ids, ids))
    assert eager.logprob.requires_grad
