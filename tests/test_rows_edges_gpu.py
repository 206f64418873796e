"""Where the row operators go wrong easily: buffers of a routing that are filled
again, derivatives that they do not have, sorted rows that are none, more slots
than 32 bits count comfortably."""
import pytest

pytestmark = pytest.mark.gpu


def test_slots_next_to_two_to_the_31(cuda):
    """The largest call: 2^31 - 1 slots, whose places come out as counted."""
    import torch
    from toy_b200 import experts as X
    n = 2 ** 31 - 1
    if torch.cuda.mem_get_info()[1] < 100 * 2 ** 30:
        pytest.skip("needs a GPU of 100 GB")
    ids = torch.zeros((n, 1), device="cuda", dtype=torch.int32)
    ids[1::2] = 1                                   # slots of two experts in turn
    ids[n - 1000000:n - 999990] = -1                # ten of none, near the end
    r = X.sort(ids, 2)
    del ids
    ones = n // 2 - 5
    zeros = n - n // 2 - 5
    assert r.offsets.tolist() == [0, zeros, zeros + ones]
    step = 1 << 27
    for a in range(0, n, step):
        slot = torch.arange(a, min(n, a + step), device="cuda")
        # of the ten slots that go nowhere five are of either expert: those of this slot's parity that lie before it
        lo = n - 1000000
        rank = slot // 2 - ((slot - lo - (slot - lo) % 2) // 2).clamp(0, 5)
        want = torch.where(slot % 2 == 1, zeros + rank, rank)
        want = torch.where((slot >= n - 1000000) & (slot < n - 999990), -1, want)
        assert torch.equal(r.pos[a:a + step, 0].long(), want)
        on = want >= 0
        assert torch.equal(r.order[want[on]].long(), slot[on])
    assert (r.order[zeros + ones:] == -1).all()
    del r, slot, rank, want, on
    torch.cuda.empty_cache()


def randn(*shape, **kw):
    import torch
    return torch.randn(shape, device="cuda", **kw)


def test_a_routing_filled_again_is_noted(cuda):
    """sort(out=) into buffers that a backward still needs: that backward is refused, not made with the new places."""
    import torch
    from toy_b200 import experts as X
    ids = torch.randint(0, 4, (10, 2), device="cuda", dtype=torch.int32)
    for op in ("dispatch", "combine"):
        r = X.sort(ids, 4)
        if op == "dispatch":
            y = X.dispatch(randn(10, 16, requires_grad=True), r)
        else:
            y = X.combine(randn(20, 16, requires_grad=True), r, torch.rand((10, 2), device="cuda"))
        again = X.sort((ids + 1) % 4, 4, out=r)
        assert again is r
        with pytest.raises(RuntimeError):
            y.sum().backward()


def test_forward_mode_is_refused(cuda):
    """A tensor with a tangent gives a result that has one, or an error; never a result without."""
    import torch
    import torch.autograd.forward_ad as fwd
    from toy_b200 import experts as X, logprobs as L
    ids = torch.randint(0, 4, (10, 2), device="cuda", dtype=torch.int32)
    r = X.sort(ids, 4)
    x, z, w = randn(10, 16), randn(20, 16), torch.rand((10, 2), device="cuda")
    t, g = torch.zeros(10, dtype=torch.int64, device="cuda"), torch.ones(10, device="cuda")
    s = L.token_logprobs(x, t)
    with fwd.dual_level():
        def dual(v):
            return fwd.make_dual(v, torch.ones_like(v))
        for call in (lambda: L.token_logprobs(dual(x), t), lambda: L.token_logprobs_grad(dual(x), t, s, g),
                     lambda: L.token_logprobs_grad(x, t, s, dual(g)), lambda: X.dispatch(dual(x), r),
                     lambda: X.dispatch(dual(x), r, out=z.clone()), lambda: X.combine(dual(z), r, w),
                     lambda: X.combine(z, r, dual(w)), lambda: X.combine(z, r, w, residual=dual(x)),
                     lambda: X.dispatch_grad(dual(z), r), lambda: X.combine_grad(dual(x), z, r, w),
                     lambda: X.combine_grad(x, z, r, dual(w)), lambda: X.dispatch(x, r, out=dual(z))):
            with pytest.raises(ValueError):
                call()
        # without tangents all of it works at such a level too
        L.token_logprobs_grad(x, t, L.token_logprobs(x, t), g)
        y = X.combine(X.dispatch(x.clone().requires_grad_(), r), r, w)
    y.sum().backward()


@pytest.mark.parametrize("K", [1, 2, 3, 9])
def test_no_sorted_rows(cuda, K):
    """Tokens of which none goes to an expert, with sorted rows cut to those there are: none."""
    import torch
    from toy_b200 import experts as X
    from toy_b200._lib import lib
    ids = torch.full((6, K), -1, device="cuda", dtype=torch.int32)
    r = X.sort(ids, 4)
    for d in (32, 33):
        x, z, w = randn(6, d), randn(6 * K, d)[:0], torch.rand((6, K), device="cuda")
        assert torch.equal(X.combine(z, r, w, residual=x), x)
        assert (X.combine(z, r) == 0).all() and (X.dispatch_grad(z, r) == 0).all()
        dz, dw = X.combine_grad(x, z, r, w)
        assert dz.shape == (0, d) and (dw == 0).all()
        assert X.dispatch(x, r, out=z) is z
        a, b, c = x.clone().requires_grad_(), z.clone().requires_grad_(), w.clone().requires_grad_()
        X.combine(b, r, c, residual=a).sum().backward()
        assert (a.grad == 1).all() and b.grad.shape == (0, d) and (c.grad == 0).all()
    assert lib().tb2_device_error() == 0


def test_results_over_their_operands(cuda):
    """Refused with ValueError where a result would lie over what it is made from; rows between each other's are not."""
    import torch
    from toy_b200 import experts as X, logprobs as L
    ids = torch.randperm(40, device="cuda").remainder(4).int()[:, None]
    r = X.sort(ids, 4)
    order = r.order.long()
    buf = randn(40, 64)
    a, b = buf[:, :32], buf[:, 32:]
    x = a.clone()
    t, g = torch.zeros(39, dtype=torch.int64, device="cuda"), torch.ones(39, device="cuda")
    s = L.token_logprobs(a[1:], t)
    for bad in (lambda: X.dispatch(a, r, out=a), lambda: X.dispatch(a, r, out=buf[:, 31:63]),
                lambda: X.combine(a, r, out=a), lambda: X.dispatch_grad(a, r, out=buf[:, 16:48]),
                lambda: X.combine(b.clone(), r, residual=a, out=buf[:, 1:33]),
                lambda: X.combine_grad(a, b, r, out=a), lambda: X.combine_grad(x, b, r, out=buf[:, 31:63]),
                lambda: L.token_logprobs_grad(a[1:], t, s, g, out=a[:39])):
        was = buf.clone()
        with pytest.raises(ValueError):
            bad()
        assert torch.equal(buf, was)
    X.dispatch(a, r, out=b)
    assert torch.equal(b, x[order]) and torch.equal(a, x)
    X.combine(a, r, out=b)
    assert torch.equal(b[order], x) and torch.equal(a, x)
    want = L.token_logprobs_grad(a[1:].clone(), t, s, g)
    assert torch.equal(L.token_logprobs_grad(a[1:], t, s, g, out=b[1:]), want)


def test_outputs_that_do_not_fit_are_not_noted(cuda):
    """A refused call has written nothing, and what autograd saved of its `out` stands."""
    import torch
    from toy_b200 import experts as X, logprobs as L
    ids = torch.randint(0, 4, (10, 2), device="cuda", dtype=torch.int32)
    r = X.sort(ids, 4)
    x, z = randn(10, 16), randn(20, 16)
    t, g = torch.zeros(10, dtype=torch.int64, device="cuda"), torch.ones(10, device="cuda")
    s = L.token_logprobs(x, t)
    for call in (lambda o: X.dispatch(x, r, out=o), lambda o: X.dispatch_grad(z, r, out=o),
                 lambda o: X.combine(z, r, out=o), lambda o: X.combine_grad(x, z, r, out=o),
                 lambda o: L.token_logprobs_grad(x, t, s, g, out=o)):
        out = randn(3, 3)
        a = torch.ones((3, 3), device="cuda", requires_grad=True)
        y = (a * out).sum()
        with pytest.raises(ValueError):
            call(out)
        y.backward()


@pytest.mark.parametrize("T,K", [(40, 1), (40, 2), (3000, 2)])
def test_small_products_behind_a_large_one(cuda, T, K):
    """combine's gradient of the weights: in each lane's 64 products one of 1 comes first, and the others, 2^-25, are
    too small to be added to it one by one."""
    import torch
    from toy_b200 import experts as X
    d = 2048
    ids = torch.randint(0, 4, (T, K), device="cuda", dtype=torch.int32)
    r = X.sort(ids, 4)
    dy = torch.full((T, d), 2.0 ** -25, device="cuda")
    dy[:, :128:4] = 1.0
    z = torch.ones((T * K, d), device="cuda")
    dw = X.combine_grad(dy, z, r)[1].double()
    want = dy[0].double().sum()
    # at most 16 products in a row, the d / 512 sums of those, and five halvings (and one rounding to spare)
    assert ((dw - want).abs() <= (16 + d / 512 + 6) * 2.0 ** -24 * want).all()


def test_a_refused_sort_notes_nothing(cuda):
    import torch
    from toy_b200 import experts as X
    ids = torch.randint(0, 4, (10, 2), device="cuda", dtype=torch.int32)
    r = X.sort(ids, 4)
    was, versions = [t.clone() for t in r], [t._version for t in r]
    for out in (r._replace(order=ids.view(-1)), r._replace(pos=r.order.view(10, 2)), r._replace(pos=r.pos.long())):
        with pytest.raises(ValueError):
            X.sort(ids, 4, out=out)
    assert [t._version for t in r] == versions and all(torch.equal(a, b) for a, b in zip(r, was))
    X.sort(ids, 4, out=r)
    assert all(t._version == v + 1 for t, v in zip(r, versions))
