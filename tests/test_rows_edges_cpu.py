"""What the row operators refuse on the host, before a GPU is touched: rows that
32-bit counts of a kernel would pass, and results that lie over what they are
made from."""
import ctypes as C

P = 1 << 20          # an address that is never followed: every call below is refused


def lib():
    from toy_b200 import _lib
    return _lib.lib()


def test_rows_of_almost_two_to_the_31_values():
    """The kernels count a row's pieces in 32 bits, up to a step past its end."""
    from toy_b200._lib import ExpertRowsArgs
    ok = dict(n_tokens=1, n_used=1, n_rows=1, row_type=30, pos=P, weights=P)
    for d in (2 ** 31 - 1, 2 ** 31 - 256):
        a = ExpertRowsArgs(**ok, d=d, x=P, ldx=d, xs=P + (1 << 40), ldxs=d)
        for f in ("tb2_expert_dispatch", "tb2_expert_combine", "tb2_expert_combine_grad"):
            assert getattr(lib(), f)(C.byref(a), None) == -1, (d, f)


def test_no_tokens_write_nothing():
    """A call without tokens ends before it looks at the rows: those that would be cleared stay."""
    from toy_b200._lib import ExpertRowsArgs
    a = ExpertRowsArgs(n_tokens=0, n_used=2, d=16, n_rows=8, row_type=0, xs=P, ldxs=16, d_xs=P, ldd=16, n_sorted=P)
    for f in ("tb2_expert_dispatch", "tb2_expert_combine", "tb2_expert_combine_grad"):
        assert getattr(lib(), f)(C.byref(a), None) == 0        # (no GPU here: nothing was launched)


def test_results_over_their_operands():
    """A result that shares memory with an operand is refused where it is not that operand in place; rows that lie
    between each other's are not."""
    from toy_b200._lib import ExpertRowsArgs, LogprobsGradArgs
    d, e = 16, 4

    def rows(**kw):
        return C.byref(ExpertRowsArgs(**{**dict(n_tokens=4, n_used=2, d=d, n_rows=8, row_type=0, x=P, ldx=64,
                                                xs=P + (1 << 20), ldxs=64, pos=P), **kw}))
    far, row = P + (2 << 20), 64 * e
    for xs in (P, P + e, P + row, P + 3 * row, P - 7 * row, P + (d - 1) * e, P - (d - 1) * e, P + row - e):
        for f in ("tb2_expert_dispatch", "tb2_expert_combine"):
            assert getattr(lib(), f)(rows(xs=xs), None) == -1, (xs - P, f)
    for res in (P + e, P + row, P - row, P + (d - 1) * e):
        assert lib().tb2_expert_combine(rows(residual=res, ldr=64), None) == -1, res - P
    for dz in (P, P + e, P + 2 * row, P + (1 << 20) + e, P + (1 << 20) - row):
        assert lib().tb2_expert_combine_grad(rows(d_xs=dz, ldd=64), None) == -1, dz - P
    grad = dict(n_rows=4, vocab=d, row_type=0, logits=P, ld=64, scale=1.0, tokens=far, stats=far, g_logprob=far, ldd=64)
    for dl in (P + e, P + row, P - row, P + (d - 1) * e, P - (d - 1) * e):
        assert lib().tb2_logprobs_grad(C.byref(LogprobsGradArgs(**grad, d_logits=dl)), None) == -1, dl - P


def test_a_sort_over_its_ids():
    """Places are scattered while ids are still read: buffers that share memory are refused."""
    from toy_b200._lib import ExpertSortArgs
    n = 1000
    ok = dict(ids=P, id_bytes=8, n_slots=n, n_experts=4, offsets=P + 8 * n, order=P + 8 * n + 20,
              pos=P + 12 * n + 20)
    for k, v in (("order", P), ("pos", P + 8 * n - 4), ("offsets", P + 8 * n - 4), ("pos", P + 12 * n + 16),
                 ("order", P + 8 * n + 16), ("pos", P + 8 * n + 20), ("ids", P + 16 * n + 16)):
        assert lib().tb2_expert_sort(C.byref(ExpertSortArgs(**{**ok, k: v})), None) == -1, (k, v - P)
    assert lib().tb2_expert_sort(C.byref(ExpertSortArgs(**ok)), None) != -1       # (no GPU: it gets as far as that)
