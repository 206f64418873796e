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
