"""More refusals of the paged KV-cache operators, before anything touches a GPU."""
import ctypes as C
import os
import sys

import pytest

pytest.importorskip("torch")
sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from test_paged_cpu import P, append_args, attend_args, kv, plan_args, release_args  # noqa: E402


@pytest.mark.parametrize("scale", [3e38, -3e38, 2.4e38])
def test_scales_past_f32(scale):
    """A finite scale whose base-2 form is not: every score, 0 too, would be infinite or NaN."""
    from toy_b200._lib import lib
    assert lib().tb2_paged_attend(C.byref(kv()), C.byref(attend_args(scale=scale)), None) == -1


# (addresses far from the others', so that an array and its result elsewhere do not overlap in part)
@pytest.mark.parametrize("what,by", [(w, b) for w in (
    "lens", "add", "table", "free_pages", "state", "lens_out", "state_out", "cu_tokens", "positions", "requests")
    for b in (1, 2)] + [("slots", 2), ("slots", 4)])
def test_plan_arrays_off_their_boundary(what, by):
    from toy_b200._lib import lib
    assert lib().tb2_paged_plan(C.byref(plan_args(**{what: P + (1 << 16) + by})), None) == -1


@pytest.mark.parametrize("by", [1, 2])
@pytest.mark.parametrize("what", ["lens", "done", "table", "free_pages", "state", "lens_out", "state_out"])
def test_release_arrays_off_their_boundary(what, by):
    from toy_b200._lib import lib
    assert lib().tb2_paged_release(C.byref(release_args(**{what: P + (1 << 16) + by})), None) == -1


@pytest.mark.parametrize("bad", [dict(positions=P + 1), dict(positions=P + 2), dict(slots=P + 4), dict(slots=P + 1)],
                         ids=str)
def test_append_arrays_off_their_boundary(bad):
    from toy_b200._lib import lib
    assert lib().tb2_paged_append(C.byref(kv()), C.byref(append_args(**bad)), None) == -1


@pytest.mark.parametrize("bad", [dict(table=P + 1), dict(table=P + 2), dict(lens=P + 2), dict(lse=P + 2),
                                 dict(lse=P + 1)], ids=str)
def test_attend_arrays_off_their_boundary(bad):
    from toy_b200._lib import lib
    assert lib().tb2_paged_attend(C.byref(kv()), C.byref(attend_args(**bad)), None) == -1
