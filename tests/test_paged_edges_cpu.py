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
