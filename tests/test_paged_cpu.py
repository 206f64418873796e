"""Refusals of the paged KV-cache operators: every bad argument is an error
code (or ValueError from the Python layer) before anything touches a GPU.
Pointers here are never followed: each call is refused on the host."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

P = 1 << 20   # a 16-byte aligned address that no call may reach


def kv(**kw):
    from toy_b200._lib import PagedKV
    d = dict(k=P, v=P, k_scale=None, v_scale=None, kv_type=0, n_pages=4, page_size=16, n_kv=2, d_head=64,
             page_stride=2 * 16 * 64, head_stride=16 * 64, tok_stride=64)
    d.update(kw)
    return PagedKV(**d)


def append_args(**kw):
    from toy_b200._lib import PagedAppendArgs
    d = dict(n_tokens=3, n_heads=4, row_type=0, q=P, ldq=256, k=P, ldk=128, v=P, ldv=128, q_out=P, ldqo=256,
             bias=None, rope=P, rope_rows=8, positions=P, slots=P)
    d.update(kw)
    return PagedAppendArgs(**d)


def attend_args(**kw):
    from toy_b200._lib import PagedAttendArgs, lib
    d = dict(n_req=2, n_heads=4, row_type=0, q=P, ldq=256, out=P, ldo=256, table=P, table_width=3, table_stride=3,
             lens=P, scale=0.125, lse=None, workspace=P, workspace_bytes=lib().tb2_paged_attend_workspace())
    d.update(kw)
    return PagedAttendArgs(**d)


def plan_args(**kw):
    from toy_b200._lib import PagedPlanArgs
    d = dict(lens=P, add=P, n_req=2, table=P, table_width=3, table_stride=3, free_pages=P, n_free=4, state=P,
             page_size=16, n_pages=4, n_tokens=5, lens_out=P, state_out=P, cu_tokens=P, slots=P, positions=P,
             requests=P)
    d.update(kw)
    return PagedPlanArgs(**d)


def release_args(**kw):
    from toy_b200._lib import PagedReleaseArgs
    d = dict(lens=P, done=P, n_req=2, table=P, table_width=3, table_stride=3, free_pages=P, n_free=4, state=P,
             page_size=16, n_pages=4, lens_out=P, state_out=P)
    d.update(kw)
    return PagedReleaseArgs(**d)


BAD_KV = [dict(k=None), dict(v=None), dict(kv_type=2), dict(kv_type=8), dict(n_pages=0), dict(page_size=0),
          dict(page_size=(1 << 20) + 1), dict(n_kv=0), dict(d_head=0), dict(d_head=48), dict(d_head=160),
          dict(k=P + 4), dict(v=P + 8), dict(tok_stride=32), dict(tok_stride=66), dict(head_stride=63),
          dict(page_stride=-2048), dict(kv_type=8, k_scale=P, v_scale=P, tok_stride=80),
          dict(kv_type=8, k_scale=P + 1, v_scale=P), dict(kv_type=1, tok_stride=68)]


@pytest.mark.parametrize("bad", BAD_KV, ids=str)
def test_bad_descriptors(bad):
    from toy_b200._lib import lib
    c = kv(**bad)
    assert lib().tb2_paged_append(C.byref(c), C.byref(append_args()), None) == -1
    assert lib().tb2_paged_attend(C.byref(c), C.byref(attend_args()), None) == -1


@pytest.mark.parametrize("bad", [
    dict(n_tokens=-1), dict(n_heads=0), dict(row_type=8), dict(row_type=3), dict(k=None), dict(v=None),
    dict(slots=None), dict(q_out=None), dict(ldq=255), dict(ldq=192), dict(ldk=64), dict(ldv=130), dict(ldqo=128),
    dict(k=P + 4), dict(v=P + 8), dict(q=P + 4), dict(q_out=P + 4), dict(row_type=1, ldk=132),
    dict(positions=None), dict(rope_rows=0), dict(rope=P + 4), dict(bias=P + 4), dict(ldqo=512)], ids=str)
def test_bad_append(bad):
    from toy_b200._lib import lib
    assert lib().tb2_paged_append(C.byref(kv()), C.byref(append_args(**bad)), None) == -1


@pytest.mark.parametrize("bad", [
    dict(n_req=-1), dict(n_heads=0), dict(n_heads=3), dict(row_type=8), dict(q=None), dict(out=None),
    dict(lens=None), dict(table=None), dict(ldq=255), dict(ldo=128), dict(q=P + 2), dict(out=P + 1),
    dict(table_width=0), dict(table_stride=2), dict(table_width=1 << 28, table_stride=1 << 28),
    dict(n_req=1 << 20, table_width=1 << 17, table_stride=1 << 17), dict(scale=float("nan")), dict(scale=float("inf")), dict(workspace=None), dict(workspace_bytes=8),
    dict(workspace=P + 8)], ids=str)
def test_bad_attend(bad):
    from toy_b200._lib import lib
    assert lib().tb2_paged_attend(C.byref(kv()), C.byref(attend_args(**bad)), None) == -1


@pytest.mark.parametrize("bad", [
    dict(n_req=0), dict(n_req=16385), dict(lens=None), dict(add=None), dict(table=None), dict(table_width=0),
    dict(table_stride=2), dict(free_pages=None), dict(n_free=-1), dict(state=None), dict(page_size=0),
    dict(page_size=(1 << 20) + 1), dict(n_pages=0), dict(n_tokens=-1), dict(n_tokens=0x7fffff01), dict(lens_out=None), dict(state_out=None),
    dict(cu_tokens=None), dict(slots=None), dict(positions=None), dict(requests=None),
    dict(table_width=1 << 28, table_stride=1 << 28), dict(lens_out=P + 4), dict(state_out=P - 8)], ids=str)
def test_bad_plan(bad):
    from toy_b200._lib import lib
    assert lib().tb2_paged_plan(C.byref(plan_args(**bad)), None) == -1


@pytest.mark.parametrize("bad", [
    dict(n_req=0), dict(n_req=16385), dict(lens=None), dict(done=None), dict(table=None), dict(table_width=0),
    dict(table_stride=2), dict(free_pages=None), dict(n_free=-1), dict(state=None), dict(page_size=0),
    dict(n_pages=0), dict(lens_out=None), dict(state_out=None), dict(lens_out=P - 4), dict(state_out=P + 12)], ids=str)
def test_bad_release(bad):
    from toy_b200._lib import lib
    assert lib().tb2_paged_release(C.byref(release_args(**bad)), None) == -1


def test_nothing_to_do_is_no_error():
    """No tokens, no requests: 0 without a launch (the pointers may be NULL)."""
    from toy_b200._lib import lib
    assert lib().tb2_paged_append(C.byref(kv()), C.byref(append_args(n_tokens=0, k=None, v=None, slots=None)),
                                  None) == 0
    assert lib().tb2_paged_attend(C.byref(kv()), C.byref(attend_args(n_req=0, q=None, out=None)), None) == 0


def test_null_structs():
    from toy_b200._lib import lib
    assert lib().tb2_paged_plan(None, None) == -1 and lib().tb2_paged_release(None, None) == -1
    assert lib().tb2_paged_append(None, C.byref(append_args()), None) == -1
    assert lib().tb2_paged_append(C.byref(kv()), None, None) == -1
    assert lib().tb2_paged_attend(None, C.byref(attend_args()), None) == -1
    assert lib().tb2_paged_attend(C.byref(kv()), None, None) == -1
    assert lib().tb2_paged_attend_workspace_init(None, 1 << 30, None) == -1
    assert lib().tb2_paged_attend_workspace_init(P, 8, None) == -1


def test_python_layer_refuses_host_tensors():
    from toy_b200 import paged
    x = torch.zeros((4, 2, 16, 64))
    with pytest.raises(ValueError):
        paged.PagedCache(x, x)
    i = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError):
        paged.plan(i, i, torch.zeros((4, 2), dtype=torch.int32), i, i, page_size=16, n_pages=4, n_tokens=4)
    with pytest.raises(ValueError):
        paged.release(i, i, torch.zeros((4, 2), dtype=torch.int32), i, i, page_size=16, n_pages=4)
