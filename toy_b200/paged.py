"""A paged key-value cache on the GPU: the device-pointer operators tb2_paged_*
(include/toy_b200.h) over torch CUDA tensors.

A serving step is `plan` (pages, block tables and the slot map for the tokens
each request appends, from lengths that stay on the GPU), then per layer
`append` (RoPE, new K and V rows into their pages) and `attend` (one new token
per request over its pages); `release` returns finished requests' pages. Every
call runs on torch's current stream of the tensors' device, synchronises
nothing and can be captured into a CUDA graph when its outputs are given.
Arguments that do not fit are refused with ValueError before anything runs.
What only the device knows (page ids, slots, positions) is checked there: see
`tb2_device_error` in the header.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

import torch

from ._lib import PagedAppendArgs, PagedAttendArgs, PagedKV, PagedPlanArgs, PagedReleaseArgs, check, lib

# ggml type ids
_ROW = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}
_CACHE = {**_ROW, torch.int8: 8}
_prepared: set = set()


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError("toy_b200.paged: " + what)


class _on:
    """The device of a call's tensors made current where it is not (and its error word set up once)."""

    def __init__(self, device: torch.device):
        self.index = device.index
        self.prev = torch.cuda.current_device()

    def __enter__(self) -> int:
        if self.prev != self.index:
            torch.cuda.set_device(self.index)
        if self.index not in _prepared:
            check(lib().tb2_paged_prepare(), "tb2_paged_prepare")
            _prepared.add(self.index)
        return torch.cuda.current_stream(self.index).cuda_stream

    def __exit__(self, *exc) -> None:
        if self.prev != self.index:
            torch.cuda.set_device(self.prev)


def _ints(t: torch.Tensor, n: int, device, what: str, dtype=torch.int32) -> int:
    _need(t.dtype == dtype and t.device == device and t.is_contiguous() and t.numel() >= n,
          f"{what}: a contiguous {dtype} tensor of {n} or more on {device}")
    return t.data_ptr()


class PagedCache:
    """One layer's page pools: k and v [n_pages, n_kv, page_size, d_head] on one GPU, f32, f16 or bf16, or int8
    quants with k_scale and v_scale fp16 [n_pages, n_kv, page_size, d_head / 32] (Q8_0). The first three axes may
    have any strides that keep rows apart and on 16-byte boundaries (a permuted [n_pages, page_size, n_kv, d_head]
    pool, a layer of a larger pool), the same for k and v; the scales' are theirs divided by 32."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: Optional[torch.Tensor] = None,
                 v_scale: Optional[torch.Tensor] = None):
        _need(k.is_cuda and k.dim() == 4 and k.dtype in _CACHE, "k: a CUDA tensor [n_pages, n_kv, page_size, d_head]")
        _need(v.shape == k.shape and v.dtype == k.dtype and v.device == k.device and v.stride() == k.stride(),
              "v: shape, type, device and strides of k")
        _need(k.stride(3) == 1, "rows of d_head values are contiguous")
        q8 = k.dtype == torch.int8
        _need((k_scale is not None) == q8 and (v_scale is not None) == q8, "scales belong to int8 pools, and only there")
        # an axis of size 1 has no stride of its own
        n_pages, n_kv, page, dh = k.shape
        strides = [k.stride(i) if k.shape[i] > 1 else k.numel() for i in range(3)]
        if q8:
            for s in (k_scale, v_scale):
                _need(s.dtype == torch.float16 and s.device == k.device and s.shape == k.shape[:3] + (dh // 32,),
                      "scales: fp16 [n_pages, n_kv, page_size, d_head / 32] on the pools' device")
                _need(all(s.shape[i] == 1 or s.stride(i) * 32 == k.stride(i) for i in range(3)) and
                      (s.shape[3] == 1 or s.stride(3) == 1), "scales: the pools' strides divided by 32")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.device, self.shape = k.device, k.shape
        self.c = PagedKV(k.data_ptr(), v.data_ptr(), k_scale.data_ptr() if q8 else None,
                         v_scale.data_ptr() if q8 else None, _CACHE[k.dtype], n_pages, page, n_kv, dh, *strides)
        self._ref = C.byref(self.c)


class Plan(NamedTuple):
    """What `plan` computed: see tb2_paged_plan."""
    lens: torch.Tensor        # [n] i32: lengths after the step
    state: torch.Tensor       # [4] i32: free pages left, status, tokens, pages taken
    cu_tokens: torch.Tensor   # [n + 1] i32
    slots: torch.Tensor       # [n_tokens] i64, -1 past the step's tokens
    positions: torch.Tensor   # [n_tokens] i32
    requests: torch.Tensor    # [n_tokens] i32, -1 past the step's tokens


def _table(table: torch.Tensor, n: int, device) -> None:
    _need(table.dim() == 2 and table.shape[0] >= n and table.dtype == torch.int32 and table.device == device and
          table.shape[1] >= 1 and table.stride(1) == 1 and (table.shape[0] == 1 or table.stride(0) >= table.shape[1]),
          "table: int32 [n_req, width] on the lengths' device, rows contiguous")


def _table_stride(table: torch.Tensor) -> int:
    return max(table.stride(0), table.shape[1])


def plan(lens: torch.Tensor, add: torch.Tensor, table: torch.Tensor, free_pages: torch.Tensor, state: torch.Tensor, *,
         page_size: int, n_pages: int, n_tokens: int, out: Optional[Plan] = None) -> Plan:
    """Pages, table entries and slots for the add[b] tokens that request b (lens[b] tokens so far) appends. `state` is
    int32 {free pages on the stack, ..}; `table` is extended in place; n_tokens is the room of the slot map (at least
    the sum of add). `out` may hold lens and state themselves. Check state[1] of the result when it reaches the host:
    a status other than 0 left everything as it was."""
    n, dev = lens.numel(), lens.device
    _need(lens.is_cuda and n >= 1 and 0 <= n_tokens < 2**31, "lens on a GPU, n_tokens not negative")
    _table(table, n, dev)
    if out is None:
        i32 = lambda k: torch.empty(k, device=dev, dtype=torch.int32)  # noqa: E731
        out = Plan(i32(n), i32(4), i32(n + 1), torch.empty(n_tokens, device=dev, dtype=torch.int64), i32(n_tokens),
                   i32(n_tokens))
    a = PagedPlanArgs(_ints(lens, n, dev, "lens"), _ints(add, n, dev, "add"), n, table.data_ptr(), table.shape[1],
                      _table_stride(table), _ints(free_pages, 0, dev, "free_pages"), free_pages.numel(),
                      _ints(state, 4, dev, "state"), page_size, n_pages, n_tokens, _ints(out.lens, n, dev, "out.lens"),
                      _ints(out.state, 4, dev, "out.state"), _ints(out.cu_tokens, n + 1, dev, "out.cu_tokens"),
                      _ints(out.slots, n_tokens, dev, "out.slots", torch.int64),
                      _ints(out.positions, n_tokens, dev, "out.positions"),
                      _ints(out.requests, n_tokens, dev, "out.requests"))
    with _on(dev) as st:
        check(lib().tb2_paged_plan(C.byref(a), st), "tb2_paged_plan")
    return out


def release(lens: torch.Tensor, done: torch.Tensor, table: torch.Tensor, free_pages: torch.Tensor, state: torch.Tensor,
            *, page_size: int, n_pages: int, lens_out: Optional[torch.Tensor] = None,
            state_out: Optional[torch.Tensor] = None) -> None:
    """The pages of every request with done[b] != 0 go back on the stack, its table row is cleared and its length set
    to 0; lens and state are updated in place unless other tensors are given."""
    n, dev = lens.numel(), lens.device
    _need(lens.is_cuda and n >= 1, "lens on a GPU")
    _table(table, n, dev)
    a = PagedReleaseArgs(_ints(lens, n, dev, "lens"), _ints(done, n, dev, "done"), n, table.data_ptr(),
                         table.shape[1], _table_stride(table), _ints(free_pages, 0, dev, "free_pages"),
                         free_pages.numel(), _ints(state, 4, dev, "state"), page_size, n_pages,
                         _ints(lens if lens_out is None else lens_out, n, dev, "lens_out"),
                         _ints(state if state_out is None else state_out, 4, dev, "state_out"))
    with _on(dev) as st:
        check(lib().tb2_paged_release(C.byref(a), st), "tb2_paged_release")


def _rows(t: torch.Tensor, n: int, heads: int, dh: int, dtype, device, what: str) -> int:
    """[n, heads, dh] with the last two axes dense: the row stride."""
    _need(t.dim() == 3 and t.shape == (n, heads, dh) and t.dtype == dtype and t.device == device and
          t.stride(2) == 1 and (heads == 1 or t.stride(1) == dh) and (n == 1 or t.stride(0) >= heads * dh),
          f"{what}: {dtype} [{n}, {heads}, {dh}] on {device}, each token's heads contiguous")
    return t.stride(0) if n > 1 else heads * dh


def append(cache: PagedCache, slots: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
           q: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None,
           positions: Optional[torch.Tensor] = None, rope: Optional[torch.Tensor] = None,
           bias: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """New rows k, v [n, n_kv, d_head] into the pages at slots (negative: not stored), q [n, n_heads, d_head] turned
    into q_out (made when None; may be q). rope: f32 [rows, d_head / 2, 2] (cos, sin), indexed by positions; bias:
    f32 [(n_heads + 2 n_kv) d_head], added first. Returns q_out."""
    _, n_kv, _, dh = cache.shape
    n, dev = k.shape[0], cache.device
    _need(k.dtype in _ROW, "rows are f32, f16 or bf16")
    ldk, ldv = _rows(k, n, n_kv, dh, k.dtype, dev, "k"), _rows(v, n, n_kv, dh, k.dtype, dev, "v")
    heads = ldq = ldqo = 0
    if q is not None:
        heads = q.shape[1]
        ldq = _rows(q, n, heads, dh, k.dtype, dev, "q")
        if q_out is None:
            q_out = torch.empty((n, heads, dh), device=dev, dtype=q.dtype)
        ldqo = _rows(q_out, n, heads, dh, k.dtype, dev, "q_out")
    _need(rope is None or (positions is not None and rope.dtype == torch.float32 and rope.device == dev and
                           rope.is_contiguous() and rope.shape[1:] == (dh // 2, 2)),
          "rope: contiguous f32 [rows, d_head / 2, 2] with positions")
    if bias is not None:
        # without q the bias still has the layout of a whole row: [n_heads | n_kv | n_kv], n_heads from its length
        if q is None:
            heads = bias.numel() // dh - 2 * n_kv
        _need(bias.dtype == torch.float32 and bias.device == dev and bias.is_contiguous() and heads >= 0 and
              bias.numel() == (heads + 2 * n_kv) * dh, "bias: contiguous f32 [(n_heads + 2 n_kv) d_head]")
    a = PagedAppendArgs(n, heads, _ROW[k.dtype], q.data_ptr() if q is not None else None, ldq, k.data_ptr(), ldk,
                        v.data_ptr(), ldv, q_out.data_ptr() if q is not None else None, ldqo,
                        bias.data_ptr() if bias is not None else None, rope.data_ptr() if rope is not None else None,
                        rope.shape[0] if rope is not None else 0,
                        _ints(positions, n, dev, "positions") if positions is not None else None,
                        _ints(slots, n, dev, "slots", torch.int64))
    with _on(dev) as st:
        check(lib().tb2_paged_append(cache._ref, C.byref(a), st), "tb2_paged_append")
    return q_out


def attend_workspace(device=None) -> torch.Tensor:
    """A workspace for `attend` on one GPU, set up. Calls that may overlap (two streams, two captured graphs) need one
    each."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    if dev.index is None:
        dev = torch.device("cuda", torch.cuda.current_device())
    with _on(dev) as st:
        w = torch.empty(lib().tb2_paged_attend_workspace(), device=dev, dtype=torch.uint8)
        check(lib().tb2_paged_attend_workspace_init(w.data_ptr(), w.numel(), st), "tb2_paged_attend_workspace_init")
    return w


def attend(cache: PagedCache, q: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, *,
           out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None, scale: Optional[float] = None,
           workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One new token per request over its pages: q [n, n_heads, d_head] (f32, f16 or bf16), table int32 [n, width],
    lens int32 [n] (the new token counted); out [n, n_heads, d_head] of q's type, lse f32 [n, n_heads] when given.
    scale defaults to d_head^-0.5; a workspace is made for the call when None."""
    _, n_kv, _, dh = cache.shape
    dev = cache.device
    _need(q.dim() == 3 and q.dtype in _ROW, "q: f32, f16 or bf16 [n, n_heads, d_head]")
    n, heads = q.shape[0], q.shape[1]
    _need(heads >= 1 and heads % n_kv == 0, "n_heads is a multiple of the cache's n_kv")
    ldq = _rows(q, n, heads, dh, q.dtype, dev, "q")
    if out is None:
        out = torch.empty((n, heads, dh), device=dev, dtype=q.dtype)
    ldo = _rows(out, n, heads, dh, q.dtype, dev, "out")
    _table(table, n, dev)
    _need(lse is None or (lse.dtype == torch.float32 and lse.device == dev and lse.is_contiguous() and
                          lse.shape == (n, heads)), "lse: contiguous f32 [n, n_heads]")
    if workspace is None:
        workspace = attend_workspace(dev)
    _need(workspace.device == dev and workspace.dtype == torch.uint8 and workspace.is_contiguous(),
          "workspace: from attend_workspace, on the cache's device")
    a = PagedAttendArgs(n, heads, _ROW[q.dtype], q.data_ptr(), ldq, out.data_ptr(), ldo, table.data_ptr(),
                        table.shape[1], _table_stride(table), _ints(lens, n, dev, "lens"),
                        dh ** -0.5 if scale is None else scale, lse.data_ptr() if lse is not None else None,
                        workspace.data_ptr(), workspace.numel())
    with _on(dev) as st:
        check(lib().tb2_paged_attend(cache._ref, C.byref(a), st), "tb2_paged_attend")
    return out
