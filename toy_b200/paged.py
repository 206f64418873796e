"""A paged key-value cache on the GPU: the device-pointer operators tb2_paged_*
(include/toy_b200.h) over torch CUDA tensors.

A serving step is `plan` (pages, block tables and the slot map for the tokens
each request appends, from lengths that stay on the GPU), then per layer
`append` (RoPE, new K and V rows into their pages) and `attend` (one new token
per request over its pages); `release` returns finished requests' pages. Every
call runs on torch's current stream of the tensors' device, synchronises
nothing and can be captured into a CUDA graph when its outputs are given.
Arguments that do not fit are refused before anything runs, tensors that do not
go together with ValueError, what the entry points themselves refuse (a page
size of 0, more than 16384 requests in a plan, rows off their 16 bytes) with
RuntimeError. What only the device knows (page ids, slots, positions) is checked there: see
`tb2_device_error` in the header. No gradient passes through these calls: with
gradients enabled, a tensor that requires one is refused.
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
_I32, _I64, _F32 = torch.int32, torch.int64, torch.float32


def _bad(what: str):
    raise ValueError("toy_b200.paged: " + what)


def _raw_stream(index: int) -> int:
    return torch.cuda.current_stream(index).cuda_stream


# (the same handle without the Stream object around it, where torch has it: these calls cost microseconds)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _raw_stream)


def _prepare(index: int) -> None:
    with torch.cuda.device(index):
        check(lib().tb2_paged_prepare(), "tb2_paged_prepare")
    _prepared.add(index)


def _call(index: int, what: str, *args) -> None:
    """An entry point on torch's current stream of GPU `index`, which is made current for the call where it is not."""
    if index not in _prepared:
        _prepare(index)
    f = getattr(lib(), what)
    if torch.cuda.current_device() == index:
        rc = f(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = f(*args, _raw_stream(index))
    if rc:
        check(rc, what)


def _wants_grad() -> None:
    """Refuses a call one of whose tensors requires a gradient, unless gradients are disabled."""
    if torch.is_grad_enabled():
        _bad("no gradient passes through this call (use it under torch.no_grad())")


def _ints(t: torch.Tensor, n: int, index: int, what: str, dtype=_I32) -> int:
    if t.dtype is not dtype or t.get_device() != index or t.numel() < n or not t.is_contiguous():
        _bad(f"{what}: a contiguous {dtype} tensor of {n} or more on cuda:{index}")
    return t.data_ptr()


class PagedCache:
    """One layer's page pools: k and v [n_pages, n_kv, page_size, d_head] on one GPU, f32, f16 or bf16, or int8
    quants with k_scale and v_scale fp16 [n_pages, n_kv, page_size, d_head / 32] (Q8_0). The first three axes may
    have any strides that keep rows apart and on 16-byte boundaries (a permuted [n_pages, page_size, n_kv, d_head]
    pool, a layer of a larger pool), the same for k and v; the scales' are theirs divided by 32."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: Optional[torch.Tensor] = None,
                 v_scale: Optional[torch.Tensor] = None):
        if not k.is_cuda or k.dim() != 4 or k.dtype not in _CACHE:
            _bad("k: a CUDA tensor [n_pages, n_kv, page_size, d_head]")
        if v.shape != k.shape or v.dtype != k.dtype or v.device != k.device or v.stride() != k.stride():
            _bad("v: shape, type, device and strides of k")
        if k.stride(3) != 1:
            _bad("rows of d_head values are contiguous")
        q8 = k.dtype == torch.int8
        if (k_scale is not None) != q8 or (v_scale is not None) != q8:
            _bad("scales belong to int8 pools, and only there")
        # an axis of size 1 has no stride of its own
        n_pages, n_kv, page, dh = k.shape
        if max(k.shape) >= 2**31:
            _bad("k: axes below 2^31")
        strides = [k.stride(i) if k.shape[i] > 1 else k.numel() for i in range(3)]
        if q8:
            for s in (k_scale, v_scale):
                if s.dtype != torch.float16 or s.device != k.device or s.shape != k.shape[:3] + (dh // 32,):
                    _bad("scales: fp16 [n_pages, n_kv, page_size, d_head / 32] on the pools' device")
                if any(s.shape[i] > 1 and s.stride(i) * 32 != k.stride(i) for i in range(3)) or \
                        (s.shape[3] > 1 and s.stride(3) != 1):
                    _bad("scales: the pools' strides divided by 32")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.device, self.index, self.shape = k.device, k.get_device(), k.shape
        self.c = PagedKV(k.data_ptr(), v.data_ptr(), k_scale.data_ptr() if q8 else None,
                         v_scale.data_ptr() if q8 else None, _CACHE[k.dtype], n_pages, page, n_kv, dh, *strides)
        self.ref = C.byref(self.c)
        if self.index not in _prepared:   # (so that a first call may be captured into a CUDA graph)
            _prepare(self.index)


class Plan(NamedTuple):
    """What `plan` computed: see tb2_paged_plan."""
    lens: torch.Tensor        # [n] i32: lengths after the step
    state: torch.Tensor       # [4] i32: free pages left, status, tokens, pages taken
    cu_tokens: torch.Tensor   # [n + 1] i32
    slots: torch.Tensor       # [n_tokens] i64, -1 past the step's tokens
    positions: torch.Tensor   # [n_tokens] i32
    requests: torch.Tensor    # [n_tokens] i32, -1 past the step's tokens


def _table(table: torch.Tensor, n: int, index: int) -> tuple:
    """(pointer, width, row stride) of a block table [n or more, width]."""
    if table.dim() != 2 or table.dtype is not _I32 or table.get_device() != index:
        _bad(f"table: int32 [n_req, width] on cuda:{index}")
    rows, width = table.shape
    stride, one = table.stride()
    if rows < n or not 0 < width < 2**31 or (one != 1 and width > 1) or (rows > 1 and stride < width):
        _bad("table: a contiguous row of at least one page, and fewer than 2^31, per request")
    return table.data_ptr(), width, stride if rows > 1 else width


def _stack(free_pages: torch.Tensor, index: int) -> tuple:
    """(pointer, entries) of the stack of free pages."""
    if free_pages.numel() >= 2**31:   # (the entry points count in 32 bits)
        _bad("free_pages: fewer than 2^31 entries")
    return _ints(free_pages, 0, index, "free_pages"), free_pages.numel()


def plan(lens: torch.Tensor, add: torch.Tensor, table: torch.Tensor, free_pages: torch.Tensor, state: torch.Tensor, *,
         page_size: int, n_pages: int, n_tokens: int, out: Optional[Plan] = None) -> Plan:
    """Pages, table entries and slots for the add[b] tokens that request b (lens[b] tokens so far) appends. `state` is
    int32 {free pages on the stack, ..}; `table` is extended in place; n_tokens is the room of the slot map (at least
    the sum of add). `out` may hold lens and state themselves. Check state[1] of the result when it reaches the host:
    a status other than 0 left everything as it was."""
    n, dev = lens.numel(), lens.get_device()
    if dev < 0 or n < 1 or max(n, page_size, n_pages, n_tokens) >= 2**31 or n_tokens < 0:
        _bad("lens: on a GPU, of one request or more; requests, page_size, n_pages and n_tokens below 2^31")
    tp, width, stride = _table(table, n, dev)
    if out is None:   # two allocations, as each call into torch is a microsecond or more
        slots = lens.new_empty(n_tokens, dtype=_I64)
        part = lens.new_empty(2 * n_tokens + 2 * n + 5, dtype=_I32)
        positions, requests, st, new_lens, cu = part.split((n_tokens, n_tokens, 4, n, n + 1))
        out = Plan(new_lens, st, cu, slots, positions, requests)
        p = part.data_ptr()
        outs = (p + 4 * (2 * n_tokens + 4), p + 8 * n_tokens, p + 4 * (2 * n_tokens + 4 + n), slots.data_ptr(), p,
                p + 4 * n_tokens)
    else:
        outs = (_ints(out.lens, n, dev, "out.lens"), _ints(out.state, 4, dev, "out.state"),
                _ints(out.cu_tokens, n + 1, dev, "out.cu_tokens"), _ints(out.slots, n_tokens, dev, "out.slots", _I64),
                _ints(out.positions, n_tokens, dev, "out.positions"),
                _ints(out.requests, n_tokens, dev, "out.requests"))
    a = PagedPlanArgs(_ints(lens, n, dev, "lens"), _ints(add, n, dev, "add"), n, tp, width, stride,
                      *_stack(free_pages, dev), _ints(state, 4, dev, "state"),
                      page_size, n_pages, n_tokens, *outs)
    _call(dev, "tb2_paged_plan", C.byref(a))
    return out


def release(lens: torch.Tensor, done: torch.Tensor, table: torch.Tensor, free_pages: torch.Tensor, state: torch.Tensor,
            *, page_size: int, n_pages: int, lens_out: Optional[torch.Tensor] = None,
            state_out: Optional[torch.Tensor] = None) -> None:
    """The pages of every request with done[b] != 0 go back on the stack, its table row is cleared and its length set
    to 0; lens and state are updated in place unless other tensors are given."""
    n, dev = lens.numel(), lens.get_device()
    if dev < 0 or n < 1 or max(n, page_size, n_pages) >= 2**31:
        _bad("lens: on a GPU, of one request or more; requests, page_size and n_pages below 2^31")
    a = PagedReleaseArgs(_ints(lens, n, dev, "lens"), _ints(done, n, dev, "done"), n, *_table(table, n, dev),
                         *_stack(free_pages, dev), _ints(state, 4, dev, "state"),
                         page_size, n_pages, _ints(lens if lens_out is None else lens_out, n, dev, "lens_out"),
                         _ints(state if state_out is None else state_out, 4, dev, "state_out"))
    _call(dev, "tb2_paged_release", C.byref(a))


def _rows(t: torch.Tensor, n: int, heads: int, dh: int, dtype, index: int, what: str) -> int:
    """The row stride of t [n, heads, dh], its last two axes dense."""
    if t.shape == (n, heads, dh) and t.dtype is dtype and t.get_device() == index:
        s0, s1, s2 = t.stride()
        if s2 == 1 and (s1 == dh or heads == 1):
            if n <= 1:
                return heads * dh
            if s0 >= heads * dh:
                return s0
    _bad(f"{what}: {dtype} [{n}, {heads}, {dh}] on cuda:{index}, each token's heads contiguous")


def append(cache: PagedCache, slots: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
           q: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None,
           positions: Optional[torch.Tensor] = None, rope: Optional[torch.Tensor] = None,
           bias: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """New rows k, v [n, n_kv, d_head] into the pages at slots (negative: not stored), q [n, n_heads, d_head] turned
    into q_out (made when None; may be q). rope: f32 [rows, d_head / 2, 2] (cos, sin), indexed by positions; bias:
    f32 [(n_heads + 2 n_kv) d_head], added first. Returns q_out."""
    _, n_kv, _, dh = cache.shape
    dev, dt = cache.index, k.dtype
    n = k.shape[0]
    if dt not in _ROW or n >= 2**31:
        _bad("rows are f32, f16 or bf16, of fewer than 2^31 tokens")
    if k.requires_grad or v.requires_grad or q is not None and q.requires_grad or \
            bias is not None and bias.requires_grad:
        _wants_grad()
    ldk, ldv = _rows(k, n, n_kv, dh, dt, dev, "k"), _rows(v, n, n_kv, dh, dt, dev, "v")
    heads = ldq = ldqo = 0
    qp = op = bp = rp = pp = None
    rows = 0
    if q is not None:
        heads = q.shape[1] if q.dim() == 3 else 0
        ldq = _rows(q, n, heads, dh, dt, dev, "q")
        if q_out is None:
            q_out = q.new_empty((n, heads, dh))
        ldqo = _rows(q_out, n, heads, dh, dt, dev, "q_out")
        qp, op = q.data_ptr(), q_out.data_ptr()
    if rope is not None:
        rows, *pairs = rope.shape
        if positions is None or rope.dtype is not _F32 or rope.get_device() != dev or not rope.is_contiguous() or \
                pairs != [dh // 2, 2]:
            _bad("rope: contiguous f32 [rows, d_head / 2, 2] with positions")
        rp = rope.data_ptr()
    if positions is not None:
        pp = _ints(positions, n, dev, "positions")
    if bias is not None:
        # without q the bias still has the layout of a whole row: [n_heads | n_kv | n_kv], n_heads from its length
        if q is None:
            heads = bias.numel() // dh - 2 * n_kv
        if bias.dtype is not _F32 or bias.get_device() != dev or not bias.is_contiguous() or heads < 0 or \
                bias.numel() != (heads + 2 * n_kv) * dh:
            _bad("bias: contiguous f32 [(n_heads + 2 n_kv) d_head]")
        bp = bias.data_ptr()
    a = PagedAppendArgs(n, heads, _ROW[dt], qp, ldq, k.data_ptr(), ldk, v.data_ptr(), ldv, op, ldqo, bp, rp, rows, pp,
                        _ints(slots, n, dev, "slots", _I64))
    _call(dev, "tb2_paged_append", cache.ref, C.byref(a))
    return q_out


def attend_workspace(device=None) -> torch.Tensor:
    """A workspace for `attend` on one GPU, set up. Calls that may overlap (two streams, two captured graphs) need one
    each."""
    dev = torch.device("cuda" if device is None else device)
    index = torch.cuda.current_device() if dev.index is None else dev.index
    w = torch.empty(lib().tb2_paged_attend_workspace(), device=torch.device("cuda", index), dtype=torch.uint8)
    _call(index, "tb2_paged_attend_workspace_init", w.data_ptr(), w.numel())
    return w


def attend(cache: PagedCache, q: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, *,
           out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None, scale: Optional[float] = None,
           workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One new token per request over its pages: q [n, n_heads, d_head] (f32, f16 or bf16), table int32 [n, width],
    lens int32 [n] (the new token counted); out [n, n_heads, d_head] of q's type, lse f32 [n, n_heads] when given.
    scale defaults to d_head^-0.5; a workspace is made for the call when None."""
    _, n_kv, _, dh = cache.shape
    dev, dt = cache.index, q.dtype
    if q.dim() != 3 or dt not in _ROW:
        _bad("q: f32, f16 or bf16 [n, n_heads, d_head]")
    if q.requires_grad or out is not None and out.requires_grad:
        _wants_grad()
    n, heads, _ = q.shape
    if heads < 1 or heads % n_kv:
        _bad("n_heads is a multiple of the cache's n_kv")
    ldq = _rows(q, n, heads, dh, dt, dev, "q")
    if out is None:
        out = q.new_empty((n, heads, dh))
    ldo = _rows(out, n, heads, dh, dt, dev, "out")
    lp = None
    if lse is not None:
        if lse.dtype is not _F32 or lse.get_device() != dev or not lse.is_contiguous() or lse.shape != (n, heads):
            _bad("lse: contiguous f32 [n, n_heads]")
        lp = lse.data_ptr()
    if workspace is None:
        workspace = attend_workspace(cache.device)
    elif workspace.get_device() != dev or workspace.dtype is not torch.uint8 or not workspace.is_contiguous():
        _bad("workspace: from attend_workspace, on the cache's device")
    a = PagedAttendArgs(n, heads, _ROW[dt], q.data_ptr(), ldq, out.data_ptr(), ldo, *_table(table, n, dev),
                        _ints(lens, n, dev, "lens"), dh ** -0.5 if scale is None else scale, lp, workspace.data_ptr(),
                        workspace.numel())
    _call(dev, "tb2_paged_attend", cache.ref, C.byref(a))
    return out
