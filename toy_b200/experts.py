"""Tokens sorted by expert and back: tb2_expert_* (include/toy_b200.h) over torch
CUDA tensors.

A mixture-of-experts block is `sort` (where each (token, choice) slot goes, from
the router's choices, on the GPU), `dispatch` (the tokens' rows in the experts'
order), the experts' products over rows offsets[e] .. offsets[e + 1], and
`combine` (the slots' rows back onto their tokens with the router's weights).
`dispatch` and `combine` are differentiable; `dispatch_grad` and `combine_grad`
are their gradients as calls of their own. Every call runs on torch's current
stream, synchronises nothing, and can be captured into a CUDA graph once
`prepare` has run. Arguments that do not fit are refused with ValueError before
anything runs; expert ids and places out of range are left out and reported on
the device (`tb2_device_error` in the header).
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from ._lib import ExpertRowsArgs, ExpertSortArgs
from ._rows import F32, I32, I64, ROW_TYPE, bad, call, dense, no_captured_leaf, no_tangent, prepare, rows, written

__all__ = ["Routing", "combine", "combine_grad", "dispatch", "dispatch_grad", "prepare", "sort"]
MAX_EXPERTS = 1024


class Routing(NamedTuple):
    """What `sort` computed: see tb2_expert_sort."""
    offsets: torch.Tensor     # [n_experts + 1] i32
    order: torch.Tensor       # [tokens * used] i32: the slots (token * used + choice) by expert, -1 past the last
    pos: torch.Tensor         # [tokens, used] i32: each slot's place in order, -1 for a slot of no expert


def sort(ids: torch.Tensor, n_experts: int, *, out: Optional[Routing] = None) -> Routing:
    """The slots of ids [tokens, used] (i32 or i64; negative: no expert) sorted by expert, each expert's in slot
    order. out: buffers to fill (a backward that still needs what they held is refused)."""
    dev, n, wide = ids.get_device(), ids.numel(), ids.dtype is I64
    if dev < 0 or ids.dim() != 2 or not (wide or ids.dtype is I32) or not ids.is_contiguous() or n >= 2**31 or \
            ids.shape[1] < 1:
        bad("ids: contiguous i32 or i64 [tokens, used] on a GPU, fewer than 2^31")
    if not 1 <= n_experts <= MAX_EXPERTS:
        bad(f"n_experts is 1 to {MAX_EXPERTS}")
    fresh = out is None
    if fresh:
        out = Routing(ids.new_empty(n_experts + 1, dtype=I32), ids.new_empty(n, dtype=I32),
                      ids.new_empty(ids.shape, dtype=I32))
    else:
        dense(out.offsets, (n_experts + 1,), I32, dev, "out.offsets")
        dense(out.order, (n,), I32, dev, "out.order")
        dense(out.pos, ids.shape, I32, dev, "out.pos")
    a = ExpertSortArgs(ids.data_ptr(), 8 if wide else 4, n, n_experts, out.offsets.data_ptr(), out.order.data_ptr(),
                       out.pos.data_ptr())
    call(dev, "tb2_expert_sort", a)
    if not fresh:
        written(*out)
    return out


def _args(r: Routing, x: torch.Tensor, xs: torch.Tensor, weights: Optional[torch.Tensor]) -> tuple:
    """(device, arguments) of tokens x [tokens, d] and sorted rows xs [rows, d]."""
    pos, dtype, dev = r.pos, x.dtype, x.get_device()
    if pos.dim() != 2 or x.dim() != 2 or xs.dim() != 2 or dtype not in ROW_TYPE or dev < 0:
        bad("rows are f32, f16 or bf16, tokens [tokens, d] and sorted rows [rows, d] on a GPU")
    shape, d, n = pos.shape, x.shape[1], xs.shape[0]
    if d < 1 or d >= 2**31 - 256 or n >= 2**31:
        bad("rows are of one value or more, and fewer than 2^31 of fewer than 2^31 - 256")
    return dev, ExpertRowsArgs(shape[0], shape[1], d, n, ROW_TYPE[dtype], x.data_ptr(),
                               rows(x, shape[0], d, dtype, dev, "tokens"), xs.data_ptr(),
                               rows(xs, n, d, dtype, dev, "sorted rows"), dense(pos, shape, I32, dev, "pos"),
                               None if weights is None else dense(weights, shape, F32, dev, "weights"))


def _sorted(r: Routing, dev: int) -> int:
    """The address of the number of sorted slots, the last of the offsets."""
    n = r.offsets.numel()
    return dense(r.offsets, (n,) if n else None, I32, dev, "offsets") + 4 * (n - 1)


def _wanted(*tensors) -> bool:
    """Whether a gradient of one of the tensors is wanted."""
    for t in tensors:
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            return True
    return False


def _no_grad(*tensors) -> None:
    if _wanted(*tensors):
        bad("no gradient passes through this call (use it under torch.no_grad())")


def _noted(out: Optional[torch.Tensor], result):
    """The result of a call that has written out: autograd is told, of a call that was not refused."""
    if out is not None:
        written(out)
    return result


def _dispatch(x, r, out):
    no_tangent(x, out)
    fresh = out is None
    if fresh:
        out = x.new_empty((r.pos.numel(), x.shape[1] if x.dim() == 2 else 0))
    dev, a = _args(r, x, out, None)
    if fresh:
        a.n_sorted = _sorted(r, dev)
    call(dev, "tb2_expert_dispatch", a)
    return out


def _combine(z, r, weights, residual, out):
    no_tangent(z, weights, residual, out)
    if out is None:
        out = z.new_empty((r.pos.shape[0], z.shape[1] if z.dim() == 2 else 0))
    dev, a = _args(r, out, z, weights)
    if residual is not None:
        a.ldr = rows(residual, a.n_tokens, a.d, z.dtype, dev, "residual")
        a.residual = residual.data_ptr()
    call(dev, "tb2_expert_combine", a)
    return out


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, offsets, order, pos):
        ctx.save_for_backward(offsets, order, pos)
        return _dispatch(x, Routing(offsets, order, pos), None)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dxs):
        return _combine(_whole(dxs), Routing(*ctx.saved_tensors), None, None, None), None, None, None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, weights, residual, offsets, order, pos):
        ctx.save_for_backward(z, weights, offsets, order, pos)
        return _combine(z, Routing(offsets, order, pos), weights, residual, None)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        z, weights, *r = ctx.saved_tensors
        need_z, need_w, need_r = ctx.needs_input_grad[:3]
        dz = dw = None
        if need_z or need_w:
            dz, dw = _combine_grad(_whole(dy), z.detach(), Routing(*r), None if weights is None else weights.detach(),
                                   None, need_z, need_w)
        return dz, dw, dy if need_r else None, None, None, None


def _whole(g: torch.Tensor) -> torch.Tensor:
    """A gradient with rows that lie apart (an expanded one has none)."""
    return g if g.stride(1) == 1 and (g.shape[0] <= 1 or g.stride(0) >= g.shape[1]) else g.contiguous()


def dispatch(x: torch.Tensor, r: Routing, *, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The rows of x [tokens, d] at their slots' places, [tokens * used, d]: rows past the last slot's are zero, or as
    they were where `out` is given. Differentiable in x (without out)."""
    if out is None and _wanted(x):
        no_tangent(x)
        no_captured_leaf(x)
        return _Dispatch.apply(x, *r)
    _no_grad(x, out)
    return _noted(out, _dispatch(x, r, out))


def dispatch_grad(dxs: torch.Tensor, r: Routing, *, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The gradient of `dispatch`: each token's sum of its slots' rows of dxs, choices ascending."""
    _no_grad(dxs, out)
    return _noted(out, _combine(dxs, r, None, None, out))


def combine(z: torch.Tensor, r: Routing, weights: Optional[torch.Tensor] = None, *,
            residual: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """residual [tokens, d] (None: 0) plus each token's sum of weights (f32 [tokens, used]; None: 1) times its slots'
    rows of z [rows, d], choices ascending, in f32, rounded once. out may be the residual. Differentiable in z, weights
    and residual (without out)."""
    if out is None and _wanted(z, weights, residual):
        no_tangent(z, weights, residual)
        no_captured_leaf(z, weights, residual)
        return _Combine.apply(z, weights, residual, *r)
    _no_grad(z, weights, residual, out)
    return _noted(out, _combine(z, r, weights, residual, out))


def _combine_grad(dy, z, r, weights, out, want_z, want_w):
    no_tangent(dy, z, weights, out)
    fresh = out is None and want_z
    if fresh:
        out = z.new_empty(z.shape)
    dev, a = _args(r, dy, z, weights)
    dw = z.new_empty(r.pos.shape, dtype=F32) if want_w else None
    if want_z:
        a.ldd = rows(out, a.n_rows, a.d, z.dtype, dev, "out")
        a.d_xs = out.data_ptr()
        if fresh:
            a.n_sorted = _sorted(r, dev)
            if not a.n_tokens:
                out.zero_()
    if want_w:
        a.d_weights = dw.data_ptr()
    call(dev, "tb2_expert_combine_grad", a)
    return out, dw


def combine_grad(dy: torch.Tensor, z: torch.Tensor, r: Routing, weights: Optional[torch.Tensor] = None, *,
                 out: Optional[torch.Tensor] = None) -> tuple:
    """(dz, dw) of `combine`: the slots' rows of dz are weights * dy, dw = <dy, z> (0 for slots of no expert). Rows of
    dz that no slot has are zero, or as they were where `out` is given; out may be z."""
    _no_grad(dy, z, weights, out)
    return _noted(out, _combine_grad(dy, z, r, weights, out, True, True))
