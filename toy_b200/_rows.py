"""What logprobs, experts and multi_adamw share: calls of the tb2_* entry points
on torch's current stream, and checks of row tensors."""
from __future__ import annotations

import torch
import torch.autograd.forward_ad as _forward_ad

from ._lib import check, lib

# ggml type ids
ROW_TYPE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}
F32, I32, I64 = torch.float32, torch.int32, torch.int64
_prepared: set = set()
_entries: dict = {}


def _raw_stream(index: int) -> int:
    return torch.cuda.current_stream(index).cuda_stream


# (the same handle without the Stream object around it, where torch has it: these calls cost microseconds)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _raw_stream)


def prepare(device=None) -> None:
    """One-time set-up on a GPU (the current one by default); a first call of any operator makes it too, but not one
    that is captured into a CUDA graph."""
    dev = torch.device("cuda" if device is None else device)
    index = torch.cuda.current_device() if dev.index is None else dev.index
    with torch.cuda.device(index):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("toy_b200: call prepare() before a first call is captured into a CUDA graph")
        check(lib().tb2_rows_prepare(), "tb2_rows_prepare")
    _prepared.add(index)


# (the current device without torch.cuda's checks around it, where torch has it)
_current = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def call(index: int, what: str, *args) -> None:
    """An entry point on torch's current stream of GPU `index`, which is made current for the call where it is not."""
    f = _entries.get(what)
    if f is None:
        f = _entries[what] = getattr(lib(), what)
    if index not in _prepared:
        prepare(torch.device("cuda", index))
    if _current() == index:
        rc = f(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = f(*args, _raw_stream(index))
    if rc == -1:
        bad(f"{what}: arguments that do not fit (a result that lies over an operand, but for those that may)")
    if rc:
        check(rc, what)


def bad(what: str):
    raise ValueError("toy_b200: " + what)


def dense(t: torch.Tensor, shape, dtype, index: int, what: str) -> int:
    """The address of a contiguous tensor of this shape and type on GPU `index`."""
    if t.shape != shape or t.dtype is not dtype or t.get_device() != index or not t.is_contiguous():
        bad(f"{what}: contiguous {dtype} {list(shape)} on cuda:{index}")
    return t.data_ptr()


def rows(t: torch.Tensor, n: int, d: int, dtype, index: int, what: str) -> int:
    """The row stride of t [n, d], each row contiguous and a row apart at least."""
    if t.shape == (n, d) and t.dtype is dtype and t.get_device() == index:
        s0, s1 = t.stride()
        if s1 == 1 or d == 1:
            if n <= 1:
                return d
            if s0 >= d:
                return s0
    bad(f"{what}: {dtype} [{n}, {d}] on cuda:{index}, rows contiguous and apart")


def written(*tensors) -> None:
    """Notes for autograd that the tensors' values have changed (what it saved of them is stale)."""
    torch.autograd.graph.increment_version([t for t in tensors if t is not None])


def no_tangent(*tensors) -> None:
    """Refuses tensors with a tangent: none of the operators has a derivative in forward mode, and a result without one
    would stand for a derivative of zero."""
    if getattr(_forward_ad, "_current_level", 0) >= 0:
        for t in tensors:
            if t is not None and _forward_ad.unpack_dual(t).tangent is not None:
                bad("no forward-mode derivative (the tensor has a tangent)")


def no_captured_leaf(*tensors) -> None:
    """Refuses a leaf's gradient in a CUDA graph: it is added to the leaf on the stream that the leaf was first used on,
    which a capture of another stream may not wait for."""
    if any(t is not None and t.requires_grad and t.is_leaf for t in tensors) and \
            torch.cuda.is_current_stream_capturing():
        raise RuntimeError("toy_b200: a leaf's gradient is not captured into a CUDA graph (capture the gradient's own "
                           "call instead)")
