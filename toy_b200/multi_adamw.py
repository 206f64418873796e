"""An AdamW step over many torch CUDA tensors in one launch, moments in 32 or in 8
bits: tb2_adamw_multi (include/toy_b200.h).

The step is the framework's own (opt_step_adamw with the 7-slot row of
`toy_b200.AdamW.hp`), its root and quotient within 2^-22. With 8 bits a weight's
two moments take 2.03 bytes instead of 8: blocks of 256 values share a power of
two, m is held as e4m3 and v as the e4m3 of its square root, each the step's
value rounded once.

Train with a seed. A step moves v by a thousandth of its way (beta2 = 0.999), and
the nearest of codes that lie 6 to 12 % apart is the one it had: without a seed v
stops growing after a dozen steps. With one, a value goes to the code above or
below with the probability of its place between them, so that v follows on
average. (Without: for states that are to be the exact ones' nearest codes, and
for moments that a step moves by more than that.)
"""
from __future__ import annotations

import ctypes as C
import warnings
from operator import attrgetter
from typing import Optional, Sequence

import numpy as np
import torch

from ._lib import AdamwMultiArgs, AdamwTensor
from ._rows import F32, I64, ROW_TYPE, bad, call, dense, prepare

__all__ = ["MultiAdamW", "prepare"]
BLOCK = 256
_HELD = torch.float8_e4m3fn
_note = torch.autograd.graph.increment_version   # of a list: autograd is told that its tensors' values have changed
_SHAPE, _DTYPE = attrgetter("shape"), attrgetter("dtype")
_POINTER, _DEVICE, _DENSE = torch.Tensor.data_ptr, torch.Tensor.get_device, torch.Tensor.is_contiguous
# tb2_adamw_tensor, by columns
_COLUMNS = np.dtype([(name, np.int64 if kind is C.c_longlong else np.uint64) for name, kind in AdamwTensor._fields_])


def _pointers(tensors: Sequence[torch.Tensor], shapes: list, dtype, index: int, what: str) -> list:
    """The addresses of contiguous tensors of these shapes, of one type, on GPU `index`. (Checked attribute by
    attribute: for hundreds of small tensors this is the call's time.)"""
    if list(map(_SHAPE, tensors)) != shapes or any(d is not dtype for d in set(map(_DTYPE, tensors))) or \
            set(map(_DEVICE, tensors)) != {index} or not all(map(_DENSE, tensors)):
        bad(f"{what}: contiguous {dtype} tensors of the weights' shapes on cuda:{index}")
    return list(map(_POINTER, tensors))


def _apart(lists: Sequence[Sequence[torch.Tensor]]) -> None:
    """Refuses tensors that share memory: a step writes all of them."""
    spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for x in lists for t in x if t.numel())
    if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
        bad("weights, copies and state do not share memory")


class MultiAdamW:
    """The optimizer of `params`: contiguous tensors of one type (f32, f16 or bf16) on one GPU. copies: tensors of their
    shapes, of one 16-bit type, that each step sets to the weights rounded (for weights kept in f32). state: (m, v,
    m_scale, v_scale) to go on from, lists of tensors that the optimizer then owns, the scales None for 32 bits;
    empty moments when None. The state is in the attributes of these names, in the memory that it has at first (copy_
    into it, or set_moments, changes it); weights and copies are followed where theirs changes, and refused where they
    no longer fit."""

    def __init__(self, params: Sequence[torch.Tensor], *, bits: int = 8, copies: Optional[Sequence] = None,
                 state: Optional[tuple] = None):
        self.params = list(params)
        if bits not in (8, 32):
            bad("bits is 8 or 32")
        if not self.params or not self.params[0].is_cuda or self.params[0].dtype not in ROW_TYPE:
            bad("params: one f32, f16 or bf16 tensor or more on a GPU")
        self.bits, self.dtype, self.index = bits, self.params[0].dtype, self.params[0].get_device()
        self.device = self.params[0].device
        n = [p.numel() for p in self.params]
        self._shapes = [p.shape for p in self.params]
        self.copies = list(copies) if copies else None
        self.copy_dtype = self.copies[0].dtype if copies else torch.bfloat16
        if copies and (len(self.copies) != len(n) or self.copy_dtype not in (torch.float16, torch.bfloat16)):
            bad("copies: one f16 or bf16 tensor per weight")
        blocks = [-(-k // BLOCK) for k in n]
        if state is None:
            def zeros(sizes, dtype):
                return [torch.zeros(k, device=self.device, dtype=dtype) for k in sizes]
            if bits == 32:
                state = (zeros(n, F32), zeros(n, F32), None, None)
            else:
                state = ([t.view(_HELD) for t in zeros(n, torch.uint8)], [t.view(_HELD) for t in zeros(n, torch.uint8)],
                         zeros(blocks, F32), zeros(blocks, F32))
        m, v, m_scale, v_scale = state
        self.m, self.v = list(m), list(v)
        held = F32 if bits == 32 else _HELD
        if (m_scale is None) != (bits == 32) or (v_scale is None) != (bits == 32):
            bad("state: scales for 8 bits, and only there")
        lists = [self.m, self.v]
        self.m_scale = self.v_scale = None
        if bits == 8:
            self.m_scale, self.v_scale = list(m_scale), list(v_scale)
            lists += [self.m_scale, self.v_scale]
        if any(len(x) != len(n) for x in lists):
            bad("state: one tensor of each kind per weight")
        at = []
        for x, sizes, dtype in zip(lists, (n, n, blocks, blocks), (held, held, F32, F32)):
            for t, k in zip(x, sizes):
                if t.numel() != k or t.dtype is not dtype or t.get_device() != self.index or not t.is_contiguous():
                    bad(f"state: contiguous {dtype} tensors of {k} values on cuda:{self.index}")
            at.append([t.data_ptr() for t in x])
        if bits == 32:
            at += [[0] * len(n)] * 2
        # (its memory stays the optimizer's whatever becomes of the tensors: a step writes there)
        self._state = [t.untyped_storage() for x in lists for t in x]
        self._n = len(n)
        self._warned = False
        self._t = np.zeros(self._n, _COLUMNS)
        for name, x in zip(("m", "v", "m_scale", "v_scale", "n"), (*at, n)):
            self._t[name] = x
        self._place()
        if self.index not in _ready():
            prepare(self.device)

    def _place(self) -> None:
        """Notes where weights and copies are, once they are what the step takes."""
        if len(self.params) != self._n or len(self.copies or self.params) != self._n:
            bad("params, copies: one tensor per weight")
        at = []
        for x, dtype, what in ((self.params, self.dtype, "params"), (self.copies or (), self.copy_dtype, "copies")):
            for t, shape in zip(x, self._shapes):
                at.append(dense(t, shape, dtype, self.index, what))
                if not at[-1] and t.numel():
                    bad(f"{what}: tensors with memory of their own")
        _apart([x for x in (self.params, self.copies, self.m, self.v, self.m_scale, self.v_scale) if x])
        self._t["p"] = at[:self._n]
        self._t["copy"] = at[self._n:] if self.copies else 0
        self._at = at

    def _follow(self) -> None:
        """Weights and copies may have other memory at each step (`p.data = ...`, a module moved or flattened)."""
        if list(map(_POINTER, [*self.params, *self.copies] if self.copies else self.params)) != self._at:
            self._place()

    def step(self, grads: Sequence[Optional[torch.Tensor]], hp, *, grad_scale: Optional[torch.Tensor] = None,
             seed=None) -> None:
        """One step on the gradients (f32, f16 or bf16, all of one type, of the weights' shapes; None: the weight and
        its moments stay). hp: the row of AdamW.hp, as an f32 [7] tensor on the GPU or as numbers; grad_scale: an f32
        tensor of one value on the GPU that every gradient is multiplied by; seed: 8-bit moments rounded at random, a
        number or an i64 tensor of one value on the GPU, another for each step (the step's own number does; without one
        they are rounded to nearest, which an optimizer's first such step warns of). A step that is captured into a CUDA
        graph takes both as tensors."""
        if len(grads) != self._n:
            bad("grads: one per weight")
        self._follow()
        numbers = not isinstance(hp, torch.Tensor) or \
            self.bits == 8 and seed is not None and not isinstance(seed, torch.Tensor)
        if numbers and torch.cuda.is_current_stream_capturing():
            bad("a captured step takes hp and seed as tensors on the GPU (numbers would stay those of the capture)")
        if not isinstance(hp, torch.Tensor):
            hp = torch.tensor([float(x) for x in hp], dtype=F32).to(self.device)
        hp_at = dense(hp, (7,), F32, self.index, "hp")
        scale_at = None
        if grad_scale is not None:
            if grad_scale.numel() != 1 or grad_scale.dtype is not F32 or grad_scale.get_device() != self.index:
                bad(f"grad_scale: one f32 value on cuda:{self.index}")
            scale_at = grad_scale.data_ptr()
        seed_at = None
        if seed is not None:
            if not isinstance(seed, torch.Tensor):
                seed = torch.full((1,), int(seed), dtype=I64, device=self.device)
            if seed.numel() != 1 or seed.dtype is not I64 or seed.get_device() != self.index:
                bad(f"seed: a number, or one i64 value on cuda:{self.index}")
            if self.bits == 8:
                seed_at = seed.data_ptr()
        grads, shapes, t = list(grads), self._shapes, self._t
        # what autograd may have saved: values that a forward reads, whether they require a gradient or not
        lists = [x for x in (self.params, self.copies, *((self.m, self.v) if self.bits == 32 else ())) if x]
        if any(g is None for g in grads):
            on = [i for i, g in enumerate(grads) if g is not None]
            if not on:
                return
            grads, shapes, t = [grads[i] for i in on], [shapes[i] for i in on], t[on]
            lists = [[x[i] for i in on] for x in lists]
        dtype = grads[0].dtype
        if dtype not in ROW_TYPE:
            bad("grads: f32, f16 or bf16")
        t["g"] = _pointers(grads, shapes, dtype, self.index, "grads")
        if seed is None and self.bits == 8 and not self._warned:
            self._warned = True
            warnings.warn("toy_b200: 8-bit moments rounded to nearest stop following the gradients after some steps; "
                          "train with MultiAdamW.step(..., seed=)", stacklevel=2)
        a = AdamwMultiArgs(t.ctypes.data, len(t), ROW_TYPE[self.dtype], ROW_TYPE[dtype], ROW_TYPE[self.copy_dtype],
                           self.bits, hp_at, scale_at, seed_at)
        call(self.index, "tb2_adamw_multi", a)
        for x in lists:
            _note(x)

    def _values(self, ms, vs, put: int) -> None:
        if len(ms) != self._n or len(vs) != self._n:
            bad("moments: one tensor of each kind per weight")
        x = self._t.copy()
        x["p"] = _pointers(ms, self._shapes, F32, self.index, "moments")
        x["copy"] = _pointers(vs, self._shapes, F32, self.index, "moments")
        call(self.index, "tb2_adamw_moments", x.ctypes.data, self._n, put)

    def _whole(self, ms, vs) -> None:
        """Refuses lists that are not a tensor of its size for every weight."""
        for x in (ms, vs):
            if [t.numel() for t in x] != [s.numel() for s in self._shapes]:
                bad("moments: one tensor of each kind per weight, of its size")

    def moments(self, *, out: Optional[tuple] = None) -> tuple:
        """(m, v): the values of the moments, lists of f32 tensors of the weights' shapes (out: such lists to fill; in
        32 bits without out the state itself)."""
        if self.bits == 32:
            if out is None:
                return ([t.view(s) for t, s in zip(self.m, self._shapes)],
                        [t.view(s) for t, s in zip(self.v, self._shapes)])
            self._whole(*out)
            for to, x in zip(out, (self.m, self.v)):
                for a, b in zip(to, x):
                    a.copy_(b.view(a.shape))
            return out
        if out is None:
            out = tuple([torch.empty(s, device=self.device, dtype=F32) for s in self._shapes] for _ in "mv")
        self._values(out[0], out[1], 0)
        for x in out:
            _note(x)
        return out

    def set_moments(self, ms: Sequence[torch.Tensor], vs: Sequence[torch.Tensor]) -> None:
        """The moments set to these values (f32, of the weights' shapes), rounded to the state's bits."""
        if self.bits == 32:
            ms, vs = list(ms), list(vs)
            self._whole(ms, vs)
            for to, x in zip((self.m, self.v), (ms, vs)):
                for a, b in zip(to, x):
                    a.copy_(b.reshape(a.shape))
            return
        self._values(list(ms), list(vs), 1)


def _ready() -> set:
    from . import _rows
    return _rows._prepared
