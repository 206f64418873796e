"""Log probabilities of given tokens, entropy and the most likely alternatives
of rows of logits, with the gradient: tb2_logprobs and tb2_logprobs_grad
(include/toy_b200.h) over torch CUDA tensors.

`token_logprobs` is differentiable in the logits (its logprob, entropy and
top_logprobs have gradients); `token_logprobs_grad` is the gradient as a call of
its own, for programs that do without autograd or want it in the logits' own
memory. Both run on torch's current stream of the logits' device, synchronise
nothing, and can be captured into a CUDA graph once `prepare` has run. Arguments
that do not fit are refused with ValueError before anything runs; tokens outside
the vocabulary are reported on the device (`tb2_device_error` in the header).
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from ._lib import LogprobsArgs, LogprobsGradArgs
from ._rows import F32, I64, ROW_TYPE, bad, call, dense, no_captured_leaf, no_tangent, prepare, rows, written

__all__ = ["TokenLogprobs", "prepare", "token_logprobs", "token_logprobs_grad"]
MAX_TOP = 32


class TokenLogprobs(NamedTuple):
    """What `token_logprobs` computed: see tb2_logprobs."""
    logprob: torch.Tensor                   # [n] f32: ln p of the row's token, 0 where the token is negative
    entropy: Optional[torch.Tensor]         # [n] f32
    top_ids: Optional[torch.Tensor]         # [n, top] i64, the largest logit first, equal ones by the lower index
    top_logprobs: Optional[torch.Tensor]    # [n, top] f32
    stats: torch.Tensor                     # [n, 2] f32: m = max(row) and ln sum exp(scale * (row - m))


def _logits(x: torch.Tensor, tokens: torch.Tensor, scale: float, top: int) -> tuple:
    """(rows, vocabulary, device, row stride) of checked logits."""
    dev, dtype = x.get_device(), x.dtype
    if dev < 0 or x.dim() != 2 or dtype not in ROW_TYPE:
        bad("logits: f32, f16 or bf16 [n, vocab] on a GPU")
    n, vocab = x.shape
    if vocab < 1 or n >= 2**31 or vocab >= 2**31:
        bad("logits: one word or more, rows and words below 2^31")
    if not 0 <= top <= MAX_TOP or top > vocab:
        bad(f"top is 0 to {MAX_TOP}, and no more than the vocabulary")
    if not 2.0**-126 <= scale <= 2.0**126:
        bad("scale is positive, and neither it nor its inverse past f32's range")
    dense(tokens, (n,), I64, dev, "tokens")
    return n, vocab, dev, rows(x, n, vocab, dtype, dev, "logits")


def _forward(x, tokens, scale, entropy, top) -> TokenLogprobs:
    n, vocab, dev, ld = _logits(x, tokens, scale, top)
    lp, stats = x.new_empty(n, dtype=F32), x.new_empty((n, 2), dtype=F32)
    ent = x.new_empty(n, dtype=F32) if entropy else None
    ids = top_lp = None
    if top:
        ids, top_lp = x.new_empty((n, top), dtype=I64), x.new_empty((n, top), dtype=F32)
    if n:
        a = LogprobsArgs(n, vocab, ROW_TYPE[x.dtype], x.data_ptr(), ld, scale, tokens.data_ptr(), lp.data_ptr(),
                         stats.data_ptr(), ent.data_ptr() if entropy else None, top, ids.data_ptr() if top else None,
                         top_lp.data_ptr() if top else None)
        call(dev, "tb2_logprobs", a)
    return TokenLogprobs(lp, ent, ids, top_lp, stats)


class _Score(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, scale, entropy, top):
        r = _forward(logits, tokens, scale, entropy, top)
        ctx.mark_non_differentiable(*[t for t in (r.stats, r.top_ids) if t is not None])
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(logits, tokens, r.stats, r.entropy, r.top_ids)
        ctx.scale = scale
        return tuple(r)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_logprob, g_entropy, _ids, g_top, _stats):
        logits, tokens, stats, ent, ids = ctx.saved_tensors
        if g_logprob is None and g_entropy is None and g_top is None:
            return None, None, None, None, None
        r = TokenLogprobs(None, ent, ids, None, stats)
        g = [None if t is None else t.to(F32).contiguous() for t in (g_logprob, g_entropy, g_top)]
        d = token_logprobs_grad(logits.detach(), tokens, r, g[0], grad_entropy=g[1], grad_top=g[2], scale=ctx.scale)
        return d, None, None, None, None


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, scale: float = 1.0, entropy: bool = False,
                   top: int = 0) -> TokenLogprobs:
    """ln p of tokens [n] (i64; negative: none, 0) under softmax(scale * logits [n, vocab]), with the rows' entropy and
    the `top` (at most 32) most likely words where asked for. Logits are f32, f16 or bf16; -inf is a word of
    probability 0. Differentiable in the logits."""
    no_tangent(logits)
    if logits.requires_grad and torch.is_grad_enabled():
        no_captured_leaf(logits)
        return TokenLogprobs(*_Score.apply(logits, tokens, scale, entropy, top))
    return _forward(logits, tokens, scale, entropy, top)


def token_logprobs_grad(logits: torch.Tensor, tokens: torch.Tensor, result: TokenLogprobs,
                        grad_logprob: Optional[torch.Tensor] = None, *, grad_entropy: Optional[torch.Tensor] = None,
                        grad_top: Optional[torch.Tensor] = None, scale: float = 1.0,
                        out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The logits' gradient, [n, vocab] of their type, from the gradients of logprob [n], entropy [n] and top_logprobs
    [n, top] (f32; None: none). `result` is token_logprobs's of the same logits, tokens and scale; out may be the logits
    themselves."""
    no_tangent(logits, grad_logprob, grad_entropy, grad_top, out)
    top = grad_top.shape[1] if grad_top is not None and grad_top.dim() == 2 else 0
    n, vocab, dev, ld = _logits(logits, tokens, scale, top)
    if torch.is_grad_enabled() and (logits.requires_grad or out is not None and out.requires_grad):
        bad("no gradient passes through token_logprobs_grad (use it under torch.no_grad())")
    g = [None if t is None else dense(t, shape, F32, dev, what) for t, shape, what in (
        (grad_logprob, (n,), "grad_logprob"), (grad_entropy, (n,), "grad_entropy"), (grad_top, (n, top), "grad_top"))]
    if grad_entropy is not None and result.entropy is None or grad_top is not None and result.top_ids is None:
        bad("result: with the entropy and the alternatives that have a gradient")
    ent = dense(result.entropy, (n,), F32, dev, "result.entropy") if grad_entropy is not None else None
    ids = dense(result.top_ids, (n, top), I64, dev, "result.top_ids") if top else None
    fresh = out is None
    if fresh:
        out = torch.empty((n, vocab), device=logits.device, dtype=logits.dtype)
    ldd = rows(out, n, vocab, logits.dtype, dev, "out")
    if n:
        a = LogprobsGradArgs(n, vocab, ROW_TYPE[logits.dtype], logits.data_ptr(), ld, scale, tokens.data_ptr(),
                             dense(result.stats, (n, 2), F32, dev, "result.stats"), ent, g[0], g[1], top,
                             g[2] if top else None, ids, out.data_ptr(), ldd)
        call(dev, "tb2_logprobs_grad", a)
    if not fresh:
        written(out)
    return out
