"""The C entries of the row operators refuse what does not fit before they touch
a GPU (-1, not an exception or an abort), and the Python layers refuse tensors
that are on none; the cases' file keeps to its ranges."""
import ctypes as C
import random

import pytest


def lib():
    from toy_b200 import _lib
    return _lib.lib()


P = 1 << 20          # an address that is never followed: every call below is refused


def test_logprobs_arguments():
    from toy_b200._lib import LogprobsArgs, LogprobsGradArgs
    ok = dict(n_rows=2, vocab=10, row_type=0, logits=P, ld=10, scale=1.0, tokens=P, logprob=P, stats=P, entropy=P,
              top=2, top_ids=P, top_logprobs=P)
    for k, v in (("n_rows", -1), ("vocab", 0), ("vocab", -3), ("row_type", 2), ("row_type", 8), ("logits", None),
                 ("logits", P + 2), ("ld", 9), ("scale", 0.0), ("scale", float("nan")), ("scale", float("inf")),
                 ("scale", -1.0), ("tokens", None), ("tokens", P + 4), ("logprob", None), ("logprob", P + 1),
                 ("stats", None), ("stats", P + 4), ("entropy", P + 2), ("top", -1), ("top", 33), ("top", 11),
                 ("top_ids", None), ("top_ids", P + 4), ("top_logprobs", None), ("top_logprobs", P + 3)):
        assert lib().tb2_logprobs(C.byref(LogprobsArgs(**{**ok, k: v})), None) == -1, (k, v)
    assert lib().tb2_logprobs(None, None) == -1
    assert lib().tb2_logprobs(C.byref(LogprobsArgs(**{**ok, "n_rows": 0})), None) == 0
    ok = dict(n_rows=2, vocab=10, row_type=30, logits=P, ld=10, scale=1.0, tokens=P, stats=P, entropy=P, g_logprob=P,
              g_entropy=P, top=2, g_top=P, top_ids=P, d_logits=P, ldd=10)
    for k, v in (("vocab", 0), ("row_type", 1 << 20), ("logits", P + 1), ("ld", 9), ("ldd", 9), ("d_logits", None),
                 ("d_logits", P + 1), ("scale", 0.0), ("tokens", None), ("stats", None), ("entropy", None), ("top", 33),
                 ("g_top", None), ("top_ids", None), ("g_logprob", P + 2), ("g_entropy", P + 1), ("scale", 1e-39),
                 ("scale", 1e38), ("ldd", 11)):      # (the logits' own memory, with another stride)
        assert lib().tb2_logprobs_grad(C.byref(LogprobsGradArgs(**{**ok, k: v})), None) == -1, (k, v)
    assert lib().tb2_logprobs_grad(None, None) == -1


def test_expert_arguments():
    from toy_b200._lib import ExpertRowsArgs, ExpertSortArgs
    ok = dict(ids=P, id_bytes=4, n_slots=8, n_experts=4, offsets=P, order=P, pos=P)
    for k, v in (("ids", None), ("ids", P + 2), ("id_bytes", 2), ("n_slots", -1), ("n_experts", 0), ("n_experts", 1025),
                 ("offsets", None), ("order", None), ("pos", None), ("pos", P + 1)):
        assert lib().tb2_expert_sort(C.byref(ExpertSortArgs(**{**ok, k: v})), None) == -1, (k, v)
    assert lib().tb2_expert_sort(C.byref(ExpertSortArgs(**{**ok, "id_bytes": 8, "ids": P + 4})), None) == -1
    ok = dict(n_tokens=4, n_used=2, d=16, n_rows=8, row_type=0, x=P, ldx=16, xs=P, ldxs=16, pos=P, weights=P,
              residual=P, ldr=16, d_xs=P, ldd=16, d_weights=P, n_sorted=P)
    every = ("tb2_expert_dispatch", "tb2_expert_combine", "tb2_expert_combine_grad")
    for k, v, calls in (("n_tokens", -1, every), ("n_used", 0, every), ("d", 0, every), ("n_rows", -1, every),
                        ("row_type", 8, every), ("x", None, every), ("x", P + 2, every), ("ldx", 15, every),
                        ("xs", None, every), ("ldxs", 15, every), ("pos", None, every), ("pos", P + 2, every),
                        ("weights", P + 2, every[1:]), ("residual", P + 2, every[1:2]), ("ldr", 15, every[1:2]),
                        ("ldd", 15, every[2:]), ("d_xs", P + 1, every[2:]), ("d_weights", P + 1, every[2:]),
                        ("n_sorted", P + 1, (every[0], every[2])), ("n_used", 1 << 30, every),
                        ("ldr", 17, every[1:2]), ("ldd", 17, every[2:])):      # (the same memory, another stride)
        for f in calls:
            assert getattr(lib(), f)(C.byref(ExpertRowsArgs(**{**ok, k: v})), None) == -1, (k, v, f)
    for f in every:
        assert getattr(lib(), f)(None, None) == -1
        assert getattr(lib(), f)(C.byref(ExpertRowsArgs(**{**ok, "n_tokens": 0})), None) == 0


def test_adamw_arguments():
    from toy_b200._lib import AdamwMultiArgs, AdamwTensor
    t_ok = dict(p=P, g=P, m=P, v=P, m_scale=P, v_scale=P, copy=P, n=5)
    a_ok = dict(n_tensors=1, p_type=0, g_type=30, copy_type=30, state_bits=8, hp=P, grad_scale=P)

    def step(t, a):
        x = (AdamwTensor * 1)(AdamwTensor(**t))
        return lib().tb2_adamw_multi(C.byref(AdamwMultiArgs(tensors=C.addressof(x), **a)), None)
    for k, v in (("p", None), ("p", P + 2), ("g", None), ("g", P + 1), ("m", None), ("v", None), ("m_scale", None),
                 ("v_scale", P + 2), ("copy", P + 1), ("n", -1), ("n", 1 << 60)):
        assert step({**t_ok, k: v}, a_ok) == -1, (k, v)
    for k, v in (("n_tensors", -1), ("p_type", 8), ("g_type", 3), ("copy_type", 0), ("state_bits", 16), ("hp", None),
                 ("hp", P + 2), ("grad_scale", P + 1), ("seed", P + 4)):
        assert step(t_ok, {**a_ok, k: v}) == -1, (k, v)
    assert step({**t_ok, "m": P + 2}, {**a_ok, "state_bits": 32}) == -1
    assert lib().tb2_adamw_multi(None, None) == -1
    assert lib().tb2_adamw_multi(C.byref(AdamwMultiArgs(tensors=None, **a_ok)), None) == -1
    assert step({**t_ok, "n": 0, "p": None}, a_ok) == 0              # an empty tensor is passed over
    x = (AdamwTensor * 1)(AdamwTensor(**{**t_ok, "copy": None}))
    assert lib().tb2_adamw_moments(C.addressof(x), 1, 0, None) == -1
    assert lib().tb2_adamw_moments(None, 1, 0, None) == -1 and lib().tb2_adamw_moments(None, 0, 0, None) == 0


def test_tensors_on_no_gpu():
    import torch
    from toy_b200 import experts, logprobs
    from toy_b200.multi_adamw import MultiAdamW
    x, t = torch.zeros((3, 8)), torch.zeros(3, dtype=torch.int64)
    r = experts.Routing(t.int(), t.int(), torch.zeros((3, 1), dtype=torch.int32))
    for bad in (lambda: logprobs.token_logprobs(x, t), lambda: experts.sort(torch.zeros((3, 1), dtype=torch.int32), 2),
                lambda: experts.dispatch(x, r), lambda: experts.combine(x, r), lambda: MultiAdamW([x])):
        with pytest.raises(ValueError):
            bad()


def test_no_session():
    f = (C.c_float * 4)()
    i = (C.c_longlong * 4)()
    assert lib().tb2_kv_logprobs(None, i, 1, 1.0, 0, f, None, None, None) == -2
    assert lib().tb2_llama_logprobs(None, i, 1, 1.0, f, None) == -2


def test_cases_keep_to_their_ranges():
    from perf import more_operators as M
    cases = M.listed()
    assert len({c["name"] for c in cases}) == len(cases)
    most = max(M.work(c)["bytes"] for c in cases)
    r = random.Random(0)
    for _ in range(300):
        assert 0 < M.work(M.draw(r))["bytes"] <= most
