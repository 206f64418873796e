"""The mixture-of-experts step with its slots sorted on the GPU: the captured step
gives the eager one's bits, whatever the routing, and a router that is not a
number makes the loss one too (and nothing else)."""
import numpy as np
import pytest

from oracle import oracle as O

pytestmark = pytest.mark.gpu


def steps(n, graph, router=None, T=96, B=2, E=16, K=4):
    from toy_b200 import LlamaConfig, LoRA, LoraOptions, RecipeOptions
    from toy_b200._lib import lib
    cfg = LlamaConfig(512, 128, 2, 2, 64, 64, 2, 1e4, 1e-5, n_experts=E, n_experts_used=K, qk_norm=2)
    rec = LoRA()
    rec.realize(cfg, 8, RecipeOptions(t_seq=T, t_batch=B, seed=21), LoraOptions(rank=8, targets=("q", "v")))
    eng = rec.lora_cache
    lib().tb2_set_use_graph(eng.sess, 1 if graph else 0)
    if router is not None:
        for blk in range(2):
            name = f"blk.{blk}.ffn_gate_inp.weight"
            eng.set_param(name, router(eng.param(name)))
    losses = []
    for step in range(1, n + 1):
        ids = O.token_ids(step, T * B, 512)
        losses.append(rec.step(ids, O.positions(T, B), O.next_token_labels(ids, T, B, 512), O.hp_lora(1e-3, step),
                               step == 1))
    return losses, eng.param("blk.1.attn_q.lora_b"), eng


@pytest.mark.parametrize("skew", [False, True])
def test_captured_steps_equal_eager_ones(cuda, skew):
    def to_few(w):          # the last experts' logits far ahead: most experts have no slot
        w = np.array(w)
        w[-5:] *= 1e-3
        w[:-5] = w[-5:].mean(axis=0)
        w[-5:] += np.sign(w[-5:]) * 2.0
        return w
    router = to_few if skew else None
    a, pa, _ = steps(4, True, router)
    b, pb, _ = steps(4, False, router)
    assert a == b and np.array_equal(pa, pb)


def test_router_that_is_not_a_number(cuda):
    from toy_b200._lib import lib
    losses, _, eng = steps(3, True, lambda w: np.full_like(w, np.nan))
    assert all(np.isnan(x) for x in losses)
    assert lib().tb2_device_error() == 0
