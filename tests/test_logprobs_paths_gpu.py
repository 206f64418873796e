"""The framework's own paths that end in log probabilities: the decoders' (the
logits stay on the GPU) against their downloaded logits, greedy continuations
against the largest logit, and the training engine's against its loss and its
logits."""
import ctypes as C

import numpy as np
import pytest

from oracle import oracle as O

pytestmark = pytest.mark.gpu


def engine(seed=5):
    from toy_b200 import FromScratch, LlamaConfig, RecipeOptions
    rec = FromScratch()
    rec.realize(LlamaConfig(512, 128, 4, 2, 32, 256, 2, 1e4, 1e-5), RecipeOptions(t_seq=64, t_batch=2, seed=seed))
    return rec


def expected(logits, tokens, scale):
    z = logits.astype(np.float64) * scale
    lp = z - z.max(-1, keepdims=True)
    lp -= np.log(np.exp(lp).sum(-1, keepdims=True))
    t = np.asarray(tokens)
    return lp, np.where(t < 0, 0.0, lp[np.arange(len(t)), np.maximum(t, 0)]), -(np.exp(lp) * lp).sum(-1)


# logits of a few units: scores and sums of 512 terms in f32, 2^-24 times some hundred roundings
TOL = 2e-5


@pytest.mark.parametrize("paged", [False, True])
def test_decoders(cuda, paged):
    from toy_b200.decode import KVDecoder, PagedKVDecoder
    eng = engine().fs_cache
    d = PagedKVDecoder(eng, 40, 3, 30, 8, "f32") if paged else KVDecoder(eng, 40, 3)
    with pytest.raises(RuntimeError):
        d.logprobs(top=1)                       # no step yet
    ids = O.token_ids(3, 3 * 5, 512).reshape(5, 3)
    for i in range(5):
        args = (ids[i],) if paged else (ids[i], np.full(3, i))
        logits = d.decode_step(*args)
    tokens = [7, -1, 511]
    got = d.logprobs(tokens, scale=0.75, entropy=True, top=9)
    lp, want, ent = expected(logits, tokens, 0.75)
    order = np.argsort(-logits, axis=-1, kind="stable")[:, :9]
    assert np.array_equal(got.top_ids, order)
    assert np.abs(got.logprob - want).max() <= TOL and np.abs(got.entropy - ent).max() <= TOL
    assert np.abs(got.top_logprobs - np.take_along_axis(lp, order, -1)).max() <= TOL
    only = d.logprobs()
    assert (only.logprob == 0).all() and only.entropy is None and only.top_ids is None
    again = d.decode_step(*((ids[0],) if paged else (ids[0], np.full(3, 5))), logits=False)
    assert again is None and np.abs(d.logprobs(entropy=True).entropy - ent).max() > 0
    with pytest.raises(ValueError):
        d.logprobs([0, 512, 0])
    with pytest.raises(ValueError):
        d.logprobs(top=33)
    d.reset()
    with pytest.raises(RuntimeError):
        d.logprobs(top=1)
    d.close()


@pytest.mark.parametrize("paged", [False, True])
def test_greedy_continuations(cuda, paged):
    """generate picks the largest logit on the GPU: the same tokens as from downloaded logits."""
    from toy_b200.decode import KVDecoder, PagedKVDecoder
    eng = engine(8).fs_cache
    prompt = O.token_ids(9, 2 * 6, 512).reshape(2, 6)
    d = PagedKVDecoder(eng, 40, 2, 30, 8, "f32") if paged else KVDecoder(eng, 40, 2)
    got = np.asarray(d.generate(prompt.tolist() if paged else prompt, 10))
    d.reset()
    pos, feed, out = 0, prompt[:, 0], []
    while len(out) < 10:
        logits = d.decode_step(feed) if paged else d.decode_step(feed, np.full(2, pos))
        pos += 1
        if pos >= 6:
            out.append(np.argmax(logits, -1))
            feed = out[-1]
        else:
            feed = prompt[:, pos]
    assert np.array_equal(got, np.stack(out, 1))
    d.close()


def test_scoring_between_the_steps_of_a_qlora(cuda):
    """The steps around it give the bits they give without (the forward's work on the second stream included)."""
    from toy_b200 import LlamaConfig, LoRA, LoraOptions, RecipeOptions

    def run(score):
        rec = LoRA()
        rec.realize(LlamaConfig(512, 128, 4, 2, 32, 256, 3, 1e4, 1e-5), 8, RecipeOptions(t_seq=64, t_batch=2, seed=2),
                    LoraOptions(rank=8, targets=("q", "v")))
        eng, out = rec.lora_cache, []
        for step in range(1, 5):
            ids = O.token_ids(step, 128, 512)
            args = (ids, O.positions(64, 2), O.next_token_labels(ids, 64, 2, 512))
            if score:
                eng.score(O.token_ids(90 + step, 128, 512), args[1], np.full(128, step))
            out.append(rec.step(*args, O.hp_lora(1e-3, step), step == 1))
        return out, eng.param("blk.2.attn_q.lora_b")

    (a, pa), (b, pb) = run(False), run(True)
    assert a == b and np.array_equal(pa, pb)


def test_training_engine(cuda):
    """A batch's log probabilities: of the labels, the mean of which is the loss; of others, from the same logits."""
    from toy_b200._lib import lib
    rec = engine(11)
    eng, n, V = rec.fs_cache, 128, 512
    with pytest.raises(RuntimeError):
        eng.token_logprobs(np.zeros(n))         # no forward yet
    ids = O.token_ids(4, n, V)
    pos, lab = O.positions(64, 2), O.next_token_labels(ids, 64, 2, V)
    lp, ent = eng.score(ids, pos, lab, entropy=True)
    logits = np.empty(n * V, np.float32)
    assert lib().tb2_debug_activation(eng.sess, 10, 0, logits.ctypes.data_as(C.POINTER(C.c_float)), n * V) == n * V
    _, want, want_ent = expected(logits.reshape(n, V), lab, 1.0)
    assert np.abs(lp - want).max() <= TOL and np.abs(ent - want_ent).max() <= TOL
    before = {k: eng.param(k) for k in eng.param_names()}
    loss = rec.step(ids, pos, lab, O.hp_lora(1e-3, 1), True)
    live = lab >= 0
    assert abs(loss - -lp[live].sum() / n) <= 1e-4 * loss
    # a step was made with the same logits; scoring itself changes nothing
    assert np.abs(eng.token_logprobs(lab) - want).max() <= TOL
    assert any(not np.array_equal(before[k], eng.param(k)) for k in before)
    after = {k: eng.param(k) for k in before}
    other = np.where(np.arange(n) % 3 == 0, -1, (lab + 7) % V)
    eng.score(ids, pos, other, scale=1.5)
    assert all(np.array_equal(after[k], eng.param(k)) for k in after)
    with pytest.raises(ValueError):
        eng.token_logprobs(np.full(n, V))
    with pytest.raises(ValueError):
        eng.token_logprobs(np.zeros(n - 1))
