"""Greedy continuations refuse prompts that there is nothing to continue from."""
import numpy as np
import pytest


@pytest.mark.parametrize("prompt", [np.zeros((2, 0)), [[], []]])
def test_an_empty_prompt(prompt):
    """A decoder has no logits to begin with, and those of an earlier step are of another sequence."""
    from toy_b200.decode import KVDecoder, StepLogprobs
    d = KVDecoder.__new__(KVDecoder)          # (no engine: the two calls that reach it are stood in for)
    d.n_seq, d.steps = 2, []
    d.decode_step = lambda tokens, positions, logits=True: d.steps.append(list(positions))
    d.logprobs = lambda **kw: StepLogprobs(None, None, np.array([[3], [4]]), None)     # an earlier step's
    with pytest.raises(ValueError):
        d.generate(prompt, 4)
    assert not d.steps
    assert d.generate(np.ones((2, 1)), 2).tolist() == [[3, 3], [4, 4]]
    assert [list(map(int, p)) for p in d.steps] == [[0, 0], [1, 1], [2, 2]]
