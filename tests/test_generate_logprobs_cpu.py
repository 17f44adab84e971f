"""What LLMEngine.generate_logprobs refuses before it takes pages for a request,
on an engine of which only what it asks is there."""

from types import SimpleNamespace

import numpy as np
import pytest

from foundry_b200.runner.engine import LLMEngine


def _engine(tp=None, vocab=4096):
    calls = []

    def generate(prompts, max_new_tokens, top):
        calls.append(top)
        return [SimpleNamespace(output=[1], logprobs=[(0.0, 0.0, [])]) for _ in prompts]

    return SimpleNamespace(tp=tp, weights=SimpleNamespace(vocab_l=vocab), _generate=generate), calls


def test_a_sharded_vocabulary_is_refused():
    eng, calls = _engine(tp=object())
    with pytest.raises(ValueError, match="whole vocabulary"):
        LLMEngine.generate_logprobs(eng, [[1]], 2, top=3)
    assert not calls


@pytest.mark.parametrize("top", [-1, 33, 2.0, 2.5, "2", None])
def test_top_is_a_whole_number_in_range(top):
    """A float got as far as the first prefill, whose pages were then not given back."""
    eng, calls = _engine()
    with pytest.raises(ValueError, match="top must be"):
        LLMEngine.generate_logprobs(eng, [[1]], 2, top=top)
    assert not calls
    for fine in (0, 5, np.int64(32)):
        assert LLMEngine.generate_logprobs(eng, [[1]], 2, top=fine) == ([[1]], [[(0.0, 0.0, [])]])
    assert [type(x) for x in calls] == [int] * 3


def test_top_is_no_more_than_the_vocabulary():
    eng, calls = _engine(vocab=4)
    with pytest.raises(ValueError, match="0 to 4"):
        LLMEngine.generate_logprobs(eng, [[1]], 2, top=5)
    assert not calls
