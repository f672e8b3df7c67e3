"""GPU test of a capture that fails on the host: cache and rules are as they were, and the next capture works."""

import pytest
import torch

import mlkit_b200 as mk
from mlkit_b200 import tp

pytestmark = pytest.mark.gpu
CONFIG = tp.DecoderConfig(layers=2, hidden=256, q_heads=4, kv_heads=2, head_dim=128, intermediate=512, vocab=512)


@pytest.mark.parametrize("failing", [1, 2, 3])
def test_a_capture_that_fails(monkeypatch, failing):
    """The first and the second step warm up, the third is captured; each raises once, after its launches."""
    model = tp.TensorParallelDecoder.synthetic(CONFIG, max_batch=2, capacity=64, page=8)
    rules = mk.LogitRules(rows=2, capacity=16)
    rules.begin(0, [5, 6, 7])
    model.cache.open(0)
    step, steps = model.step, []

    def fails(*arguments):
        steps.append(1)
        result = step(*arguments)
        if len(steps) == failing:
            raise RuntimeError("a step that fails")
        return result

    monkeypatch.setattr(model, "step", fails)
    with pytest.raises(RuntimeError, match="a step that fails"):
        model.capture(2, greedy=True, rules=rules)
    monkeypatch.setattr(model, "step", step)
    assert rules.lengths.tolist() == [3, 0] and model.cache.lengths.tolist() == model.cache.held == [0, -1]
    run = model.capture(2, greedy=True, rules=rules)
    picked = run.replay().tolist()
    assert rules.lengths.tolist() == [4, 1] and rules.tokens[0, 3] == picked[0] and model.cache.lengths.tolist() == [1, -1]
