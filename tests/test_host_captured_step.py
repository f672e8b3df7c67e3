"""What a captured step leaves behind when its warm-up fails, on the CPU with stubs for the streams."""

from contextlib import nullcontext

import pytest
import torch

import mlkit_b200 as mk
from mlkit_b200 import tp


class Stream:
    waits = []

    def __init__(self, name):
        self.name = name

    def wait_stream(self, other):
        self.waits.append((self.name, other.name))


class Model:
    """A decoder whose second step fails, after both have observed a token."""

    device = torch.device("cpu")

    def __init__(self):
        self.cache = mk.PagedCache(rows=2, columns=2, kv_heads=1, head_dim=64, layers=0, device="cpu")
        self.steps = 0

    def step(self, tokens, positions, greedy=False, rules=None):
        self.steps += 1
        rules.observe(torch.tensor([40 + self.steps, 50 + self.steps]))
        if self.steps == 2:
            raise RuntimeError("a step that fails")


def test_a_capture_that_fails_leaves_rules_and_cache_as_they_were(monkeypatch):
    for name, value in (("Stream", lambda device=None: Stream("side")), ("current_stream", lambda device=None: Stream("current")),
                        ("stream", lambda stream: nullcontext()), ("synchronize", lambda device=None: None)):
        monkeypatch.setattr(torch.cuda, name, value)
    Stream.waits.clear()
    model, rules = Model(), mk.LogitRules(rows=3, capacity=8, device="cpu")
    model.cache.open(1)
    rules.begin(0, [5, 6, 7])
    rules.begin(1, range(8))                    # a full history
    with pytest.raises(RuntimeError, match="a step that fails"):
        tp.CapturedStep(model, 2, True, rules)
    assert rules.lengths.tolist() == [3, 8, 0]
    assert rules.tokens[0, :3].tolist() == [5, 6, 7] and rules.tokens[1].tolist() == list(range(8))
    assert model.cache.lengths.tolist() == model.cache.held == [-1, 0]
    assert Stream.waits == [("side", "current"), ("current", "side")]      # what is taken back comes behind the steps
