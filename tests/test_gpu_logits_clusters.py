"""GPU test of how many CTAs a row of logits gets: no more than the GPU holds at once."""

import pytest
import torch

from mlkit_b200 import kernels
from tests.test_gpu_logits_buffers import given, quickest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("more", [17, 36, 76])
def test_fewer_rows_take_no_longer(more):
    """Where a row's cluster is too wide for all rows to run at once, some wait for a second turn: a third more time."""
    calls = []
    for rows in (more - 2, more - 1, more):
        logits, tokens, arguments = given(rows, 50257, 900, [900] * rows, torch.float32, biases=7)
        out = torch.empty_like(logits)
        calls.append(lambda logits=logits, tokens=tokens, out=out, arguments=arguments: kernels.adjust_logits(logits, tokens=tokens, out=out, **arguments))
    times = quickest(calls, 25)
    print(more, times)
    assert times[0] < 1.15 * times[2] and times[1] < 1.15 * times[2], times
