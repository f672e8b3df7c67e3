"""GPU test of how many CTAs a row of logits gets: no more than the GPU holds at once."""

import pytest
import torch

from mlkit_b200 import kernels
from tests.test_gpu_logits_buffers import given, quickest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("more", [17, 36, 76])
def test_fewer_rows_take_no_longer(more):
    """Where a row's cluster is too wide for all rows to run at once, some wait for a second turn: a third more time for 15 and
    16 rows than for 17."""
    calls = []
    for rows in (more - 2, more - 1, more):
        logits, tokens, arguments = given(rows, 50257, 900, [900] * rows, torch.float32, biases=7)
        out = torch.empty_like(logits)
        calls.append(lambda logits=logits, tokens=tokens, out=out, arguments=arguments: kernels.adjust_logits(logits, tokens=tokens, out=out, **arguments))
    times = quickest(calls, 25)
    print(more, times)
    assert times[0] < 1.25 * times[2] and times[1] < 1.25 * times[2], times


def test_sizes_that_are_new_within_a_capture():
    """How many clusters fit is asked while the stream is captured."""
    logits, tokens, arguments = given(11, 23456, 70, [70] * 11, torch.float32)
    out, expected = torch.empty_like(logits), torch.empty_like(logits)
    kernels.adjust_logits(logits[:3], tokens=tokens[:3], out=expected[:3], **{name: value[:3] for name, value in arguments.items()})
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        kernels.adjust_logits(logits, tokens=tokens, out=out, **arguments)
    graph.replay()
    kernels.adjust_logits(logits, tokens=tokens, out=expected, **arguments)
    assert torch.equal(out, expected)
