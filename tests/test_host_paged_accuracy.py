"""The bounds of the accuracy tests reject what they are there to reject: fewer 16-bit parts, emulated on the CPU."""

import pytest
import torch

from tests.paged_accuracy import cancelling_case, rotary_case

HALF, BRAIN = torch.float16, torch.bfloat16


@pytest.mark.parametrize("dtype,enough", [(HALF, 2), (BRAIN, 3)])
@pytest.mark.parametrize("width", [64, 128, 256])
def test_parts_of_a_rotated_query(dtype, enough, width):
    _, _, _, _, shares, slack = rotary_case(dtype, width=width)
    off = lambda count: float(((shares(count) - shares()).abs() / (slack * shares())).max())
    assert off(enough) < 0.25 and off(enough - 1) > 2


@pytest.mark.parametrize("dtype", [HALF, BRAIN])
@pytest.mark.parametrize("width", [64, 128, 256])
def test_parts_of_a_softmax_weight(dtype, width):
    _, _, _, outputs, bound = cancelling_case(dtype, width=width)
    off = lambda count: float(((outputs(count) - outputs()).abs() / bound).max())
    assert off(2) < 0.5 and off(1) > 20
