"""GPU tests of how exact attention over pages is: queries at the edge of their type, softmax weights that nearly cancel."""

import pytest
import torch

from mlkit_b200 import kernels
from tests.paged_reference import STEP, rotated

pytestmark = pytest.mark.gpu
HALF, BRAIN = torch.float16, torch.bfloat16
THETA = 500000.0


def test_rotated_queries_beyond_the_range_of_their_type():
    """Two halves of 60000 turn to up to 84853, which fp16 does not have; scores, weights and outputs are finite all the same.

    The keys are zero but for the dimensions 5 and 5 + width / 2, up to 2^-13: a score is the sum of two exact products
    of about 1, off by some steps of 2^-23 of them and by the rotation's own error (below 2^-21)."""
    width, n = 64, 40
    keys = torch.zeros(1, 1, 48, width, dtype=HALF)
    keys[0, 0, :n, 5] = 2.0 ** -13
    keys[0, 0, :n, 5 + width // 2] = torch.linspace(-1, 1, n).half() * 2.0 ** -13
    values = torch.randn(1, 1, 48, width, generator=torch.Generator().manual_seed(0)).half()
    qkv = torch.zeros(1, 3 * width, dtype=HALF)
    qkv[0, :width] = 60000.0
    weights, out = torch.zeros(1, 1, 48, device="cuda"), torch.empty(1, 1, width, dtype=HALF, device="cuda")
    held = torch.tensor([n], dtype=torch.int32).cuda()
    # position 1: the frequency of dimension 5 turns by 0.13, to 51700 and 67300
    kernels.paged_rope_attention_decode(qkv.cuda(), torch.ones_like(held), held, keys.cuda(), values.cuda(), torch.zeros(1, 1, dtype=torch.int32).cuda(),
                                        out, q_heads=1, kv_heads=1, head_dim=width, theta=THETA, weights=weights)
    query = rotated(qkv[:, :width], 1, THETA)
    assert query.abs().max() > 65504
    keys[0, 0, n] = 0                                            # the new token's key and value are zero
    values[0, 0, n] = 0
    scores = (keys[0, 0, :n + 1].double() @ query[0]) * width ** -0.5
    share = torch.softmax(scores, 0)
    slack = 2 * 4 * 2.0 ** -21 + 2.0 ** -20                      # scores are below 4
    assert scores.abs().max() < 4
    assert ((weights.cpu().double()[0, 0, :n + 1] - share).abs() <= slack * share).all()
    expected, mass = share @ values[0, 0, :n + 1].double(), share @ values[0, 0, :n + 1].double().abs()
    assert ((out.cpu().double()[0, 0] - expected).abs() <= STEP[HALF] * expected.abs() + (2 * slack + 2.0 ** -22) * mass + 2.0 ** -25).all()
