"""GPU tests of how exact attention over pages is: queries at the edge of their type, softmax weights that nearly cancel."""

import pytest
import torch

from mlkit_b200 import kernels
from tests.paged_accuracy import cancelling_case, rotary_case
from tests.paged_reference import STEP, rotated, slots_of

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


def paged(data, page, seed=0):
    """[rows, heads, n, ...] in pages of a pool in random order, with their tables."""
    rows, heads, n = data.shape[:3]
    columns = -(-n // page)
    order = torch.randperm(rows * columns, generator=torch.Generator().manual_seed(seed)).view(rows, columns)
    padded = torch.zeros(rows, heads, columns * page, *data.shape[3:], dtype=data.dtype)
    padded[:, :, :n] = data
    pool = torch.zeros(rows * columns, heads, page, *data.shape[3:], dtype=data.dtype)
    pool[order] = padded.unflatten(2, (columns, page)).transpose(1, 2)
    return pool, order.int()


@pytest.mark.parametrize("dtype", [HALF, BRAIN])
@pytest.mark.parametrize("width,n", [(64, 90), (128, 90), (192, 31), (256, 90), (128, 5000)])
def test_accumulated_weights_of_large_rotated_queries(dtype, width, n):
    """A query in one 16-bit part fails this by 240 times and more, a bf16 one in two by 2.7 times and more."""
    queries, keys, values, positions, shares, slack = rotary_case(dtype, width=width, n=n)
    rows, heads = queries.shape[:2]
    (k_pages, tables), (v_pages, _) = paged(torch.nn.functional.pad(keys, (0, 0, 0, 1)), 16), paged(torch.nn.functional.pad(values, (0, 0, 0, 1)), 16)
    qkv = torch.cat((queries, torch.zeros(rows, 2 * heads, width, dtype=dtype)), 1).flatten(1)
    weights, out = torch.zeros(k_pages.shape[:3], device="cuda"), torch.empty(rows, heads, width, dtype=dtype, device="cuda")
    kernels.paged_rope_attention_decode(qkv.cuda(), positions.cuda(), torch.full((rows,), n, dtype=torch.int32).cuda(), k_pages.cuda(), v_pages.cuda(),
                                        tables.cuda(), out, q_heads=heads, kv_heads=heads, head_dim=width, theta=THETA, scale=1.0, weights=weights)
    expected = shares()
    got = torch.stack([slots_of(weights.cpu(), tables[row], n + 1) for row in range(rows)]).double()
    off = (got - expected).abs() / (slack * expected)
    assert (off <= 1).all(), float(off.max())


@pytest.mark.parametrize("dtype", [HALF, BRAIN])
@pytest.mark.parametrize("width,n", [(64, 24), (128, 24), (192, 7), (256, 24), (64, 4000)])
def test_softmax_weights_that_nearly_cancel(dtype, width, n):
    """Weights in one 16-bit part fail this by 30 times and more at 24 slots."""
    queries, keys, values, outputs, bound = cancelling_case(dtype, width=width, n=n)
    (k_pages, tables), (v_pages, _) = paged(keys[None], 16), paged(values[None], 16)
    out = torch.empty(1, *queries.shape, dtype=dtype, device="cuda")
    kernels.paged_attention_decode(queries[None].cuda(), torch.tensor([n], dtype=torch.int32).cuda(), k_pages.cuda(), v_pages.cuda(), tables.cuda(), out,
                                   scale=1.0)
    off = (out.cpu().double()[0] - outputs()).abs() / bound
    assert (off <= 1).all(), float(off.max())
