"""Cases that tell how many 16-bit parts the attention over pages holds a rotated query and a softmax weight in, with bounds
that are close enough for it: few products a score, large scores, values that nearly cancel."""

import torch

from tests.paged_reference import STEP, rotated

THETA = 500000.0
# What two 16-bit parts leave out of a softmax weight, relative: half a step of the rest, which is at most half a step of the whole
# and lies one binade below that at its largest.  fp16: 2^-11 * 2^-12, doubled.
LEFT_OUT = {torch.float16: 2.0 ** -22, torch.bfloat16: 2.0 ** -17}


def parts_of(x, dtype, count):
    """``x`` (64 bits) as the sum of ``count`` values of ``dtype``, each the rounding of what those before left out."""
    total = torch.zeros_like(x)
    for _ in range(count):
        total = total + (x - total).to(dtype).double()
    return total


def rotary_case(dtype, *, rows=4, heads=8, width=128, n=90, size=8.0, seed=0):
    """Large queries against keys with two dimensions that are not zero, so a score is the sum of two products.  The new token's key
    is zero.  ``share`` [rows, heads, n + 1], ``slack`` [rows, heads, 1] of its relative error, and a function of the parts of a query.

    A score's error: the angle in turns is rounded to 2^-26 (2^-23.3 of a radian), sine and cosine come with two steps (2^-23),
    the turn's products and sum with one and a half: below 5 * 2^-24 of (|low| + |high|) |k|.  The products are exact, their sum, the
    scale, the difference to the maximum and to the sum's logarithm are rounded: 8 * 2^-24 of the largest sum |q k|.  A query in
    two fp16 parts leaves 2^-23 of itself out, one in three bf16 parts less: within the same.  A weight is off by both its own
    score's error and the others' (hence twice), by exp2, by the logarithm and the sum: 2^-20."""
    generator = torch.Generator().manual_seed(seed)
    half, at = width // 2, 3
    queries = (torch.randn(rows, heads, width, generator=generator) * size).to(dtype)
    keys = torch.zeros(rows, heads, n, width, dtype=dtype)
    keys[..., at], keys[..., at + half] = (torch.rand(rows, heads, n, generator=generator).sub(0.5).mul(2).to(dtype) for _ in range(2))
    values = torch.randn(rows, heads, n, width, generator=generator).to(dtype)
    positions = torch.randint(0, 5000, (rows,), generator=generator).to(torch.int32)
    turned = torch.stack([rotated(queries[m], int(positions[m]), THETA) for m in range(rows)])
    wide = torch.cat((keys.double(), torch.zeros(rows, heads, 1, width, dtype=torch.float64)), 2)

    def shares(count=None):
        held = turned if count is None else parts_of(turned, dtype, count)
        return torch.softmax(torch.einsum("mhd,mhnd->mhn", held, wide), 2)

    pair = queries[..., at].double().abs() + queries[..., at + half].double().abs()
    reach = pair[..., None] * (keys[..., at].double().abs() + keys[..., at + half].double().abs())
    sums = torch.einsum("mhd,mhnd->mhn", turned.abs(), wide.abs())
    slack = 2 * (5 * 2.0 ** -24 * reach.amax(2, keepdim=True) + 8 * 2.0 ** -24 * sums.amax(2, keepdim=True)) + 2.0 ** -20
    return queries, keys, values, positions, shares, slack


def cancelling_case(dtype, *, heads=8, width=64, n=24, seed=0):
    """One product a score, and values of which the heaviest slot's take back what the others add up to: the output is small
    against the sum of |w v|, so its own rounding hides nothing.  ``(queries, keys, values, outputs, bound)``, the third a
    function of the parts of a softmax weight.

    A score's product is exact; scale, maximum and logarithm cost 8 * 2^-24 of it, exp2 and the sum 2^-20, above and below
    the division.  The parts leave ``LEFT_OUT`` of a weight out, and the output is rounded once."""
    generator = torch.Generator().manual_seed(seed)
    queries = torch.zeros(heads, width, dtype=dtype)
    queries[:, 0] = (torch.rand(heads, generator=generator) + 0.5).to(dtype)
    keys = torch.zeros(heads, n, width, dtype=dtype)
    keys[..., 0] = torch.randn(heads, n, generator=generator).clamp(-2, 2).to(dtype)
    keys[:, 0, 0] = 2.5
    values = torch.randn(heads, n, width, generator=generator).to(dtype)
    scores = torch.einsum("hd,hnd->hn", queries.double(), keys.double())
    share = torch.softmax(scores, 1)
    values[:, 0] = (-torch.einsum("hn,hnd->hd", share[:, 1:], values[:, 1:].double()) / share[:, :1]).to(dtype)

    def outputs(count=None):
        weight = torch.exp(scores - scores.amax(1, keepdim=True))
        held = weight if count is None else parts_of(weight, dtype, count)
        return torch.einsum("hn,hnd->hd", held, values.double()) / weight.sum(1, keepdim=True)

    slack = 8 * 2.0 ** -24 * scores.abs().amax(1, keepdim=True) + 2.0 ** -20
    mass = torch.einsum("hn,hnd->hd", share, values.double().abs())
    bound = STEP[dtype] * outputs().abs() + (LEFT_OUT[dtype] + 2 * slack) * mass + 2.0 ** -25
    return queries, keys, values, outputs, bound
