"""GPU tests of the penalties, biases and masks on logits, against a 64-bit restatement."""

import math

import pytest
import torch

from mlkit_b200 import kernels
from tests.paged_reference import STEP, adjusted

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def check(rows, vocab, offset, width, history, biases, masked, dtype, *, long=True, in_place=False, parts="rfpbmq", seed=0):
    generator = torch.Generator().manual_seed(seed)
    random = lambda *shape: torch.rand(shape, generator=generator)
    logits = (torch.randn(rows, width, generator=generator) * 3).to(dtype)
    tokens = (random(rows, history) ** 3 * (vocab + 4)).long() - 2          # some ids are none of the vocabulary
    lengths = torch.randint(-1, history + 9, (rows,), generator=generator).int()
    lengths[0] = history
    prompts = torch.randint(-1, history + 9, (rows,), generator=generator).int()
    repetition, frequency, presence = random(rows) + 0.7, random(rows) - 0.2, random(rows) - 0.2
    bias_tokens = (torch.randint(-1, vocab, (rows, biases), generator=generator) // 3 * 2).int()   # many twice
    bias = torch.randn(rows, biases, generator=generator) * 4
    mask = torch.randint(-(1 << 31), 1 << 31, (rows, -(-(offset + width) // 32)), generator=generator).int()
    if masked and rows > 2:
        mask[1] = 0                                                           # a grammar that allows nothing
        mask[2] = -1
    best, picked = torch.zeros(rows, dtype=torch.int64, device="cuda"), torch.zeros(rows, dtype=torch.int64, device="cuda")
    given = logits.cuda()
    out = given if in_place else torch.full_like(given, 9.0)
    gpu = lambda x, part=None: x.cuda() if part is None or part in parts else None
    kernels.adjust_logits(given, tokens=gpu(tokens if long else tokens.int()) if history else None,
                          lengths=gpu(lengths) if history else None, prompts=gpu(prompts, "q") if history else None,
                          repetition=gpu(repetition, "r") if history else None, frequency=gpu(frequency, "f") if history else None,
                          presence=gpu(presence, "p") if history else None, bias_tokens=gpu(bias_tokens) if biases else None,
                          bias=gpu(bias) if biases else None, mask=gpu(mask) if masked else None, offset=offset, best=best,
                          picked=picked, out=None if in_place else out)
    if not in_place:
        assert torch.equal(given.cpu(), logits)
    got = out.cpu()
    for m in range(rows):
        held = min(max(int(lengths[m]), 0), history)
        expected = adjusted(
            logits[m], offset, history=tokens[m, :held].tolist(), prompt=int(prompts[m]) if "q" in parts else 0,
            repetition=float(repetition[m]) if "r" in parts else 1.0, frequency=float(frequency[m]) if "f" in parts else 0.0,
            presence=float(presence[m]) if "p" in parts else 0.0,
            biases=list(zip(bias_tokens[m].tolist(), bias[m].tolist())), mask=[int(w) & 0xffffffff for w in mask[m]] if masked else None)
        # a division or product, two differences, a product and a sum in fp32, each off by half a step of what passes through
        counts = torch.bincount(tokens[m, :held].clamp(min=0), minlength=offset + width + 4)[offset:offset + width]
        through = logits[m].double().abs() * 2 + counts * 1.0 + 2
        if biases:
            inside = (bias_tokens[m] >= offset) & (bias_tokens[m] < offset + width)
            through.index_add_(0, bias_tokens[m][inside].long() - offset, bias[m][inside].double().abs())
        bound = STEP[dtype] * expected.abs() + 6 * 2.0 ** -24 * through
        fine = torch.isfinite(expected)
        assert torch.equal(got[m].double()[~fine], expected[~fine])
        off = (got[m].double() - expected).abs()
        assert (off[fine] <= bound[fine]).all(), (m, float((off / bound)[fine].max()))
    # the pick is the result's own, the lowest token on a tie
    top = torch.where(got == got.amax(1, keepdim=True), torch.arange(width), width).amin(1) + offset
    assert torch.equal(picked.cpu(), top)
    assert torch.equal(kernels.tokens_of_keys(best).cpu(), top)
    if dtype == torch.float16:
        keys = torch.zeros(rows, dtype=torch.int64, device="cuda")
        kernels.argmax_keys(out, keys, offset=offset)
        assert torch.equal(keys, best)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,offset,width", [(1, 1000, 0, 1000), (5, 997, 0, 997), (3, 4000, 1999, 2001), (4, 33, 32, 1),
                                                     (3, 70001, 0, 70001), (2, 300000, 100001, 199999)])
def test_adjusted_logits(dtype, rows, vocab, offset, width):
    check(rows, vocab, offset, width, 40, 9, True, dtype)


@pytest.mark.parametrize("parts", ["r", "f", "p", "fq", "rp", ""])
def test_parts_of_the_penalties(parts):
    check(3, 500, 100, 300, 200, 0, False, torch.float32, parts=parts)


@pytest.mark.parametrize("history,biases,masked", [(0, 0, False), (0, 0, True), (0, 5, False), (1, 0, False), (3000, 0, True), (9, 1500, False)])
def test_histories_biases_and_masks_alone(history, biases, masked):
    check(4, 2000, 0, 2000, history, biases, masked, torch.bfloat16, long=False)


@pytest.mark.parametrize("rows,vocab,history,biases", [(2, 20000, 6144, 0), (2, 20000, 6000, 145), (3, 30011, 20000, 700), (1, 140000, 9000, 0)])
def test_histories_beyond_the_table(rows, vocab, history, biases):
    """More tokens than the hash table of a CTA takes, and as many as it just takes."""
    check(rows, vocab, 0, vocab, history, biases, False, torch.float32)


def test_a_table_full_of_different_tokens():
    """6144 different tokens, the most of a table, in one slice and over several; and 6145."""
    for history, step in ((6144, 1), (6144, 3), (6145, 1)):
        tokens = (torch.arange(history) * step).view(1, -1)
        width = int(tokens.max()) + 10
        logits = torch.randn(1, width, generator=torch.Generator().manual_seed(0))
        out = kernels.adjust_logits(logits.cuda(), tokens=tokens.cuda(), lengths=torch.tensor([history], dtype=torch.int32).cuda(),
                                    presence=torch.tensor([2.0]).cuda())
        expected = logits.clone()
        expected[0, tokens[0]] -= 2.0
        assert torch.equal(out.cpu(), expected)


@pytest.mark.parametrize("rows", [1, 9, 200])
def test_in_place_and_batches(rows):
    check(rows, 3000, 0, 3000, 64, 4, True, torch.float16, in_place=True, long=rows == 9)


def test_biases_of_one_token_many_times():
    """1500 entries of three tokens: added up in their order in 64 bits, whichever threads meet them."""
    entries = torch.randint(0, 3, (2, 1500), generator=torch.Generator().manual_seed(0)) * 400 + 17
    values = torch.randn(2, 1500, generator=torch.Generator().manual_seed(1)) * 100
    logits = torch.zeros(2, 1000, device="cuda")
    outs = [kernels.adjust_logits(logits.clone(), bias_tokens=entries.int().cuda(), bias=values.cuda()) for _ in range(5)]
    expected = torch.zeros(2, 1000, dtype=torch.float64).scatter_add_(1, entries, values.double()).float()
    for out in outs:
        assert torch.equal(out.cpu(), expected)


def test_zeros_of_both_signs_tie():
    logits = torch.full((3, 5000), -1.0)
    logits[0, 700], logits[0, 701], logits[1, 4000], logits[1, 4999], logits[2, 3] = -0.0, 0.0, 0.0, -0.0, -0.0
    for dtype in DTYPES:
        picked = torch.zeros(3, dtype=torch.int64, device="cuda")
        kernels.adjust_logits(logits.to(dtype).cuda(), picked=picked)
        assert picked.tolist() == [700, 4000, 3]


def test_one_token_many_times():
    """A count that a 16-bit type would round: 5001 occurrences, of which 5000 generated."""
    tokens = torch.full((1, 5001), 7, dtype=torch.int64, device="cuda")
    logits = torch.ones(1, 64, device="cuda")
    out = kernels.adjust_logits(logits.clone(), tokens=tokens, lengths=torch.tensor([5001], dtype=torch.int32, device="cuda"),
                                prompts=torch.tensor([1], dtype=torch.int32, device="cuda"),
                                frequency=torch.tensor([0.5], device="cuda"))
    assert float(out[0, 7]) == 1.0 - 2500.0 and torch.equal(out[0, :7], logits[0, :7]) and torch.equal(out[0, 8:], logits[0, 8:])


def test_logits_that_are_not_finite():
    logits = torch.tensor([[math.nan, 1.0, math.inf, -math.inf, 2.0], [math.nan] * 5, [-math.inf] * 5, [3.0, math.inf, math.inf, 0, 0]])
    picked = torch.zeros(4, dtype=torch.int64, device="cuda")
    mask = torch.tensor([[0b11011], [31], [31], [31]], dtype=torch.int32, device="cuda")
    out = kernels.adjust_logits(logits.half().cuda(), mask=mask, picked=picked).cpu()
    assert torch.isnan(out[0, 0]) and out[0, 2] == -math.inf and torch.isnan(out[1]).all()
    assert picked.tolist() == [4, 0, 0, 1]


def test_rows_with_strides():
    wide = torch.randn(4, 900, device="cuda").half()
    logits, out = wide[:, 100:800], torch.zeros(4, 1000, device="cuda").half()[:, 7:707]
    tokens = torch.randint(0, 700, (4, 64), device="cuda")
    arguments = {"lengths": torch.full((4,), 20, dtype=torch.int32, device="cuda"), "repetition": torch.full((4,), 1.3, device="cuda")}
    expected = kernels.adjust_logits(logits.contiguous(), tokens=tokens[:, 10:30].contiguous(), **arguments)
    kernels.adjust_logits(logits, tokens=tokens[:, 10:30], out=out, **arguments)
    assert torch.equal(out, expected)


def test_adjusted_logits_in_a_graph():
    logits, tokens = torch.randn(3, 5000, device="cuda"), torch.randint(0, 5000, (3, 100), device="cuda")
    lengths, out = torch.full((3,), 10, dtype=torch.int32, device="cuda"), torch.empty(3, 5000, device="cuda")
    presence = torch.full((3,), 2.0, device="cuda")
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kernels.adjust_logits(logits, tokens=tokens, lengths=lengths, presence=presence, out=out)
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            kernels.adjust_logits(logits, tokens=tokens, lengths=lengths, presence=presence, out=out)
    torch.cuda.synchronize()
    lengths.fill_(100)
    graph.replay()
    torch.cuda.synchronize()
    expected = kernels.adjust_logits(logits, tokens=tokens, lengths=lengths, presence=presence, out=torch.empty_like(out))
    assert torch.equal(out, expected) and (out != logits).sum() > 200


def test_logits_and_results_beside_each_other():
    buffer = torch.randn(5, 2000, device="cuda").half()
    expected = kernels.adjust_logits(buffer[:, :1000].contiguous(), mask=torch.full((5, 32), 0x0F0F0F0F, dtype=torch.int32, device="cuda"))
    left = buffer[:, :1000].clone()
    kernels.adjust_logits(buffer[:, :1000], mask=torch.full((5, 32), 0x0F0F0F0F, dtype=torch.int32, device="cuda"), out=buffer[:, 1000:])
    assert torch.equal(buffer[:, 1000:], expected) and torch.equal(buffer[:, :1000], left)
