"""GPU tests of logit penalties in buffers that are wider than their texts, as ``LogitRules`` keeps them."""

import pytest
import torch

import mlkit_b200 as mk
from mlkit_b200 import kernels

pytestmark = pytest.mark.gpu


def given(rows, vocab, capacity, lengths, dtype, biases=5, seed=0):
    generator = torch.Generator().manual_seed(seed)
    random = lambda *shape: torch.rand(shape, generator=generator)
    logits = (torch.randn(rows, vocab, generator=generator) * 3).to(dtype).cuda()
    tokens = (random(rows, capacity) ** 4 * vocab).long().cuda()
    held = torch.tensor(lengths, dtype=torch.int32).cuda()
    arguments = {"lengths": held, "prompts": held // 3, "repetition": (random(rows) + 0.8).cuda(), "frequency": random(rows).cuda(),
                 "presence": random(rows).cuda(), "bias_tokens": torch.randint(0, vocab, (rows, biases), generator=generator).int().cuda(),
                 "bias": torch.randn(rows, biases, generator=generator).cuda()}
    return logits, tokens, arguments


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(6, 30011), (200, 5000), (1, 140000)])
def test_the_width_of_a_buffer_changes_no_result(dtype, rows, vocab):
    """Texts of every kind in one batch: none, some, as many as the table just takes with the biases, and more."""
    lengths = [(0, 300, 6139, 6140, 20000, 1)[row % 6] if rows > 1 else 6139 for row in range(rows)]
    logits, tokens, arguments = given(rows, vocab, 32768, lengths, dtype)
    picked, together = torch.zeros(rows, dtype=torch.int64, device="cuda"), torch.empty_like(logits)
    kernels.adjust_logits(logits, tokens=tokens, out=together, picked=picked, **arguments)
    for row in range(min(rows, 12)):
        one = {name: value[row:row + 1] for name, value in arguments.items()}
        alone, best = torch.empty_like(logits[:1]), torch.zeros(1, dtype=torch.int64, device="cuda")
        kernels.adjust_logits(logits[row:row + 1], tokens=tokens[row:row + 1, :max(1, lengths[row])], out=alone, picked=best, **one)
        assert torch.equal(alone[0], together[row]) and int(best) == int(picked[row]), row


def quickest(calls, repeats=40):
    """The shortest device time of each call in us, taken in turn; a call's launches are queued behind a copy of 1 GB, so the
    host's side is over before they begin."""
    wait = torch.empty(1 << 29, dtype=torch.uint8, device="cuda"), torch.empty(1 << 29, dtype=torch.uint8, device="cuda")
    times = [[] for _ in calls]
    for _ in range(repeats):
        for call, into in zip(calls, times):
            begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            wait[0].copy_(wait[1])
            begin.record()
            for _ in range(4):
                call()
            end.record()
            end.synchronize()
            into.append(begin.elapsed_time(end) * 250)
    return [min(into) for into in times]


@pytest.mark.parametrize("rows", [1, 8, 128])
def test_a_short_text_in_a_wide_buffer_is_a_short_call(rows):
    """By the width of the buffer it would take several chunks with the largest table each: 1.5 to 4 times the time.  The larger
    table alone takes up to 1.11 times."""
    logits, tokens, arguments = given(rows, 128256, 32768, [300] * rows, torch.bfloat16)
    narrow, out = tokens[:, :300].contiguous(), torch.empty_like(logits)
    wide, fitting = quickest([lambda: kernels.adjust_logits(logits, tokens=tokens, out=out, **arguments),
                              lambda: kernels.adjust_logits(logits, tokens=narrow, out=out, **arguments)])
    print(f"{rows} rows: buffer of 32768 {wide:.1f} us, of 300 {fitting:.1f} us")
    assert wide < 1.35 * fitting, (wide, fitting)


def test_rules_at_the_length_of_a_context():
    """``LogitRules`` of 32768 tokens and of 64 give the same logits and picks."""
    results = []
    for capacity in (64, 32768):
        rules = mk.LogitRules(rows=3, capacity=capacity, biases=2, vocab=20000)
        generator = torch.Generator(device="cuda").manual_seed(0)
        for row in range(3):
            rules.begin(row, range(7 * row), repetition=1.2, frequency=0.3, bias={5: 1.0})
        for _ in range(20):
            logits = torch.randn(3, 20000, device="cuda", generator=generator).half()
            picked = torch.empty(3, dtype=torch.int64, device="cuda")
            rules.apply(logits, picked=picked)
            rules.observe(picked)
        results.append((logits, picked, rules.tokens[:, :64]))
    for one, other in zip(*results):
        assert torch.equal(one, other)
