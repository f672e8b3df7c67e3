"""GPU tests of the decoder over a paged cache: the attention, the eviction and the logit rules as a serving loop runs them."""

import math

import pytest
import torch

import mlkit_b200 as mk
from mlkit_b200 import kernels, tp
from tests.paged_reference import adjusted, slots_of
from tests.test_gpu_tp import build_model, dense_reference_step, quantised_block, rel

pytestmark = pytest.mark.gpu
CONFIG = tp.DecoderConfig(layers=2, hidden=256, q_heads=4, kv_heads=2, head_dim=128, intermediate=512, vocab=512)


@pytest.fixture(scope="module")
def parts():
    generator = torch.Generator(device="cuda").manual_seed(7)
    random = lambda *shape: torch.randn(shape, device="cuda", generator=generator)
    blocks = [quantised_block(CONFIG, 50 + i) for i in range(CONFIG.layers)]
    return blocks, random(CONFIG.vocab, CONFIG.hidden).half(), (random(CONFIG.hidden).abs() + 0.5).half(), (random(CONFIG.vocab, CONFIG.hidden) * 0.05).half()


def references(rows):
    shape = (rows, CONFIG.kv_heads, 64, CONFIG.head_dim)
    return [[torch.zeros(shape, device="cuda") for _ in range(CONFIG.layers)] for _ in range(2)]


@pytest.mark.parametrize("page", [1, 5, 16])
@pytest.mark.parametrize("captured", [False, True])
def test_paged_decoder_matches_dense_reference(parts, page, captured):
    """Three rows that begin at different steps, one of them twice."""
    model = build_model(CONFIG, *parts, page=page)
    cache, (k_ref, v_ref) = model.cache, references(3)
    run = model.capture(3) if captured else None
    assert cache.held == [-1] * 4 and len(cache.free) == cache.pages      # capturing took nothing
    generator = torch.Generator(device="cuda").manual_seed(page)
    for step in range(9):
        if step in (0, 1, 4):
            cache.open({0: 1, 1: 0, 4: 2}[step])
        if step == 6:
            cache.release(1)
            cache.open(1)
        tokens = torch.randint(0, CONFIG.vocab, (3,), device="cuda", generator=generator)
        rows = [row for row in range(3) if cache.held[row] >= 0]
        positions = torch.tensor([max(0, held) for held in cache.held[:3]], dtype=torch.int32, device="cuda")
        if captured:
            run.tokens.copy_(tokens)
            run.positions.copy_(positions)
            logits = run.replay()
        else:
            logits = model.step(tokens, positions)
        expected = dense_reference_step(CONFIG, *parts, tokens, positions, k_ref, v_ref)
        assert rel(logits[rows], expected[rows]) < 1e-2, step
    assert cache.lengths.tolist() == cache.held == [8, 3, 5, -1] and kernels.decode_status() == 0


@pytest.mark.parametrize("captured", [False, True])
def test_rules_of_a_greedy_decoder(parts, captured):
    model = build_model(CONFIG, *parts, page=8)
    plain = build_model(CONFIG, *parts, page=8)
    rules = mk.LogitRules(rows=4, capacity=16, biases=3, vocab=CONFIG.vocab)
    settings = [dict(repetition=1.3, presence=0.5, bias={7: 2.5, 300: -4.0}), dict(frequency=0.8, prompt=[3, 3, 9]), {}]
    for row, setting in enumerate(settings):
        rules.begin(row, setting.pop("prompt", []), **setting)
        for m in (model, plain):
            m.cache.open(row)
    allowed = list(range(0, CONFIG.vocab, 3))
    rules.allow(2, allowed)
    run = model.capture(3, greedy=True, rules=rules) if captured else None
    histories = [[], [3, 3, 9], []]
    tokens = torch.tensor([3, 9, 200], device="cuda")
    for step in range(6):
        positions = torch.full((3,), step, dtype=torch.int32, device="cuda")
        raw = plain.step(tokens, positions).clone()
        if captured:
            run.tokens.copy_(tokens)
            run.positions.copy_(positions)
            picked = run.replay().clone()
        else:
            picked = model.step(tokens, positions, greedy=True, rules=rules)
        for row, setting in enumerate(settings):
            setting = dict(setting)
            expected = adjusted(raw[row].cpu(), 0, history=histories[row], prompt=3 if row == 1 else 0,
                                biases=list(setting.pop("bias", {}).items()), **setting)
            if row == 2:
                expected[[t for t in range(CONFIG.vocab) if t not in allowed]] = -math.inf
            # the pick is the reference's, up to what the rounding of the result to fp16 makes equal
            best = float(expected.max())
            assert float(expected[picked[row]]) >= best - 2 * 2.0 ** -11 * abs(best)
            histories[row].append(int(picked[row]))
        assert rules.lengths.tolist() == [step + 1, step + 4, step + 1, 0]
        tokens = picked
    assert [rules.tokens[row, :int(rules.lengths[row])].tolist() for row in range(3)] == histories
    assert all(token in allowed for token in histories[2])


def test_decoder_evicts_and_goes_on(parts):
    """Captured steps, eviction, captured steps: as a decoder whose cache was given the kept slots from the start."""
    model = build_model(CONFIG, *parts, page=4, track_weights=True)
    other = build_model(CONFIG, *parts, page=16)
    cache, run = model.cache, model.capture(2)
    generator = torch.Generator(device="cuda").manual_seed(1)
    tokens_of = lambda: torch.randint(0, CONFIG.vocab, (2,), device="cuda", generator=generator)
    cache.open(0)
    for step in range(30):
        if step == 20:
            cache.open(1)
        run.tokens.copy_(tokens_of())
        run.positions.copy_(torch.tensor([step, max(0, step - 20)], dtype=torch.int32))
        run.replay()
    total = cache.weights[0][cache.owned[0]].sum(-1).sum(0)[0]
    # every step's weights add up to one for each of the two query heads of a group: 30 steps of sums of about a thousand
    # terms of 2^-23 each
    assert abs(float(total) - 60.0) < 60 * 2.0 ** -13
    before = [[slots_of(pool.cpu(), cache.tables[0].cpu(), 30) for pool in pools] for pools in (cache.k_pages, cache.v_pages)]
    weights = [slots_of(pool.cpu(), cache.tables[0].cpu(), 30) for pool in cache.weights]
    kept = cache.evict(13, sinks=2, recent=4)
    assert list(kept) == [0] and cache.held == [13, 10, -1, -1] == cache.lengths.tolist()
    assert sorted(sum(cache.owned, []) + cache.free) == list(range(cache.pages))
    for row in (0, 1):
        other.cache.open(row)
    for layer in range(CONFIG.layers):
        index = kept[0][layer].cpu().long()
        assert (index[:, :2] == torch.arange(2)).all() and (index[:, -4:] == torch.arange(26, 30)).all()
        take = lambda data: data.gather(1, index[:, :, None].expand(-1, -1, CONFIG.head_dim))
        keys, values = (take(data[layer]) for data in before)
        assert torch.equal(slots_of(cache.k_pages[layer].cpu(), cache.tables[0].cpu(), 13), keys)
        assert torch.equal(slots_of(cache.weights[layer].cpu(), cache.tables[0].cpu(), 13), weights[layer].gather(1, index))
        other.cache.write(layer, 0, keys.cuda(), values.cuda())
        other.cache.write(layer, 1, *(slots_of(pool[layer].cpu(), cache.tables[1].cpu(), 10).cuda() for pool in (cache.k_pages, cache.v_pages)))
    other.cache.extend(0, 13)
    other.cache.extend(1, 10)
    for step in range(30, 36):        # the text goes on at its positions, whatever was evicted
        run.tokens.copy_(tokens_of())
        run.positions.copy_(torch.tensor([step, step - 20], dtype=torch.int32))
        assert rel(run.replay(), other.step(run.tokens, run.positions)) < 2e-3
    assert cache.held == [19, 16, -1, -1] and kernels.decode_status() == 0


def test_an_eager_step_without_a_page_left_changes_nothing(parts):
    model = build_model(CONFIG, *parts, page=2, pages=2)
    for row in (0, 1):
        model.cache.open(row)
    tokens, positions = torch.tensor([1, 2], device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    for _ in range(2):
        model.step(tokens, positions)
    before = [pool.clone() for pool in model.cache.k_pages]
    with pytest.raises(RuntimeError, match="free pages"):
        model.step(tokens, positions)
    assert model.cache.held[:2] == [2, 2] and all(torch.equal(*pair) for pair in zip(before, model.cache.k_pages))


def test_rules_that_do_not_fit_are_refused_before_the_step(parts):
    model = build_model(CONFIG, *parts, page=8)
    model.cache.open(0)
    tokens, positions = torch.tensor([1, 2], device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    for rules in (mk.LogitRules(rows=1, capacity=4), mk.LogitRules(rows=2, capacity=4, vocab=CONFIG.vocab - 1)):
        with pytest.raises(ValueError, match="rules of"):
            model.step(tokens, positions, greedy=True, rules=rules)
    assert model.cache.held[0] == 0 and int(model.cache.lengths[0]) == 0


def test_decoders_refuse_what_does_not_belong_together():
    with pytest.raises(ValueError, match="page size"):
        tp.TensorParallelDecoder(CONFIG, track_weights=True)
    with pytest.raises(ValueError, match="page size"):
        tp.TensorParallelDecoder(CONFIG, pages=8)
    with pytest.raises(ValueError, match="cache.write"):
        tp.TensorParallelDecoder(CONFIG, page=16).fill_cache(3)
