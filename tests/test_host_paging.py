"""The bookkeeping of the paged cache and of the logit rules, on the CPU; their kernels are tested on a GPU."""

import pytest
import torch

import mlkit_b200 as mk


def cache(**changed):
    return mk.PagedCache(**({"rows": 3, "columns": 4, "kv_heads": 2, "head_dim": 64, "page": 8, "pages": 6, "layers": 2, "device": "cpu"} | changed))


def consistent(c):
    owned = [page for pages in c.owned for page in pages]
    assert sorted(owned + c.free) == list(range(c.pages))           # every page is free or one row's
    assert c.lengths.tolist() == c.held
    for row, pages in enumerate(c.owned):
        assert c.tables[row, :len(pages)].tolist() == pages


def step(c, batch):
    c.prepare(batch)
    c.count(batch)
    c.advance(batch)


def test_pages_are_taken_as_sequences_grow_and_given_back():
    c = cache()
    c.open(0)
    c.open(2)
    for _ in range(9):
        step(c, 3)
        consistent(c)
    assert c.held == [9, -1, 9] and [len(pages) for pages in c.owned] == [2, 0, 2]
    c.release(0)
    c.open(0)
    c.open(1)
    consistent(c)
    step(c, 3)
    assert c.held == [1, 1, 10] and len(c.free) == 2
    step(c, 2)                                                       # the third row is behind the batch
    assert c.held == [2, 2, 10]
    c.release(1)
    c.release(1)                                                     # nothing to give back
    consistent(c)


def test_a_pool_that_is_used_up_refuses_before_anything_changes():
    c = cache(pages=3)
    for row in range(3):
        c.open(row)
    for _ in range(8):
        step(c, 3)
    with pytest.raises(RuntimeError, match="free pages"):
        c.prepare(3)
    consistent(c)
    assert c.held == [8, 8, 8] and not c.free
    c.release(1)
    c.prepare(1)
    with pytest.raises(RuntimeError, match="free pages"):
        c.prepare(3)


def test_a_sequence_does_not_outgrow_its_row():
    c = cache(pages=20)
    c.open(1)
    c.reserve(1, 32)
    with pytest.raises(ValueError, match="exceeds"):
        c.reserve(1, 33)
    for _ in range(32):
        step(c, 3)
    with pytest.raises(ValueError, match="exceeds"):
        c.prepare(3)
    consistent(c)


def test_rows_in_use_and_not():
    c = cache()
    c.open(0)
    with pytest.raises(ValueError, match="in use"):
        c.open(0)
    with pytest.raises(ValueError, match="not in use"):
        c.reserve(1, 3)
    with c.idle():
        step(c, 3)
        assert c.lengths.tolist() == [-1, -1, -1]
    assert c.lengths.tolist() == c.held == [0, -1, -1] and len(c.free) == 6


def test_prompts_are_written_behind_the_slots():
    c = cache(track_weights=True)
    c.open(1)
    step(c, 2)
    for weights in c.weights:
        weights.fill_(3.0)
    keys, values = torch.randn(2, 12, 64), torch.randn(2, 12, 64)
    for layer in range(2):
        c.write(layer, 1, keys + layer, values - layer)
    c.extend(1, 12)
    consistent(c)
    assert c.held == [-1, 13, -1]
    for layer in range(2):
        for slot in range(1, 13):
            page, at = c.owned[1][slot // 8], slot % 8
            assert torch.equal(c.k_pages[layer][page, :, at], (keys[:, slot - 1] + layer).half())
            assert torch.equal(c.v_pages[layer][page, :, at], (values[:, slot - 1] - layer).half())
            assert not c.weights[layer][page, :, at].any()
    assert float(c.weights[0][c.owned[1][0], 0, 0]) == 3.0
    with pytest.raises(ValueError, match="keys and values"):
        c.write(0, 1, keys[:1], values)


def test_an_eviction_that_fails_leaves_the_cache_as_it_was():
    """On the CPU the kernel's wrapper refuses the pools."""
    c = cache(track_weights=True)
    c.open(0)
    for _ in range(20):
        step(c, 1)
    before = (list(c.free), [list(pages) for pages in c.owned], list(c.held), c.tables.clone())
    with pytest.raises(ValueError, match="CUDA"):
        c.evict(10)
    assert before[:3] == (c.free, c.owned, c.held) and torch.equal(before[3], c.tables)
    consistent(c)


def test_what_a_cache_refuses():
    for changed in ({"rows": 0}, {"columns": 0}, {"page": 0}, {"pages": 0}, {"head_dim": 96}, {"dtype": torch.float32}, {"kv_heads": 0}):
        with pytest.raises(ValueError):
            cache(**changed)
    with pytest.raises(ValueError, match="tracks weights"):
        cache().evict(4)
    for budget, sinks, recent in ((0, 0, 0), (4, 3, 2), (4, -1, 0)):
        with pytest.raises(ValueError):
            cache(track_weights=True).evict(budget, sinks=sinks, recent=recent)


def rules(**changed):
    return mk.LogitRules(**({"rows": 2, "capacity": 4, "biases": 2, "vocab": 70, "device": "cpu"} | changed))


def test_histories_grow_to_their_capacity():
    r = rules()
    r.begin(1, [5, 6, 7], repetition=1.5, presence=0.5)
    assert r.lengths.tolist() == [0, 3] and r.prompts.tolist() == [0, 3] and r.repetition.tolist() == [1.0, 1.5]
    for token in (11, 12, 13):
        r.observe(torch.tensor([token, token + 20]))
    assert r.tokens.tolist() == [[11, 12, 13, -1], [5, 6, 7, 31]] and r.lengths.tolist() == [3, 4]
    r.observe(torch.tensor([14]))                                    # a batch of one row
    assert r.tokens[0].tolist() == [11, 12, 13, 14] and r.lengths.tolist() == [4, 4]
    r.begin(1)
    assert r.lengths.tolist() == [4, 0] and r.repetition.tolist() == [1.0, 1.0] and r.presence.tolist() == [0.0, 0.0]


def test_biases_and_masks_of_a_row():
    r = rules()
    r.begin(0, bias={3: 1.5, 69: -2.0})
    assert r.bias_tokens.tolist() == [[3, 69], [-1, -1]] and r.bias[0].tolist() == [1.5, -2.0]
    r.allow(1, [0, 31, 32, 69])
    assert [word & 0xffffffff for word in r.mask[1].tolist()] == [1 | 1 << 31, 1, 1 << 5] and r.mask[0].tolist() == [-1] * 3
    r.allow(1, [])
    assert r.mask[1].tolist() == [0, 0, 0]
    r.begin(1, bias={4: 0.5})
    assert r.mask[1].tolist() == [-1] * 3 and r.bias_tokens[1].tolist() == [4, -1]
    r.begin(0)
    assert r.bias_tokens[0].tolist() == [-1, -1]


def test_what_rules_refuse():
    r = rules()
    for call in (lambda: r.begin(0, range(5)), lambda: r.begin(0, repetition=0.0), lambda: r.begin(0, bias={1: 1.0, 2: 1.0, 3: 1.0}),
                 lambda: r.allow(0, [70]), lambda: rules(vocab=None).allow(0, [1]), lambda: rules(biases=0).begin(0, bias={1: 1.0}),
                 lambda: rules(rows=0), lambda: rules(capacity=0)):
        with pytest.raises(ValueError):
            call()
