"""GPU tests of the paged cache's bookkeeping beside work that is under way."""

import pytest
import torch

import mlkit_b200 as mk

pytestmark = pytest.mark.gpu


def work(seconds=0.3):
    """Copies that keep the stream busy, and the event behind them."""
    data = torch.empty(1 << 30, dtype=torch.uint8, device="cuda"), torch.empty(1 << 30, dtype=torch.uint8, device="cuda")
    for _ in range(int(seconds * 3000)):
        data[0].copy_(data[1])
    event = torch.cuda.Event()
    event.record()
    return event


def grown(cache, rows):
    """Rows that each need a page for their next token."""
    cache.prepare(rows)
    cache.count(rows)
    cache.advance(rows)


def test_pages_are_taken_without_waiting_for_the_stream():
    cache = mk.PagedCache(rows=6, columns=40, kv_heads=1, head_dim=64, page=1, layers=1, track_weights=True)
    for row in (0, 2, 3, 5):
        cache.open(row)
    for _ in range(3):
        grown(cache, 6)
    cache.evict(2)          # kernels that are called for the first time are loaded, for which the device is waited for
    for _ in range(2):
        grown(cache, 6)
    cache.open(1)
    cache.release(1)
    torch.cuda.synchronize()
    event = work()
    for _ in range(5):
        grown(cache, 6)
    assert not event.query()
    kept = cache.evict(4, sinks=1)
    assert not event.query() and sorted(kept) == [0, 2, 3, 5]
    cache.release(0)
    cache.open(1)
    cache.extend(1, 3)
    assert not event.query()
    torch.cuda.synchronize()
    assert cache.held == cache.lengths.tolist() == [-1, 3, 4, 4, -1, 4]
    for row in (1, 2, 3, 5):
        assert cache.tables[row, :len(cache.owned[row])].tolist() == cache.owned[row]
    assert sorted(sum(cache.owned, []) + cache.free) == list(range(cache.pages))


def test_page_numbers_arrive_in_the_order_of_the_stream():
    """Numbers of many calls are under way at once: none is overwritten before it is copied."""
    cache = mk.PagedCache(rows=40, columns=50, kv_heads=1, head_dim=64, page=1, layers=0)
    for row in range(40):
        cache.open(row)
    event = work(0.2)
    for _ in range(45):
        grown(cache, 40)
    assert not event.query()
    torch.cuda.synchronize()
    for row in range(40):
        assert cache.tables[row].tolist() == cache.owned[row] + [-1] * 5
    assert cache.lengths.tolist() == cache.held == [45] * 40
