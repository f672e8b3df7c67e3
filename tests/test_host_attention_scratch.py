"""The states and workspaces of attention over pages, as host threads ask for them: the class on the CPU, with a stub for the
stream it waits for."""

import threading
import time

import pytest
import torch

from mlkit_b200 import kernels


class SlowStream:
    """A stream whose wait gives the other threads their turn."""

    def synchronize(self):
        time.sleep(0.05)


@pytest.fixture
def on_the_cpu(monkeypatch):
    monkeypatch.setattr(kernels.torch.cuda, "current_stream", lambda index=None: SlowStream())
    monkeypatch.setattr(kernels, "_capturing", lambda: False)


def in_threads(count, work):
    """``work(i)`` in ``count`` threads that begin together; their results."""
    results, failures, gate = [None] * count, [], threading.Barrier(count)

    def run(i):
        try:
            gate.wait()
            results[i] = work(i)
        except Exception as error:
            failures.append(error)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(count)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert not failures, failures
    return results


def test_threads_with_a_stream_each_get_states_of_their_own(on_the_cpu):
    scratch = kernels._AttentionScratch()
    given = in_threads(6, lambda i: scratch.of("cpu", 100 + i, 64)[0])
    everything = given + scratch.left
    assert len(set(everything)) == len(everything)
    ordered = sorted(everything)
    assert all(after - before >= kernels.STATE_BYTES for before, after in zip(ordered, ordered[1:]))


def test_threads_that_come_first_share_one_scratch(on_the_cpu, monkeypatch):
    monkeypatch.setattr(kernels, "_attention_scratch", {})
    create = kernels._AttentionScratch

    def slowly():
        time.sleep(0.02)
        return create()

    monkeypatch.setattr(kernels, "_AttentionScratch", slowly)
    given = in_threads(4, lambda i: kernels._scratch("cpu"))
    assert all(scratch is given[0] for scratch in given)


@pytest.mark.parametrize("rope", [False, True])
def test_no_call_of_another_thread_comes_between_the_launches_of_a_call(on_the_cpu, monkeypatch, rope):
    """The C entry stands for two launches; a workspace that threads share must not be rewritten between them."""
    monkeypatch.setattr(kernels, "_attention_scratch", {})
    monkeypatch.setattr(kernels, "_plans", {})
    monkeypatch.setattr(kernels, "_current_device", lambda: "cpu")
    monkeypatch.setattr(kernels, "_raw_stream", lambda index: 7)
    inside, overlaps = [], []

    def entry(*arguments):
        inside.append(1)
        time.sleep(0.02)
        overlaps.append(len(inside))
        inside.pop()
        return 0

    monkeypatch.setattr(kernels, "_plan_rope_attention" if rope else "_plan_attention", lambda *arguments: ("cpu", entry, 64, ()))
    rows, pages = torch.zeros(2, 4, 64), torch.zeros(3, 2, 16, 64)
    held, tables, weights = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 1, dtype=torch.int32), torch.zeros(3, 2, 16)

    def call(i):
        if rope:
            kernels.paged_rope_attention_decode(rows.view(2, 256), held, held, pages, pages, tables, rows, q_heads=4, kv_heads=2,
                                                head_dim=64, theta=1e4, weights=weights)
        else:
            kernels.paged_attention_decode(rows, held, pages, pages, tables, rows, weights=weights)

    in_threads(4, call)
    assert overlaps == [1, 1, 1, 1]


def test_after_an_eager_call_there_are_states_for_a_whole_capture(on_the_cpu, monkeypatch):
    scratch = kernels._AttentionScratch()
    for attempt in range(5):
        scratch.of("cpu", 7 + attempt, 64)
        assert len(scratch.left) >= kernels.STATES
        monkeypatch.setattr(kernels, "_capturing", lambda: True)
        given = [scratch.of("cpu", 7, 64)[0] for _ in range(100)]
        monkeypatch.setattr(kernels, "_capturing", lambda: False)
        blocks = [(block.data_ptr(), block.data_ptr() + block.numel()) for block in scratch.blocks]
        assert all(any(low <= state < high for low, high in blocks) for state in given)      # none is its graph's to clear
