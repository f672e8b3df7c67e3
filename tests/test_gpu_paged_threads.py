"""GPU test of attention with accumulated weights from two host threads that share a stream."""

import threading

import pytest
import torch

from mlkit_b200 import kernels
from tests.paged_reference import make_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("own_streams", [False, True])
def test_threads_accumulate_their_own_weights(own_streams):
    """Each thread's accumulator and output as without the other, bit for bit: results do not depend on what runs beside them."""
    cases = []
    for seed, lengths in enumerate(([900, 40, 333], [5000, 17])):
        keys, values, tables, weights = make_cache(lengths, kv_heads=2, head_dim=64, page=16, dtype=torch.float16, seed=seed)
        q = torch.randn(len(lengths), 8, 64, generator=torch.Generator().manual_seed(seed)).half().cuda()
        cases.append((q, torch.tensor(lengths, dtype=torch.int32).cuda(), keys.cuda(), values.cuda(), tables.cuda(), weights))
    calls = 300

    def run(case, out, weights):
        for _ in range(calls):
            kernels.paged_attention_decode(*case[:5], out, weights=weights)

    alone = [(torch.empty_like(case[0]), case[5].cuda()) for case in cases]
    for case, given in zip(cases, alone):
        run(case, *given)
    torch.cuda.synchronize()
    together = [(torch.empty_like(case[0]), case[5].cuda()) for case in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    gate, failures = threading.Barrier(len(cases)), []

    def thread(i):
        try:
            torch.cuda.synchronize()
            gate.wait()
            if own_streams:
                with torch.cuda.stream(streams[i]):
                    run(cases[i], *together[i])
            else:
                run(cases[i], *together[i])
        except Exception as error:
            failures.append(error)

    threads = [threading.Thread(target=thread, args=(i,)) for i in range(len(cases))]
    for one in threads:
        one.start()
    for one in threads:
        one.join()
    torch.cuda.synchronize()
    assert not failures
    for one, other in zip(alone, together):
        assert torch.equal(one[0], other[0]) and torch.equal(one[1], other[1])
    assert kernels.decode_status() == 0
