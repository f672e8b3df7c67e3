"""What the operators over a paged cache and on logits refuse, on the host alone: no call here reaches a device."""

import pytest
import torch

from mlkit_b200 import _native, kernels

F16, BF16, F32 = _native.F16, _native.BF16, _native.F32
POINTER = 1 << 20
ARGUMENT, UNSUPPORTED, ALIGNMENT, CUDA = -1, -2, -3, -4
needs_no_device = pytest.mark.skipif(torch.cuda.is_available(), reason="an accepted call would launch on made-up addresses")

READ = dict(q=POINTER, lengths=POINTER, k=POINTER, v=POINTER, tables=POINTER, out=2 * POINTER, weights=None, rows=2, q_heads=8, kv_heads=2,
            head_dim=128, page=16, columns=4, pages=10, page_stride=2 * 16 * 128, head_stride=16 * 128, slot_stride=128,
            table_stride=4, q_row=8 * 128, q_head=128, scale=0.1, dtype=F16, state=POINTER, workspace=POINTER, size=1 << 40, stream=None)
EVICT = dict(k=POINTER, v=POINTER, weights=POINTER, tables=POINTER, lengths=POINTER, new=POINTER, kept=POINTER, rows=2, kv_heads=2,
             head_dim=128, page=16, columns=4, new_columns=2, pages=10, page_stride=2 * 16 * 128, head_stride=16 * 128, slot_stride=128,
             table_stride=4, new_stride=2, budget=32, sinks=1, recent=4, stream=None)
ADJUST = dict(logits=POINTER, out=POINTER, tokens=POINTER, lengths=POINTER, prompts=None, repetition=None, frequency=None, presence=None,
              bias_tokens=None, bias=None, mask=None, best=None, picked=None, rows=2, width=1000, stride=1000, out_stride=1000,
              history=5, tokens_stride=5, biases=0, bias_stride=0, words=0, mask_stride=0, offset=0, long=1, dtype=F16, stream=None)


def read(**changed):
    return _native.library().mkb_paged_attention_decode(*(READ | changed).values())


def rope(**changed):
    given = READ | changed
    positions, theta = given.pop("positions", POINTER), given.pop("theta", 1e4)
    given.pop("q_head")
    values = list(given.items())
    at = [name for name, _ in values].index("scale")
    plain = [value for _, value in values]
    return _native.library().mkb_paged_rope_attention_decode(plain[0], positions, *plain[1:at], theta, *plain[at:])


def evict(**changed):
    return _native.library().mkb_paged_evict(*(EVICT | changed).values())


def adjust(**changed):
    return _native.library().mkb_adjust_logits(*(ADJUST | changed).values())


@needs_no_device
@pytest.mark.parametrize("call", [read, rope])
def test_attention_takes(call):
    for changed in ({}, {"dtype": BF16}, {"head_dim": 64}, {"head_dim": 192, "slot_stride": 192}, {"head_dim": 256}, {"q_heads": 2}, {"q_heads": 36}, {"page": 1},
                    {"page": 100}, {"weights": POINTER}):
        assert call(**changed) == CUDA, changed        # accepted: the launch fails, there being no device
    assert call(rows=0) == 0


@needs_no_device
@pytest.mark.parametrize("call", [read, rope])
def test_attention_refuses(call):
    for code, changes in (
            (ARGUMENT, [{name: None} for name in ("q", "lengths", "k", "v", "tables", "out")]),
            (ARGUMENT, [{"rows": -1}, {"q_heads": 0}, {"q_heads": 7}, {"kv_heads": 0}, {"page": 0}, {"columns": 0}, {"pages": 0},
                        {"state": None}, {"state": POINTER + 2}, {"workspace": None}, {"size": 1000}, {"table_stride": -1}, {"slot_stride": -8}, {"scale": float("nan")}, {"scale": float("inf")}]),
            (UNSUPPORTED, [{"dtype": F32}, {"dtype": 9}, {"head_dim": 32}, {"head_dim": 96}, {"head_dim": 320}, {"rows": 70000},
                           {"columns": 1 << 20, "page": 1 << 10}, {"pages": 1 << 30, "page_stride": 1 << 20}]),
            (ARGUMENT, [{"workspace": POINTER + 8}]),
            (ALIGNMENT, [{"q": POINTER + 2}, {"k": POINTER + 8}, {"v": POINTER + 8}, {"out": 2 * POINTER + 8}, {"slot_stride": 132},
                         {"page_stride": 4100}, {"head_stride": 2052}, {"q_row": 1028}])):
        for changed in changes:
            assert call(**changed) == code, (changed, _native.library().mkb_last_error())


@needs_no_device
def test_outputs_that_overlap():
    row = 8 * 128 * 2
    assert read(out=POINTER) == CUDA                                        # in place
    assert read(out=POINTER, q_row=8 * 128 + 64) == ARGUMENT and read(out=POINTER, q_head=256, q_row=2048) == ARGUMENT
    assert read(out=POINTER + row) == ARGUMENT and read(out=POINTER - row) == ARGUMENT
    assert read(out=POINTER + 2 * row) == CUDA and read(out=POINTER - 2 * row) == CUDA
    qkv = 12 * 128 * 2
    assert rope(out=POINTER, q_row=qkv // 2) == ARGUMENT and rope(out=POINTER + 2 * qkv, q_row=qkv // 2) == CUDA
    assert adjust(out=POINTER + 2000) == ARGUMENT and adjust(out=POINTER + 4000) == CUDA and adjust(out=POINTER, out_stride=1001) == ARGUMENT
    beside = {"stride": 2100, "out_stride": 2100}      # two blocks of 1000 columns in rows of 2100
    assert adjust(out=POINTER + 2000, **beside) == CUDA == adjust(out=POINTER - 2000, **beside) == adjust(out=POINTER + 2200, **beside)
    assert adjust(out=POINTER + 1998, **beside) == ARGUMENT == adjust(out=POINTER + 2202, **beside) == adjust(out=POINTER - 1998, **beside)


@needs_no_device
def test_rotary_attention_refuses():
    for changed in ({"positions": None}, {"theta": 0.0}, {"theta": -1.0}, {"theta": float("nan")}, {"theta": float("inf")}):
        assert rope(**changed) == ARGUMENT, changed


@needs_no_device
def test_eviction_takes_and_refuses():
    for changed in ({}, {"sinks": 0, "recent": 0}, {"sinks": 28}, {"new_columns": 4, "budget": 100}):
        assert evict(**changed) == CUDA, changed
    assert evict(rows=0) == 0
    for changed in (*({name: None} for name in ("k", "v", "weights", "tables", "lengths", "new", "kept")), {"rows": -1}, {"budget": 0},
                    {"sinks": -1}, {"recent": -1}, {"sinks": 29}, {"recent": 32}, {"budget": 33}, {"new_columns": 0}, {"pages": 0}):
        assert evict(**changed) == ARGUMENT, changed
    assert evict(head_dim=80) == UNSUPPORTED and evict(k=POINTER + 4) == ALIGNMENT


@needs_no_device
def test_logits_taken_and_refused():
    for changed in ({}, {"dtype": F32}, {"tokens": None, "lengths": None}, {"mask": POINTER, "words": 32}, {"stride": 0, "out": 2 * POINTER},
                    {"bias": POINTER, "bias_tokens": POINTER, "biases": 3}, {"history": 0, "lengths": None}):
        assert adjust(**changed) == CUDA, changed
    assert adjust(rows=0) == 0
    for changed in ({"logits": None}, {"out": None}, {"lengths": None}, {"rows": -1}, {"width": 0}, {"offset": -1}, {"history": -1},
                    {"bias": POINTER}, {"bias_tokens": POINTER}, {"mask": POINTER, "words": 31}, {"mask": POINTER, "words": 32, "offset": 25},
                    {"out_stride": 999}, {"offset": (1 << 31) - 5}):
        assert adjust(**changed) == ARGUMENT, changed
    assert adjust(dtype=7) == UNSUPPORTED


def test_wrappers_refuse_host_tensors():
    pages, rows = torch.zeros(4, 1, 16, 64, dtype=torch.float16), torch.zeros(2, dtype=torch.int32)
    tables, q = torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, 4, 64, dtype=torch.float16)
    for call in (lambda: kernels.paged_attention_decode(q, rows, pages, pages, tables, q),
                 lambda: kernels.paged_rope_attention_decode(q.view(2, -1), rows, rows, pages, pages, tables, q, q_heads=2, kv_heads=1,
                                                             head_dim=64, theta=1e4),
                 lambda: kernels.evict_pages(pages, pages, torch.zeros(4, 1, 16), tables, rows, tables, budget=3),
                 lambda: kernels.adjust_logits(q.view(2, -1))):
        with pytest.raises(ValueError, match="CUDA"):
            call()
