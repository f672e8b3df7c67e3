"""GPU tests of attention over a paged cache and of eviction from it, against 64-bit restatements."""

import pytest
import torch

from mlkit_b200 import kernels
from tests.paged_reference import STEP, attend, evicted, make_cache, rotated, slots_of

pytestmark = pytest.mark.gpu
HALF, BRAIN = torch.float16, torch.bfloat16
THETA = 500000.0


def on_gpu(tensor):
    """A copy on the device with the same strides."""
    if tensor.dim() == 4 and not tensor.is_contiguous():
        return tensor.permute(0, 2, 1, 3).contiguous().cuda().permute(0, 2, 1, 3)
    return tensor.cuda()


def check_read(lengths, q_heads, kv_heads, head_dim, page, dtype, *, slots_first=False, columns=None, weigh=False, scale=None, seed=0):
    keys, values, tables, weights = make_cache(lengths, kv_heads=kv_heads, head_dim=head_dim, page=page, dtype=dtype,
                                               slots_first=slots_first, columns=columns, seed=seed)
    q = torch.randn(len(lengths), q_heads, head_dim, generator=torch.Generator().manual_seed(seed + 1)).to(dtype)
    out = torch.full_like(q, 7.0).cuda()
    held = weights.cuda() if weigh else None
    kernels.paged_attention_decode(q.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), on_gpu(keys), on_gpu(values),
                                   tables.cuda(), out, scale=scale, weights=held)
    got, added = out.cpu().double(), weights.double().clone()
    slack_of = torch.zeros_like(added)
    for row, n in enumerate(lengths):
        if n <= 0:
            assert torch.equal(got[row], torch.zeros_like(got[row])), row
            continue
        expected, bound, share, slack = attend(q[row].double(), slots_of(keys, tables[row], n), slots_of(values, tables[row], n),
                                               head_dim ** -0.5 if scale is None else scale, dtype, False)
        assert ((got[row] - expected).abs() <= bound).all(), (row, float(((got[row] - expected).abs() / bound).max()))
        slot = torch.arange(n)
        into = (tables[row, slot // page].long(), slice(None), slot % page)
        added[into] += share.sum(1).t()
        slack_of[into] = (share * slack).sum(1).t()
    if weigh:
        bound = slack_of + added * 2.0 ** -22
        assert ((held.cpu().double() - added).abs() <= bound).all()
    assert kernels.decode_status() == 0


@pytest.mark.parametrize("dtype", [HALF, BRAIN])
@pytest.mark.parametrize("head_dim", [64, 128, 192, 256])
@pytest.mark.parametrize("q_heads,kv_heads", [(4, 4), (8, 2), (5, 1), (8, 1), (18, 2), (16, 1), (40, 2)])
def test_attention_over_pages(dtype, head_dim, q_heads, kv_heads):
    check_read([1, 0, 37, -1, 16, 130, 515], q_heads, kv_heads, head_dim, 16, dtype, weigh=head_dim == 128 or q_heads == 18)


@pytest.mark.parametrize("page", [1, 2, 7, 16, 24, 64, 100, 256])
@pytest.mark.parametrize("slots_first", [False, True])
def test_pages_of_any_size_and_order(page, slots_first):
    check_read([3 * page, 3 * page + 1, max(1, 3 * page - 1), 1, 333], 8, 2, 64, page, HALF, slots_first=slots_first, weigh=True)


@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 1000, 4095, 4097])
def test_one_sequence_of_any_length(length):
    check_read([length], 4, 1, 128, 16, BRAIN, weigh=True)


@pytest.mark.parametrize("rows,longest", [(1, 40000), (3, 20000), (130, 300), (700, 40)])
def test_many_and_long_sequences(rows, longest):
    generator = torch.Generator().manual_seed(rows)
    lengths = torch.randint(-1, longest, (rows,), generator=generator).tolist()
    lengths[0] = longest
    check_read(lengths, 8, 2, 64, 32, HALF, weigh=True)


def test_tables_wider_than_the_lengths():
    check_read([100, 5, 0], 8, 1, 128, 16, HALF, columns=4000, weigh=True)


def test_a_scale_of_its_own():
    for scale in (0.0, 0.3, -0.2, 1.0):
        check_read([70, 200], 8, 2, 128, 16, HALF, scale=scale, weigh=True)


def test_sharp_and_flat_maps():
    """One slot far above thousands: the others' weights are below the 16-bit type's range and count together all the same."""
    n, width = 5000, 64
    keys = torch.zeros(1, 1, n, width)
    keys[0, 0, 1234, 0] = 8.0
    values = torch.randn(1, 1, n, width, generator=torch.Generator().manual_seed(3)) + 1
    values[0, 0, 1234] = 0.0
    keys, values = keys.half(), values.half()
    table = torch.zeros(1, 1, dtype=torch.int32)
    for top in (1.5, 2.0):      # exp(-12) and exp(-16) below the one slot: 5000 of them weigh 3 % and 0.06 %
        q = torch.zeros(1, 1, width, dtype=HALF)
        q[0, 0, 0] = top
        out = torch.empty_like(q).cuda()
        kernels.paged_attention_decode(q.cuda(), torch.tensor([n], dtype=torch.int32).cuda(), keys.cuda(), values.cuda(),
                                       table.cuda(), out, scale=1.0)
        expected, bound, _, _ = attend(q[0].double(), keys[0], values[0], 1.0, HALF, False)
        assert ((out.cpu().double()[0] - expected).abs() <= bound).all()


def test_queries_tables_and_pages_with_strides():
    lengths, q_heads, kv_heads, width = [40, 3, 129], 8, 2, 128
    keys, values, tables, _ = make_cache(lengths, kv_heads=kv_heads, head_dim=width, page=16, dtype=HALF)
    both = torch.stack((keys, values), 1).cuda()                              # keys and values of a page side by side
    wide = torch.randn(3, 2 * q_heads + 1, width, dtype=HALF, generator=torch.Generator().manual_seed(1))
    q = wide[:, 1::2]
    apart = torch.full((3, tables.shape[1] + 5), -1, dtype=torch.int32)
    apart[:, 2:2 + tables.shape[1]] = tables
    plain, strided = torch.empty(3, q_heads, width, dtype=HALF, device="cuda"), torch.empty(3, q_heads * width, dtype=HALF, device="cuda")
    held = torch.tensor(lengths, dtype=torch.int32).cuda()
    kernels.paged_attention_decode(q.contiguous().cuda(), held, keys.cuda(), values.cuda(), tables.cuda(), plain)
    kernels.paged_attention_decode(wide.cuda()[:, 1::2], held, both[:, 0], both[:, 1], apart.cuda()[:, 2:2 + tables.shape[1]], strided)
    assert torch.equal(plain.view(3, -1), strided)


def rope_case(lengths, positions, q_heads, kv_heads, width, page, dtype, slots_first=False, seed=0):
    keys, values, tables, weights = make_cache(lengths, kv_heads=kv_heads, head_dim=width, page=page, dtype=dtype,
                                               slots_first=slots_first, seed=seed, spare=1)
    qkv = torch.randn(len(lengths), (q_heads + 2 * kv_heads) * width, generator=torch.Generator().manual_seed(seed + 1)).to(dtype)
    return keys, values, tables, weights, qkv, torch.tensor(lengths, dtype=torch.int32), torch.tensor(positions, dtype=torch.int32)


def check_rope(lengths, positions, q_heads, kv_heads, width, page, dtype, *, slots_first=False, weigh=False, seed=0):
    keys, values, tables, weights, qkv, held, at = rope_case(lengths, positions, q_heads, kv_heads, width, page, dtype, slots_first, seed)
    k_gpu, v_gpu, w_gpu = on_gpu(keys), on_gpu(values), weights.cuda() if weigh else None
    out = torch.full((len(lengths), q_heads, width), 7.0, dtype=dtype, device="cuda")
    before = qkv.cuda()
    given = before.clone()
    kernels.paged_rope_attention_decode(given, at.cuda(), held.cuda(), k_gpu, v_gpu, tables.cuda(), out, q_heads=q_heads,
                                        kv_heads=kv_heads, head_dim=width, theta=THETA, weights=w_gpu)
    assert torch.equal(given, before)
    got, k_got, v_got = out.cpu().double(), k_gpu.cpu(), v_gpu.cpu()
    added, slack_of = weights.double().clone(), torch.zeros(weights.shape, dtype=torch.float64)
    touched = torch.zeros(keys.shape[0], page, dtype=torch.bool)
    for row, n in enumerate(lengths):
        if n < 0:
            assert torch.equal(got[row], torch.zeros_like(got[row]))
            continue
        q, k, v = qkv[row].view(-1, width).split((q_heads, kv_heads, kv_heads))
        id, slot = int(tables[row, n // page]), n % page
        touched[id, slot] = True
        turned = rotated(k, positions[row], THETA)
        # turned in 64 bits, rounded to 32 (2^-24 of the value, at most 2^-13 of half a step) and then to the cache's type
        assert ((k_got[id, :, slot].double() - turned).abs() <= STEP[dtype] * (1 + 2.0 ** -12) * turned.abs() + 2.0 ** -25).all()
        assert torch.equal(v_got[id, :, slot], v)
        expected, bound, share, slack = attend(rotated(q, positions[row], THETA), slots_of(k_got, tables[row], n + 1),
                                               slots_of(v_got, tables[row], n + 1), width ** -0.5, dtype, True)
        assert ((got[row] - expected).abs() <= bound).all(), (row, float(((got[row] - expected).abs() / bound).max()))
        slots = torch.arange(n + 1)
        into = (tables[row, slots // page].long(), slice(None), slots % page)
        added[id, :, slot] = 0
        added[into] += share.sum(1).t()
        slack_of[into] = (share * slack).sum(1).t()
    keep = ~touched[:, None, :, None]
    for new, old in ((k_got, keys), (v_got, values)):        # nothing else was written, bit for bit
        assert torch.equal(torch.where(keep, new, 0).view(torch.int16), torch.where(keep, old, 0).view(torch.int16))
    if weigh:
        assert ((w_gpu.cpu().double() - added).abs() <= slack_of + added * 2.0 ** -22).all()
    assert kernels.decode_status() == 0


@pytest.mark.parametrize("dtype", [HALF, BRAIN])
@pytest.mark.parametrize("head_dim", [64, 128, 192, 256])
@pytest.mark.parametrize("q_heads,kv_heads", [(2, 2), (8, 2), (20, 2), (24, 1)])
def test_rotary_append_and_attention(dtype, head_dim, q_heads, kv_heads):
    check_rope([0, 15, 16, -1, 200, 1, 47], [0, 15, 900, 4, 200, 131071, 47], q_heads, kv_heads, head_dim, 16, dtype,
               weigh=head_dim in (64, 128))


@pytest.mark.parametrize("page,slots_first", [(1, False), (3, True), (24, False), (64, True)])
def test_rotary_append_into_pages_of_any_size(page, slots_first):
    check_rope([page - 1, page, 5 * page, 0, 777], [3, 2, 1000000, 0, 5], 8, 2, 128, page, HALF, slots_first=slots_first, weigh=True)


@pytest.mark.parametrize("rows", [1, 64, 300])
def test_rotary_append_of_batches(rows):
    generator = torch.Generator().manual_seed(rows)
    lengths = torch.randint(-1, 400, (rows,), generator=generator).tolist()
    lengths[0] = 5000
    check_rope(lengths, [max(0, n) + 3 for n in lengths], 8, 2, 64, 16, BRAIN, weigh=True)


def test_rotary_rows_with_a_stride():
    keys, values, tables, _, qkv, held, at = rope_case([33, 5], [33, 9], 4, 1, 64, 16, HALF)
    outs = []
    for wide in (False, True):
        source = qkv.cuda()
        if wide:
            held_wide = torch.zeros(2, qkv.shape[1] + 64, dtype=HALF, device="cuda")
            held_wide[:, 32:32 + qkv.shape[1]] = source
            source = held_wide[:, 32:32 + qkv.shape[1]]
        outs.append(torch.empty(2, 256, dtype=HALF, device="cuda"))
        kernels.paged_rope_attention_decode(source, at.cuda(), held.cuda(), keys.cuda(), values.cuda(), tables.cuda(), outs[-1],
                                            q_heads=4, kv_heads=1, head_dim=64, theta=THETA)
    assert torch.equal(*outs)


@pytest.mark.parametrize("rope", [False, True])
def test_lengths_and_pages_out_of_range_are_left_out(rope):
    lengths = [40, 40, 40]
    keys, values, tables, weights, qkv, held, at = rope_case(lengths, lengths, 4, 1, 64, 16, HALF)
    k_gpu, v_gpu, w_gpu = keys.cuda(), values.cuda(), weights.cuda()

    def call(tables, held, weigh=None):
        out = torch.empty(3, 4, 64, dtype=HALF, device="cuda")
        if rope:
            kernels.paged_rope_attention_decode(qkv.cuda(), at.cuda(), held.cuda(), k_gpu, v_gpu, tables.cuda(), out, q_heads=4,
                                                kv_heads=1, head_dim=64, theta=THETA, weights=weigh)
        else:
            kernels.paged_attention_decode(qkv.cuda().view(3, 6, 64)[:, :4], held.cuda(), k_gpu, v_gpu, tables.cuda(), out, weights=weigh)
        return out

    good = call(tables, held)
    assert kernels.decode_status() == 0
    for entry in (-1, keys.shape[0], 1 << 30, -(1 << 31)):
        bad = tables.clone()
        bad[1, 1] = entry
        out = call(bad, held, w_gpu)
        assert kernels.decode_status() != 0 and kernels.decode_status() == 0
        assert torch.equal(out[0], good[0]) and torch.equal(out[2], good[2]) and torch.isfinite(out).all()
    if not rope:         # the slots of the page that is none are left out: the softmax is over the others
        n = [*range(16), *range(32, 40)]
        bad = tables.clone()
        bad[1, 1] = -1
        out = call(bad, held).cpu().double()[1]
        expected, bound, _, _ = attend(qkv.view(3, 6, 64)[1, :4].double(), slots_of(keys, tables[1], 40)[:, n],
                                       slots_of(values, tables[1], 40)[:, n], 64 ** -0.5, HALF, False)
        assert ((out - expected).abs() <= bound).all() and kernels.decode_status() != 0
    k_before = k_gpu.clone()
    for n in (tables.shape[1] * 16 + (0 if rope else 1), 1 << 30, (1 << 31) - 1):
        beyond = held.clone()
        beyond[2] = n
        out = call(tables, beyond)
        assert kernels.decode_status() != 0
        assert torch.equal(out[:2], good[:2])
    assert torch.equal(k_gpu.view(torch.int16), k_before.view(torch.int16))


def test_queries_that_are_not_numbers():
    """A NaN stays with its head, in short sequences and in those that several CTAs share."""
    lengths = [5, 9000]
    keys, values, tables, _ = make_cache(lengths, kv_heads=2, head_dim=64, page=16, dtype=HALF)
    q = torch.randn(2, 8, 64).half().cuda()
    good, out = torch.empty_like(q), torch.empty_like(q)
    arguments = (torch.tensor(lengths, dtype=torch.int32).cuda(), keys.cuda(), values.cuda(), tables.cuda())
    kernels.paged_attention_decode(q, *arguments, good)
    q[:, 3, 7] = float("nan")
    kernels.paged_attention_decode(q, *arguments, out)
    assert torch.isnan(out[:, 3]).all()
    assert torch.equal(out[:, [0, 1, 2, 4, 5, 6, 7]], good[:, [0, 1, 2, 4, 5, 6, 7]])


def test_every_page_out_of_range():
    keys, values, tables, _ = make_cache([40], kv_heads=1, head_dim=64, page=16, dtype=HALF)
    out = torch.full((1, 4, 64), 7.0, dtype=HALF, device="cuda")
    kernels.paged_attention_decode(torch.ones(1, 4, 64, dtype=HALF, device="cuda"), torch.tensor([40], dtype=torch.int32).cuda(),
                                   keys.cuda(), values.cuda(), torch.full_like(tables, -1).cuda(), out)
    assert torch.equal(out, torch.zeros_like(out)) and kernels.decode_status() != 0


def test_results_repeat_bit_for_bit():
    lengths = [2000, 17, 0, 900, 5000]
    keys, values, tables, weights = make_cache(lengths, kv_heads=2, head_dim=128, page=16, dtype=BRAIN)
    q, held = torch.randn(5, 16, 128).to(BRAIN).cuda(), torch.tensor(lengths, dtype=torch.int32).cuda()
    keys, values, tables = keys.cuda(), values.cuda(), tables.cuda()
    first = None
    for _ in range(20):
        out, added = torch.empty_like(q), weights.cuda()
        kernels.paged_attention_decode(q, held, keys, values, tables, out, weights=added)
        first = first or (out, added)
        assert torch.equal(out, first[0]) and torch.equal(added, first[1])


def test_steps_in_a_row_without_waiting():
    """Lengths, tables and queries change on the device between calls: as with a wait behind every kernel, bit for bit."""
    results = []
    for wait in (False, True):
        lengths = [200, 33, 700, 5]
        keys, values, tables, weights, _, held, _ = rope_case(lengths, lengths, 8, 2, 64, 16, HALF, seed=4)
        wide = torch.full((4, 80), -1, dtype=torch.int32)
        wide[:, :tables.shape[1]] = tables
        fresh = iter(range(keys.shape[0], keys.shape[0] + 40))
        for row in range(4):
            for column in range(-(-(lengths[row] + 1) // 16), -(-(lengths[row] + 121) // 16)):
                wide[row, column] = next(fresh)
        more = lambda pool: torch.cat((pool, torch.zeros(40, *pool.shape[1:], dtype=pool.dtype))).cuda()
        k, v, w, held, tables, shown = more(keys), more(values), more(weights), held.cuda(), torch.full_like(wide, -1).cuda(), wide.cuda()
        generator, out = torch.Generator(device="cuda").manual_seed(0), []
        for step in range(120):
            qkv = torch.randn(4, 12 * 64, device="cuda", generator=generator).half()
            tables.copy_(shown)
            out.append(torch.empty(4, 8, 64, dtype=HALF, device="cuda"))
            kernels.paged_rope_attention_decode(qkv, held, held, k, v, tables, out[-1], q_heads=8, kv_heads=2, head_dim=64, theta=THETA, weights=w)
            held.add_(1)
            if wait:
                torch.cuda.synchronize()
        results.append((torch.stack(out), k, v, w, held))
    for one, other in zip(*results):
        assert torch.equal(one.view(torch.int16) if one.dtype == HALF else one, other.view(torch.int16) if other.dtype == HALF else other)
    assert kernels.decode_status() == 0


def test_streams_and_graphs_that_overlap():
    """Two graphs captured on one stream and replayed on two at once, between eager calls on a third; lengths change in place."""
    cases = []
    for seed in range(3):
        lengths = [3000 + 500 * seed, 40, 700]
        keys, values, tables, weights = make_cache(lengths, kv_heads=2, head_dim=128, page=16, dtype=HALF, seed=seed)
        q = torch.randn(3, 8, 128, generator=torch.Generator().manual_seed(seed)).half()
        cases.append({"q": q.cuda(), "held": torch.tensor(lengths, dtype=torch.int32).cuda(), "k": keys.cuda(), "v": values.cuda(),
                      "t": tables.cuda(), "out": torch.empty(3, 8, 128, dtype=HALF, device="cuda"), "w": weights.cuda()})

    def call(c, out=None):
        kernels.paged_attention_decode(c["q"], c["held"], c["k"], c["v"], c["t"], c["out"] if out is None else out)

    expected = {}
    for shorter in (0, 1):
        for i, c in enumerate(cases):
            if shorter:
                c["held"].sub_(7)
            expected[i, shorter] = torch.empty_like(c["out"])
            call(c, expected[i, shorter])
    for c in cases:
        c["held"].add_(7)
    graphs, side = [], torch.cuda.Stream()
    torch.cuda.synchronize()
    for c in cases[:2]:
        with torch.cuda.stream(side):
            call(c)
            side.synchronize()
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=side):
                call(c)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for shorter in (0, 1):
        torch.cuda.synchronize()
        for _ in range(30):
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
            with torch.cuda.stream(streams[2]):
                call(cases[2])
        torch.cuda.synchronize()
        for i, c in enumerate(cases):
            assert torch.equal(c["out"], expected[i, shorter]), (i, shorter)
            c["held"].sub_(7)


def test_captured_calls_when_no_cleared_state_is_left(monkeypatch):
    """Their graphs clear one of their own; and a captured call never shares one with another."""
    lengths = [3000, 40]
    keys, values, tables, weights = make_cache(lengths, kv_heads=1, head_dim=64, page=16, dtype=HALF)
    q, held = torch.randn(2, 8, 64).half().cuda(), torch.tensor(lengths, dtype=torch.int32).cuda()
    pool = (held, keys.cuda(), values.cuda(), tables.cuda())
    expected = torch.empty_like(q)
    kernels.paged_attention_decode(q, *pool, expected)
    scratch = kernels._attention_scratch[q.device.index]
    outs, graphs, side, left = [], [], torch.cuda.Stream(), len(scratch.left)
    for attempt in range(4):
        if attempt == 2:
            monkeypatch.setattr(scratch, "left", [])
        outs.append(torch.empty_like(q))
        graphs.append(torch.cuda.CUDAGraph())
        torch.cuda.synchronize()
        with torch.cuda.graph(graphs[-1], stream=side):
            kernels.paged_attention_decode(q, *pool, outs[-1])
        if attempt < 2:
            assert len(scratch.left) == left - attempt - 1
    for _ in range(20):
        for graph, stream in zip(graphs, [torch.cuda.Stream() for _ in graphs]):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out, expected) for out in outs)


def test_attention_in_place():
    lengths = [2500, 3, 0, 90]
    keys, values, tables, _ = make_cache(lengths, kv_heads=2, head_dim=128, page=16, dtype=HALF)
    q = torch.randn(4, 8, 128).half().cuda()
    pool = (torch.tensor(lengths, dtype=torch.int32).cuda(), keys.cuda(), values.cuda(), tables.cuda())
    out = torch.empty_like(q)
    kernels.paged_attention_decode(q, *pool, out)
    kernels.paged_attention_decode(q, *pool, q)
    assert torch.equal(q, out)


def test_sequences_that_share_pages():
    """A common prefix is in two tables: read by both, written by neither."""
    keys, values, tables, _ = make_cache([40, 40], kv_heads=1, head_dim=64, page=16, dtype=HALF)
    tables[1, :2] = tables[0, :2]
    q = torch.randn(2, 4, 64).half()
    out = torch.empty(2, 4, 64, dtype=HALF, device="cuda")
    kernels.paged_attention_decode(q.cuda(), torch.tensor([40, 40], dtype=torch.int32).cuda(), keys.cuda(), values.cuda(), tables.cuda(), out)
    for row in (0, 1):
        expected, bound, _, _ = attend(q[row].double(), slots_of(keys, tables[row], 40), slots_of(values, tables[row], 40), 0.125, HALF, False)
        assert ((out.cpu().double()[row] - expected).abs() <= bound).all()


def test_layouts_are_told_apart():
    """Calls of one shape and other strides, types or tables, in turn: none takes another's checked layout."""
    lengths = [33, 70]
    for attempt in range(2):
        for dtype, slots_first, columns in ((HALF, False, None), (BRAIN, False, None), (HALF, True, None), (HALF, False, 9), (HALF, False, None)):
            check_read(lengths, 4, 2, 64, 16, dtype, slots_first=slots_first, columns=columns, weigh=attempt == 1)
    q, pages = torch.zeros(2, 4, 64, dtype=HALF, device="cuda"), torch.zeros(9, 2, 16, 64, dtype=HALF, device="cuda")
    tables, held = torch.zeros(2, 3, dtype=torch.int32, device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda")
    good = dict(q=q, lengths=held, k_pages=pages, v_pages=pages.clone(), tables=tables, out=torch.empty_like(q))
    kernels.paged_attention_decode(**good)
    for name, bad in (("q", q.to(BRAIN)), ("q", q[:, :, ::2]), ("lengths", held.long()), ("lengths", held[:1]), ("k_pages", pages.to(BRAIN)),
                      ("v_pages", pages[:8]), ("v_pages", pages.permute(0, 1, 3, 2)), ("tables", tables.long()), ("tables", tables[:1]),
                      ("tables", tables.t().contiguous().t()), ("out", q[:1]), ("out", q.float()), ("out", q.cpu()), ("lengths", held.cpu()),
                      ("tables", tables.cpu()), ("k_pages", pages.cpu())):
        for _ in range(2):
            with pytest.raises(ValueError):
                kernels.paged_attention_decode(**(good | {name: bad}))
    for weights in (torch.zeros(9, 2, 16, dtype=HALF, device="cuda"), torch.zeros(9, 2, 15, device="cuda"), torch.zeros(9, 2, 16)):
        with pytest.raises(ValueError):
            kernels.paged_attention_decode(**good, weights=weights)


def test_pools_whose_offsets_pass_32_bits():
    """Elements beyond 2^32 bytes and 2^31 elements: the last pages of a pool of 2^32 + bytes."""
    page, heads, width = 256, 8, 128
    pages = (1 << 31) // (page * heads * width) + 9
    keys, values = (torch.empty(pages, heads, page, width, dtype=HALF, device="cuda") for _ in range(2))
    lengths, last = [700], [pages - 1, pages - 3, pages - 2]
    small_k, small_v, tables, _ = make_cache(lengths, kv_heads=heads, head_dim=width, page=page, dtype=HALF, extra=0)
    far = torch.empty_like(tables)
    for column, id in enumerate(last):
        keys[id], values[id], far[0, column] = small_k[tables[0, column]].cuda(), small_v[tables[0, column]].cuda(), id
    q, held = torch.randn(1, 16, width).half().cuda(), torch.tensor(lengths, dtype=torch.int32).cuda()
    near, distant = torch.empty_like(q), torch.empty_like(q)
    kernels.paged_attention_decode(q, held, small_k.cuda(), small_v.cuda(), tables.cuda(), near)
    kernels.paged_attention_decode(q, held, keys, values, far.cuda(), distant)
    assert torch.equal(near, distant)


# ------------------------------------------------------------------------------------------------ eviction


def check_evict(lengths, kv_heads, width, page, budget, sinks, recent, dtype, *, slots_first=False, shape_weights=None, seed=0):
    keys, values, tables, weights = make_cache(lengths, kv_heads=kv_heads, head_dim=width, page=page, dtype=dtype,
                                               slots_first=slots_first, seed=seed, extra=2 + sum(-(-min(max(n, 0), budget) // page) for n in lengths))
    if shape_weights is not None:
        weights = shape_weights(weights)
    taken = set()
    for row, n in enumerate(lengths):
        taken |= set(tables[row, :-(-max(n, 0) // page)].tolist())
    free = [id for id in range(keys.shape[0]) if id not in taken]
    fresh = torch.full((len(lengths), -(-budget // page)), -7, dtype=torch.int32)
    for row, n in enumerate(lengths):
        for column in range(-(-min(max(n, 0), budget) // page)):
            fresh[row, column] = free.pop()
    k_gpu, v_gpu, w_gpu = on_gpu(keys), on_gpu(values), weights.cuda()
    kept = kernels.evict_pages(k_gpu, v_gpu, w_gpu, tables.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), fresh.cuda(),
                               budget=budget, sinks=sinks, recent=recent).cpu()
    expected_k, expected_v, expected_w = keys.clone(), values.clone(), weights.clone()
    for row, n in enumerate(lengths):
        for head in range(kv_heads):
            slots = evicted(slots_of(weights, tables[row], n)[head], budget, sinks, recent) if n > 0 else []
            assert kept[row, head].tolist() == slots + [-1] * (budget - len(slots)), (row, head)
            old, new = torch.tensor(slots, dtype=torch.long), torch.arange(len(slots))
            source = (tables[row, old // page].long(), head, old % page)
            target = (fresh[row, new // page].long(), head, new % page)
            for data, given in ((expected_k, keys), (expected_v, values), (expected_w, weights)):
                data[target] = given[source]
    assert torch.equal(k_gpu.cpu().view(torch.int16), expected_k.view(torch.int16))
    assert torch.equal(v_gpu.cpu().view(torch.int16), expected_v.view(torch.int16))
    assert torch.equal(w_gpu.cpu().view(torch.int32), expected_w.view(torch.int32))
    assert kernels.decode_status() == 0


@pytest.mark.parametrize("lengths,budget,sinks,recent", [
    ([50, 20, 0, -1, 33], 32, 2, 8), ([100], 1, 0, 0), ([100], 1, 1, 0), ([100], 1, 0, 1), ([64], 64, 3, 4), ([65], 64, 32, 32),
    ([5000, 1, 1025, 1024], 1024, 4, 100), ([300, 299], 299, 0, 0), ([3000], 2999, 0, 2999)])
def test_eviction_keeps_the_heaviest(lengths, budget, sinks, recent):
    check_evict(lengths, 2, 64, 16, budget, sinks, recent, HALF)


@pytest.mark.parametrize("dtype", [HALF, BRAIN])
@pytest.mark.parametrize("width", [64, 128, 192, 256])
@pytest.mark.parametrize("page,slots_first", [(1, False), (7, True), (16, False), (64, True)])
def test_eviction_moves_rows(dtype, width, page, slots_first):
    check_evict([90, 40, 131], 3, width, page, 60, 4, 10, dtype, slots_first=slots_first)


@pytest.mark.parametrize("kind", ["equal", "few", "zeros", "wild", "subnormal"])
def test_ties_and_odd_weights(kind):
    def shape(weights):
        if kind == "equal":
            return torch.full_like(weights, 0.25)
        if kind == "few":
            return (weights * 2).floor()
        if kind == "zeros":        # a negative zero equals zero
            return torch.where(weights > 1.5, 0.0, -0.0) * 1.0
        if kind == "subnormal":
            return weights.sub(1.5) * 2.0 ** -140
        wild = torch.tensor([float("nan"), float("inf"), -float("inf"), -1.0])
        return torch.where(weights > 2, wild[(weights * 1000).long() % 4], weights)
    check_evict([700, 130, 64], 2, 64, 16, 100, 4, 20, HALF, shape_weights=shape)


def test_eviction_of_long_sequences():
    check_evict([40000, 70001], 1, 64, 64, 5000, 4, 512, BRAIN)


def test_evicted_sequences_share_no_pages_with_a_prefix_of_others():
    """Two sequences that share their first pages are evicted: the shared pages stay as they were."""
    keys, values, tables, weights = make_cache([64, 64], kv_heads=1, head_dim=64, page=16, dtype=HALF, extra=5)
    tables[1, :2] = tables[0, :2]
    free = [id for id in range(keys.shape[0]) if id not in set(tables.flatten().tolist())][:4]
    fresh = torch.tensor([free[:2], free[2:]], dtype=torch.int32)
    k_gpu, v_gpu, w_gpu = keys.cuda(), values.cuda(), weights.cuda()
    held = torch.tensor([64, 64], dtype=torch.int32).cuda()
    kept = kernels.evict_pages(k_gpu, v_gpu, w_gpu, tables.cuda(), held, fresh.cuda(), budget=32, recent=4).cpu()
    for row in (0, 1):
        slots = evicted(slots_of(weights, tables[row], 64)[0], 32, 0, 4)
        assert kept[row, 0].tolist() == slots
        assert torch.equal(slots_of(k_gpu.cpu(), fresh[row], 32)[0], slots_of(keys, tables[row], 64)[0, slots])
    for id in set(tables.flatten().tolist()):
        assert torch.equal(k_gpu[id].cpu(), keys[id])


def test_eviction_with_pages_out_of_range():
    keys, values, tables, weights = make_cache([64, 64], kv_heads=1, head_dim=64, page=16, dtype=HALF, extra=5)
    k_gpu, v_gpu, w_gpu = keys.cuda(), values.cuda(), weights.cuda()
    held = torch.tensor([64, 64], dtype=torch.int32).cuda()
    free = [id for id in range(keys.shape[0]) if id not in set(tables.flatten().tolist())]
    for old, new in ((-1, free[2]), (1 << 30, free[2]), (int(tables[1, 1]), keys.shape[0]), (int(tables[1, 1]), -(1 << 31))):
        bad, fresh = tables.clone(), torch.tensor([free[:2], [free[3], new]], dtype=torch.int32)
        bad[1, 1] = old
        kept = kernels.evict_pages(k_gpu, v_gpu, w_gpu, bad.cuda(), held, fresh.cuda(), budget=32, recent=4).cpu()
        assert kernels.decode_status() != 0
        assert kept[0, 0].tolist() == evicted(slots_of(weights, tables[0], 64)[0], 32, 0, 4)
        assert torch.equal(slots_of(k_gpu.cpu(), fresh[0], 32)[0], slots_of(keys, tables[0], 64)[0, kept[0, 0].long()])
    kernels.evict_pages(k_gpu, v_gpu, w_gpu, tables.cuda(), torch.tensor([65, 1 << 30], dtype=torch.int32).cuda(),
                        torch.tensor([free[:2], free[2:4]], dtype=torch.int32).cuda(), budget=32, recent=4)
    assert kernels.decode_status() != 0
